// kv_abi.cu -- the b200q8_kv_* entry points: argument checks and dispatch.
#include "kv_device.cuh"

#include <cmath>

namespace b200q8 {
b200q8_status_t set_error(b200q8_status_t code, const char * fmt, ...);
b200q8_status_t cuda_error(cudaError_t e, const char * what);
int             current_sm_count();

namespace {

constexpr int64_t kMaxCells = (int64_t) 1 << 30;

bool kv_shape_ok(int64_t n_slots, int64_t n_ctx, int64_t n_kv, int64_t head_dim) {
    return n_slots >= 1 && n_slots <= (1 << 20) && n_ctx >= 64 && n_ctx <= kMaxCells && n_ctx % 64 == 0 && n_kv >= 1 &&
           n_kv <= 1024 && head_dim >= 32 && head_dim <= 256 && head_dim % 32 == 0;
}

bool kv_type_ok(int32_t t) {
    return t == B200Q8_KV_Q4_0 || t == B200Q8_KV_Q8_0;
}

int element_bytes(int32_t type) {
    return type == B200Q8_SRC_F32 ? 4 : type == B200Q8_SRC_F16 || type == B200Q8_SRC_BF16 ? 2 : 0;
}

bool is_aligned(const void * p, size_t a) {
    return reinterpret_cast<uintptr_t>(p) % a == 0;
}

b200q8_status_t kv_views(const char * what, const b200q8_kv_cache * cache, const b200q8_kv_batch * batch,
                         KvCacheView & c, KvRuns & b) {
    if (cache == nullptr || batch == nullptr) {
        return set_error(B200Q8_ERR_INVALID_ARG, "%s: null cache or batch", what);
    }
    if (!kv_type_ok(cache->type_k) || !kv_type_ok(cache->type_v) ||
        !kv_shape_ok(cache->n_slots, cache->n_ctx, cache->n_kv, cache->head_dim)) {
        return set_error(B200Q8_ERR_INVALID_ARG,
                         "%s: bad cache (types Q4_0 or Q8_0; n_ctx a multiple of 64 up to 2^30; head_dim a multiple "
                         "of 32 up to 256; n_slots up to 2^20, n_kv up to 1024)", what);
    }
    if (cache->sinks < 0 || cache->ring < 0 || cache->ring > 1 || (cache->ring && cache->sinks >= cache->n_ctx)) {
        return set_error(B200Q8_ERR_INVALID_ARG, "%s: sinks must not be negative, and leave cells to a ring", what);
    }
    const void * arrays[4] = { cache->k_codes, cache->k_scales, cache->v_codes, cache->v_scales };
    for (const void * p : arrays) {
        if (p == nullptr || !is_aligned(p, 16)) {
            return set_error(B200Q8_ERR_INVALID_ARG, "%s: the cache's arrays must be 16-byte aligned device memory",
                             what);
        }
    }
    const int64_t n = batch->n_seqs, m = batch->n_tokens;
    if (n < 0 || n > 65535 || m < 0 || m > INT32_MAX || batch->max_len < 0 || batch->max_len > kMaxCells ||
        (batch->starts == nullptr && m != n)) {
        return set_error(B200Q8_ERR_INVALID_ARG,
                         "%s: bad batch (up to 65535 runs; without starts, one row a run)", what);
    }
    if (n > 0 && m > 0 &&
        (batch->pos == nullptr || !is_aligned(batch->pos, 4) || !is_aligned(batch->starts, 4) ||
         !is_aligned(batch->slots, 4) || batch->max_len < 1)) {
        return set_error(B200Q8_ERR_INVALID_ARG, "%s: the batch needs pos, 4-byte aligned arrays and max_len >= 1",
                         what);
    }
    if (batch->slots == nullptr && n > cache->n_slots) {
        return set_error(B200Q8_ERR_INVALID_ARG, "%s: %lld runs need explicit slots beyond n_slots", what,
                         (long long) n);
    }
    c.codes[0]  = static_cast<uint8_t *>(cache->k_codes);
    c.codes[1]  = static_cast<uint8_t *>(cache->v_codes);
    c.scales[0] = static_cast<__half *>(cache->k_scales);
    c.scales[1] = static_cast<__half *>(cache->v_scales);
    c.four[0]   = cache->type_k == B200Q8_KV_Q4_0;
    c.four[1]   = cache->type_v == B200Q8_KV_Q4_0;
    c.n_slots   = (int) cache->n_slots;
    c.n_ctx     = (int) cache->n_ctx;
    c.n_kv      = (int) cache->n_kv;
    c.nb        = (int) cache->head_dim / 32;
    c.sinks     = cache->sinks;
    c.ring      = cache->ring ? (int) cache->n_ctx - cache->sinks : 0;
    b.starts    = batch->starts;
    b.pos       = batch->pos;
    b.slots     = batch->slots;
    b.n_seqs    = (int) n;
    b.n_tokens  = (int) m;
    b.max_len   = batch->starts ? (int) batch->max_len : 1;
    b.slot_base = 0;
    return B200Q8_OK;
}

// Checks of an array of rows of `values` values; *wide: whether 4 values can be accessed at a time.
bool rows_ok(const void * p, size_t stride, int es, int64_t values, int64_t rows, int * wide) {
    if (p == nullptr || !is_aligned(p, es) || stride % es != 0 || (rows > 1 && stride < (size_t) values * es)) {
        return false;
    }
    *wide = *wide && is_aligned(p, 4 * es) && (rows == 1 || stride % (4 * es) == 0);
    return true;
}

b200q8_status_t kv_rows(const char * what, bool write, const b200q8_kv_cache * cache, const b200q8_kv_batch * batch,
                        const void * k, size_t k_stride, const void * v, size_t v_stride, int32_t type,
                        b200q8_stream_t stream) {
    KvRowsArgs            a  = {};
    cudaStream_t          st = reinterpret_cast<cudaStream_t>(stream);
    const b200q8_status_t s  = kv_views(what, cache, batch, a.c, a.b);
    if (s != B200Q8_OK) {
        return s;
    }
    const int es = element_bytes(type);
    if (es == 0) {
        return set_error(B200Q8_ERR_INVALID_ARG, "%s: unknown element type %d", what, type);
    }
    if (write && a.c.ring && a.b.max_len > a.c.ring) {
        return set_error(B200Q8_ERR_INVALID_ARG, "%s: a run of up to %d rows does not fit the ring's %d cells", what,
                         a.b.max_len, a.c.ring);
    }
    if (a.b.n_seqs == 0 || a.b.n_tokens == 0) {
        return B200Q8_OK;
    }
    const int64_t values = (int64_t) a.c.n_kv * a.c.nb * 32;
    if ((int64_t) a.b.max_len * a.c.n_kv * a.c.nb > UINT32_MAX) {
        return set_error(B200Q8_ERR_UNSUPPORTED, "%s: max_len * n_kv * head_dim / 32 must fit in 32 bits", what);
    }
    a.wide = 1;
    if (!rows_ok(k, k_stride, es, values, a.b.n_tokens, &a.wide) ||
        !rows_ok(v, v_stride, es, values, a.b.n_tokens, &a.wide)) {
        return set_error(B200Q8_ERR_INVALID_ARG, "%s: bad row pointer, alignment or stride", what);
    }
    a.src[0] = k;
    a.src[1] = v;
    a.dst[0] = const_cast<void *>(k);
    a.dst[1] = const_cast<void *>(v);
    a.stride[0] = k_stride;
    a.stride[1] = v_stride;
    a.type      = type;
    const cudaError_t e = write ? launch_kv_write(a, st) : launch_kv_read(a, st);
    return e == cudaSuccess ? B200Q8_OK : cuda_error(e, what);
}

}  // namespace

cudaError_t kv_device_status(unsigned * word, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(word, g_kv_status, sizeof(*word));
    if (e == cudaSuccess && clear && *word != 0u) {
        const unsigned zero = 0u;
        e                   = cudaMemcpyToSymbol(g_kv_status, &zero, sizeof(zero));
    }
    return e;
}

}  // namespace b200q8

using namespace b200q8;

extern "C" {

size_t b200q8_kv_codes_bytes(int32_t type, int64_t n_slots, int64_t n_ctx, int64_t n_kv, int64_t head_dim) {
    if (!kv_type_ok(type) || !kv_shape_ok(n_slots, n_ctx, n_kv, head_dim)) {
        return 0;
    }
    return (size_t) n_slots * n_ctx * n_kv * (type == B200Q8_KV_Q4_0 ? head_dim / 2 : head_dim);
}

size_t b200q8_kv_scales_bytes(int64_t n_slots, int64_t n_ctx, int64_t n_kv, int64_t head_dim) {
    return kv_shape_ok(n_slots, n_ctx, n_kv, head_dim) ? (size_t) n_slots * n_ctx * n_kv * (head_dim / 32) * 2 : 0;
}

b200q8_status_t b200q8_kv_write(const b200q8_kv_cache * cache, const b200q8_kv_batch * batch, const void * k,
                                size_t k_row_stride, const void * v, size_t v_row_stride, int32_t src_type,
                                b200q8_stream_t stream) {
    return kv_rows("kv_write", true, cache, batch, k, k_row_stride, v, v_row_stride, src_type, stream);
}

b200q8_status_t b200q8_kv_read(const b200q8_kv_cache * cache, const b200q8_kv_batch * batch, void * k,
                               size_t k_row_stride, void * v, size_t v_row_stride, int32_t dst_type,
                               b200q8_stream_t stream) {
    return kv_rows("kv_read", false, cache, batch, k, k_row_stride, v, v_row_stride, dst_type, stream);
}

b200q8_status_t b200q8_kv_attend(const b200q8_kv_cache * cache, const b200q8_kv_batch * batch, const void * q,
                                 size_t q_row_stride, void * out, size_t out_row_stride, int32_t type, int64_t n_head,
                                 int64_t window, float scale, b200q8_stream_t stream) {
    KvAttendArgs          a  = {};
    cudaStream_t          st = reinterpret_cast<cudaStream_t>(stream);
    const b200q8_status_t s  = kv_views("kv_attend", cache, batch, a.c, a.b);
    if (s != B200Q8_OK) {
        return s;
    }
    const int es = element_bytes(type);
    if (es == 0) {
        return set_error(B200Q8_ERR_INVALID_ARG, "kv_attend: unknown element type %d", type);
    }
    if (n_head < 1 || n_head % a.c.n_kv != 0 || n_head / a.c.n_kv > 64) {
        return set_error(B200Q8_ERR_INVALID_ARG, "kv_attend: n_head (%lld) must be 1 to 64 times n_kv (%d)",
                         (long long) n_head, a.c.n_kv);
    }
    if (window < 0 || !std::isfinite(scale)) {
        return set_error(B200Q8_ERR_INVALID_ARG, "kv_attend: window must not be negative and scale finite");
    }
    if (a.c.ring && (window == 0 || window > a.c.ring || window + a.b.max_len - 1 > a.c.ring)) {
        return set_error(B200Q8_ERR_INVALID_ARG,
                         "kv_attend: a ring cache needs a window, and window + max_len - 1 at most its %d cells",
                         a.c.ring);
    }
    if (a.b.n_seqs == 0 || a.b.n_tokens == 0) {
        return B200Q8_OK;
    }
    if ((int64_t) a.b.max_len * (n_head / a.c.n_kv) > INT32_MAX / 2) {
        return set_error(B200Q8_ERR_UNSUPPORTED, "kv_attend: max_len * n_head / n_kv must stay below 2^30");
    }
    const int64_t values = n_head * a.c.nb * 32;
    int           wide   = 1;
    if (!rows_ok(q, q_row_stride, es, values, a.b.n_tokens, &wide) ||
        !rows_ok(out, out_row_stride, es, values, a.b.n_tokens, &wide)) {
        return set_error(B200Q8_ERR_INVALID_ARG, "kv_attend: bad row pointer, alignment or stride");
    }
    a.q          = q;
    a.out        = out;
    a.q_stride   = q_row_stride;
    a.out_stride = out_row_stride;
    a.type       = type;
    a.n_head     = (int) n_head;
    a.group      = (int) n_head / a.c.n_kv;
    a.wide       = wide;
    a.window     = window > kMaxCells ? 0 : (int) window;  // wider than any prefix of a plain cache
    a.scale      = scale != 0.0f ? scale : 1.0f / sqrtf((float) (a.c.nb * 32));
    const cudaError_t e = launch_kv_attend(a, st, current_sm_count());
    return e == cudaSuccess ? B200Q8_OK : cuda_error(e, "kv_attend launch");
}

}  // extern "C"
