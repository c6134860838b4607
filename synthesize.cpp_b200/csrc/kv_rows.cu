// kv_rows.cu -- rows of keys and values into the quantised cache, and back.
//
// Writing: four lanes hold one 32-value block, eight consecutive values each -
// a key row's chunk of the block, or two neighbouring chunks of a value row.
// The largest magnitude is folded over the four lanes by shuffles, each lane
// rounds its own values, and its codes are one or two aligned stores.  It is
// bound by the rounding, about ten operations a value: 12 prompts (12187 rows
// of 8 heads of 128) take 34 us, 3.4 TB/s (with four values a lane 41 us: half
// of the work was addresses and folds).
// Reading back: eight lanes a block, so that a lane's four floats are next to
// its neighbour's in one store (eight a lane write half sectors: 149 us
// against 123 us for 65536 rows); bound by the floats it writes, 5.0 TB/s.
// Either is bound by launch and memory latency when a call has few rows.
#include "common.cuh"
#include "kv_device.cuh"

#include <algorithm>

namespace b200q8 {
namespace {

constexpr int kRowThreads = 256;

// A group of LANES lanes keeps one block of the row (its head and place are found once) and
// goes down the tokens of the CTA's tile.  grid: x over token tiles times
// chunks of blocks, y over keys and values, z over runs.
struct RowsWork {
    int    unit, head, block;   // of the row
    int    token, step, tokens; // first token, and on to the end in steps
    bool   some;
    size_t plane;               // (slot, head)'s first cell
};

template <int LANES>
__device__ __forceinline__ RowsWork rows_work(const KvRowsArgs & a, const KvRun & r, int per_cta) {
    constexpr int kGroups = kRowThreads / LANES;
    RowsWork  w;
    const int per    = a.c.n_kv * a.c.nb;
    const int chunks = (per + kGroups - 1) / kGroups;
    const int group  = threadIdx.x / LANES;
    const int tile = chunks == 1 ? blockIdx.x : blockIdx.x / chunks, chunk = chunks == 1 ? 0 : blockIdx.x % chunks;
    w.step   = max(1, kGroups / per);  // tokens side by side when a row has few blocks
    const int side = per < kGroups ? group / per : 0;
    w.unit   = per < kGroups ? group % per : chunk * kGroups + group;
    w.some   = w.unit < per && side < w.step;
    w.unit   = w.some ? w.unit : 0;
    w.head   = w.unit / a.c.nb;
    w.block  = w.unit % a.c.nb;
    w.token  = tile * per_cta + side;
    w.tokens = w.some ? min(r.len, (tile + 1) * per_cta) : 0;
    w.plane  = ((size_t) r.slot * a.c.n_kv + w.head) * a.c.n_ctx;
    return w;
}

// kAhead: tokens whose rows a thread loads before it uses one.
template <int kAhead>
__global__ void __launch_bounds__(kRowThreads) kv_write_kernel(const KvRowsArgs a, const int per_cta) {
    pdl_launch_dependents();
    pdl_wait_primary();
    const int   t = blockIdx.y;
    const KvRun r = kv_run(a.b, a.c, blockIdx.z);
    if (!r.ok) {
        if (blockIdx.x == 0 && t == 0 && threadIdx.x == 0) {
            kv_report();
        }
        return;
    }
    const int      part = threadIdx.x & 3;
    const RowsWork w    = rows_work<4>(a, r, per_cta);
    const int      es   = a.type == kSrcF32 ? 4 : 2;
    const bool     four = a.c.four[t] != 0;
    const size_t   row_bytes = (size_t) (a.c.nb * (four ? 16 : 32));
    const uint8_t * src = static_cast<const uint8_t *>(a.src[t]) + (size_t) r.row * a.stride[t] +
                          (size_t) (w.unit * 32 + part * 8) * es;
    // the lane's codes: eight of a key chunk, or four of each of two value chunks
    uint8_t *        codes  = a.c.codes[t] + w.plane * row_bytes + kv_code_offset(t, four, a.c.nb, w.block, 2 * part);
    const int        apart  = kv_code_offset(t, four, a.c.nb, w.block, 2 * part + 1) - kv_code_offset(t, four, a.c.nb, w.block, 2 * part);
    unsigned short * scales = reinterpret_cast<unsigned short *>(a.c.scales[t]) + w.plane * a.c.nb + w.block;
    // shuffles below take whole warps: every group makes as many rounds
    for (int first = w.token; __any_sync(0xffffffffu, first < w.tokens); first += kAhead * w.step) {
        uint4 raw[kAhead][2];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int token = first + k * w.step;
            raw[k][0] = raw[k][1] = make_uint4(0u, 0u, 0u, 0u);
            if (token < w.tokens) {
                raw[k][0] = load4_raw(src + (size_t) token * a.stride[t], es, a.wide);
                raw[k][1] = load4_raw(src + (size_t) token * a.stride[t] + 4 * es, es, a.wide);
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int      token = first + k * w.step;
            const float4   x = widen4(raw[k][0], a.type), y = widen4(raw[k][1], a.type);
            const float    v[8] = { x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w };
            unsigned       code[2] = { 0u, 0u };  // of the first and the last four values
            unsigned short scale;
            float          own = 0.0f;  // NaN if a value is
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                own = max_nan(own, fabsf(v[e]));
            }
            if (four) {
                // the largest magnitude (NaN if there is one), then the sign of the first value that has it
                float top = max_nan(own, __shfl_xor_sync(0xffffffffu, own, 1));
                top       = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
                float mine = 0.0f;
#pragma unroll
                for (int e = 7; e >= 0; --e) {
                    mine = fabsf(v[e]) == top ? v[e] : mine;
                }
                const unsigned shift = threadIdx.x & 28;
                const unsigned have  = __ballot_sync(0xffffffffu, own == top) >> shift & 0xfu;
                const unsigned minus = __ballot_sync(0xffffffffu, mine < 0.0f) >> shift & 0xfu;
                const float    d     = __fmul_rn((have & (0u - have)) & minus ? -top : top, -0.125f);
                const float    id    = d != 0.0f ? __frcp_rn(d) : 0.0f;
                // floor(x / d + 8.5) in 0 .. 15: added to 2^23 rounding down, it is in the low bits (NaN, from 0 * inf, gives 0)
                unsigned n[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = __fadd_rn(__fmul_rn(v[e], id), 8.5f);
                    n[e]          = __float_as_uint(__fadd_rd(fminf(fmaxf(f, 0.0f), 15.5f), 8388608.0f));
                }
                code[0] = n[0] + 16u * n[1] + 256u * n[2] + 4096u * n[3];  // 16 bits; 2^23's own lie above
                code[1] = n[4] + 16u * n[5] + 256u * n[6] + 4096u * n[7];
                scale   = !(top <= 3.40282347e38f) ? 0x7e00u : __half_as_ushort(__float2half_rn(d));
            } else {
                const float top = block_amax<4, 8>(v, part);
                const float d   = __fmul_rn(top, 0.00787401574803149606f);  // RN(1/127): the header's definition
                const float id  = d != 0.0f ? __frcp_rn(d) : 0.0f;
                // own > top: a value before the block's last NaN, which the fold of magnitudes leaves out
                if (__all_sync(0xffffffffu, top >= 1e-30f && top <= 1e30f && own <= top)) {
                    // |x / d| <= 127.5: round(|x / d|) cut to whole numbers on top of 2^23; sums cut off, not
                    // rounded, so that 0.49999997 + 0.5 stays below 1
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float    f = __fmul_rn(v[e], id);
                        const unsigned n = __float_as_uint(__fadd_rz(__fadd_rz(fabsf(f), 0.5f), 8388608.0f));
                        code[e >> 2] |= ((f < 0.0f ? 0u - n : n) & 0xffu) << (8 * (e & 3));
                    }
                } else {  // zeros, tiny and huge blocks, and what is not finite
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        code[e >> 2] |= (unsigned) (uint8_t) (int8_t) quant_code<B200Q8_QUANT_REF>(v[e], id) << (8 * (e & 3));
                    }
                }
                scale = isnan(d) ? 0x7e00u : __half_as_ushort(__float2half_rn(d));
            }
            if (token < w.tokens) {
                const size_t cell = (size_t) kv_cell(a.c, r.pos + token);
                uint8_t *    to   = codes + cell * row_bytes;
                if (four && t == 0) {
                    *reinterpret_cast<unsigned *>(to) = prmt(code[0], code[1], 0x5410u);
                } else if (four) {
                    *reinterpret_cast<unsigned short *>(to)         = (unsigned short) code[0];
                    *reinterpret_cast<unsigned short *>(to + apart) = (unsigned short) code[1];
                } else if (t == 0) {
                    *reinterpret_cast<uint2 *>(to) = make_uint2(code[0], code[1]);
                } else {
                    *reinterpret_cast<unsigned *>(to)         = code[0];
                    *reinterpret_cast<unsigned *>(to + apart) = code[1];
                }
                if (part == 0) {
                    scales[cell * a.c.nb] = scale;
                }
            }
        }
    }
}

// The same work the other way; a bad run's rows are zeroed, which may be more
// than max_len of them.
template <int kAhead>
__global__ void __launch_bounds__(kRowThreads) kv_read_kernel(const KvRowsArgs a, const int per_cta) {
    pdl_launch_dependents();
    pdl_wait_primary();
    const int   t = blockIdx.y;
    const KvRun r = kv_run(a.b, a.c, blockIdx.z);
    const int   es = a.type == kSrcF32 ? 4 : 2;
    if (!r.ok) {
        if (blockIdx.x == 0 && t == 0 && threadIdx.x == 0) {
            kv_report();
        }
        const int quads = a.c.n_kv * a.c.nb * 8;
        for (int m = blockIdx.x; m < r.len; m += gridDim.x) {
            for (int i = threadIdx.x; i < quads; i += kRowThreads) {
                store4(static_cast<uint8_t *>(a.dst[t]) + (size_t) (r.row + m) * a.stride[t] + (size_t) (4 * i) * es,
                       a.type, a.wide, make_float4(0.f, 0.f, 0.f, 0.f));
            }
        }
        return;
    }
    const int       part = threadIdx.x & 7;
    const RowsWork  w    = rows_work<8>(a, r, per_cta);
    const bool      four = a.c.four[t] != 0;
    const size_t    row_bytes = (size_t) (a.c.nb * (four ? 16 : 32));
    uint8_t *       dst = static_cast<uint8_t *>(a.dst[t]) + (size_t) r.row * a.stride[t] + (size_t) (w.unit * 32 + part * 4) * es;
    const uint8_t * codes = a.c.codes[t] + w.plane * row_bytes + kv_code_offset(t, four, a.c.nb, w.block, part);
    const __half *  scales = a.c.scales[t] + w.plane * a.c.nb + w.block;
    for (int first = w.token; first < w.tokens; first += kAhead * w.step) {
        unsigned code[kAhead];
        float    d[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int    token = first + k * w.step;
            const size_t cell  = token < w.tokens ? (size_t) kv_cell(a.c, r.pos + token) : 0;
            code[k] = 0;
            d[k]    = 0.0f;
            if (token < w.tokens) {
                code[k] = four ? *reinterpret_cast<const unsigned short *>(codes + cell * row_bytes)
                               : *reinterpret_cast<const unsigned *>(codes + cell * row_bytes);
                d[k]    = __half2float(scales[cell * a.c.nb]);
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int      token = first + k * w.step;
            const unsigned c     = code[k];
            float4         x;
            if (four) {
                x = make_float4((float) ((int) (c & 15u) - 8), (float) ((int) (c >> 4 & 15u) - 8),
                                (float) ((int) (c >> 8 & 15u) - 8), (float) ((int) (c >> 12) - 8));
            } else {
                x = make_float4((float) (int8_t) c, (float) (int8_t) (c >> 8), (float) (int8_t) (c >> 16),
                                (float) (int8_t) (c >> 24));
            }
            x = make_float4(x.x * d[k], x.y * d[k], x.z * d[k], x.w * d[k]);
            if (token < w.tokens) {
                store4(dst + (size_t) token * a.stride[t], a.type, a.wide, x);
            }
        }
    }
}

// Tokens a CTA takes: enough for its loads to overlap, few when the call is
// small (a step's single rows: one at a time).
int side_by_side(const KvRowsArgs & a, int groups) {
    return std::max(1, groups / (a.c.n_kv * a.c.nb));
}

bool few_rows(const KvRowsArgs & a, int groups) {
    return a.b.max_len <= 2 * side_by_side(a, groups);
}

int rows_per_cta(const KvRowsArgs & a, int groups) {
    const int side = side_by_side(a, groups);
    return side * (few_rows(a, groups) ? 1 : a.b.max_len <= 64 * side ? 4 : 8);
}

dim3 rows_grid(const KvRowsArgs & a, int groups, int per_cta) {
    const int chunks = (a.c.n_kv * a.c.nb + groups - 1) / groups;
    return dim3((unsigned) ((a.b.max_len + per_cta - 1) / per_cta * chunks), 2, (unsigned) a.b.n_seqs);
}

// Programmatic dependent launch: the kernel may start while the one before it
// in the stream ends; it touches memory after griddepcontrol.wait.
template <typename F>
cudaError_t launch_rows(F fn, const KvRowsArgs & a, int groups, cudaStream_t stream) {
    const int          per_cta = rows_per_cta(a, groups);
    cudaLaunchConfig_t cfg     = {};
    cfg.gridDim                = rows_grid(a, groups, per_cta);
    cfg.blockDim               = dim3(kRowThreads);
    cfg.stream                 = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs                                          = attr;
    cfg.numAttrs                                       = 1;
    return cudaLaunchKernelEx(&cfg, fn, a, per_cta);
}

}  // namespace

cudaError_t launch_kv_write(const KvRowsArgs & a, cudaStream_t stream) {
    constexpr int kGroups = kRowThreads / 4;
    return launch_rows(few_rows(a, kGroups) ? kv_write_kernel<1> : kv_write_kernel<4>, a, kGroups, stream);
}

cudaError_t launch_kv_read(const KvRowsArgs & a, cudaStream_t stream) {
    constexpr int kGroups = kRowThreads / 8;
    return launch_rows(few_rows(a, kGroups) ? kv_read_kernel<1> : kv_read_kernel<4>, a, kGroups, stream);
}

}  // namespace b200q8
