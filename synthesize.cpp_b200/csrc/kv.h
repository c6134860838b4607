// kv.h -- the quantised key/value cache: device-side views and launchers (internal).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace b200q8 {

// A cache as the kernels see it (layout: b200q8_kv_cache in b200q8.h).
struct KvCacheView {
    uint8_t * codes[2];   // keys, values
    __half *  scales[2];
    int       four[2];    // 1: Q4_0, 0: Q8_0
    int       n_slots, n_ctx, n_kv, nb;  // nb: 32-value blocks of a head row
    int       sinks;
    int       ring;       // cells that positions >= sinks go round, 0: no ring
};

// The runs of a call (b200q8_kv_batch).
struct KvRuns {
    const int32_t * starts;
    const int32_t * pos;
    const int32_t * slots;
    int             n_seqs, n_tokens, max_len;
    int             slot_base;  // without slots: run i is slot slot_base + i
};

struct KvRowsArgs {
    KvCacheView  c;
    KvRuns       b;
    const void * src[2];     // write: rows of keys and of values
    void *       dst[2];     // read
    size_t       stride[2];  // bytes between rows
    int          type;       // SrcType
    int          wide;       // rows may be accessed 4 values at a time
};

struct KvAttendArgs {
    KvCacheView  c;
    KvRuns       b;
    const void * q;
    void *       out;
    size_t       q_stride, out_stride;  // bytes between rows
    int          type;                  // SrcType of q and out
    int          n_head, group;         // group = n_head / n_kv
    int          window;                // 0: the whole prefix
    int          wide;                  // rows may be accessed 4 values at a time
    float        scale;
};

cudaError_t launch_kv_write(const KvRowsArgs & a, cudaStream_t stream);
cudaError_t launch_kv_read(const KvRowsArgs & a, cudaStream_t stream);
// The kernel for few query rows (tokens x heads of a kv head): up to kv_attend_few_rows of heads of nb blocks, 4 or
// 8 warps a CTA.
int          kv_attend_few_rows(int nb);
const void * kv_attend_few(int nb, int warps, int k4, int v4);
// The kernel for prompts of heads of nb blocks (fn null: none), its rows a CTA, threads and shared memory.
struct KvAttendMany {
    const void * fn = nullptr;
    int          rows = 0, threads = 0;
    size_t       smem = 0;
};
KvAttendMany kv_attend_many(int nb, int k4, int v4, int type);
// Sets the attributes of the kernel that such a call launches (launches do it too; a capture should not).
cudaError_t  prepare_kv_attend(const KvAttendArgs & a, int sm_count);
cudaError_t  launch_kv_attend(const KvAttendArgs & a, cudaStream_t stream, int sm_count);

// The cache kernels' status word on the current device (their translation unit has one of its own; the first error
// wins), cleared if clear.  Synchronises with nothing but the copy.
cudaError_t kv_device_status(unsigned * word, bool clear);

}  // namespace b200q8
