// kv_attend_many.cu -- attention over the quantised cache for prompts: 128
// query rows a CTA on the 5th-generation tensor cores (tcgen05, TMEM).
//
// Both products of a prompt are matrix-matrix products, so here the cache is
// turned into fp16 operands once per 128 rows instead of once per warp.  Keys
// and values (code * scale: 19 bits or fewer) are an fp16 value plus the fp16
// value of what that leaves over, exactly; so are q and the weights, to 22
// bits: a product is hi*hi + hi*lo + lo*hi, good to 2^-21.  With PARTS = 1
// (bf16 rows) q is one fp16 value, which holds its 8 bits.  Weights have both
// parts for every type: with one, a tenth of the results of bf16 prompts were
// rounded the other way, and a row's bits went by its call's length.  Key
// scales of a tile and value scales of a group of tiles are first multiplied by
// a power of two that follows the largest, so that fp16's range costs no bits
// to scales down to 2^-15 of the largest of their 64 cells; below, a value
// scale is held to 2^-26 of it (a key's to 2^-32).
//
// Roles of the 16 warps, handing over through mbarriers: one warp fetches
// 64-cell tiles of the cache by bulk copies and looks for what is seen of them
// and their largest scales; six warps write them to shared
// memory as operands (keys as they lie, values transposed, both in the
// 128-byte swizzle); one thread issues the MMAs S = Q K^T and O += P V,
// whichever is ready, Q and P from TMEM; eight warps hold two threads a row,
// which read S, form the weights and write them over it as P.  O accumulates
// in TMEM over a group of kFoldTiles tiles with one reference for the weights,
// then it is added to fp32 sums in registers (the tensor cores' sums lose a
// bit now and then, and a moved reference would mean rescaling TMEM); a group
// is cut short where a weight would pass 2^15.  S and O have two buffers each,
// operand tiles up to three: copies, conversion, MMAs and weights of
// neighbouring tiles overlap.
//
// A 4096-token prompt over 4-bit caches, 16 heads of 128 in F32: 271 us (254
// TFLOP/s of attention, which take three times as many fp16 ones; on mma.sync
// 797 us).  Ragged bf16 prompts (5761 rows after up to 901, Q8_0): 257 us, with
// weights of one part 244.  What bounds it is the chain of a tile: it takes the row warps
// about 2300 cycles, the code warps 1900 and the tensor cores 1536.
#include "kv_attend.cuh"

namespace b200q8 {
namespace {

constexpr int kManyRows    = 128;
constexpr int kManyCells   = 64;   // a tile
constexpr int kRowWarps    = 8;
constexpr int kCodeWarps   = 6;
constexpr int kMmaWarp = kRowWarps + kCodeWarps, kCopyWarp = kMmaWarp + 1;
constexpr int kManyThreads = 32 * (kCopyWarp + 1);
constexpr int kFoldTiles   = 2;
constexpr int kManyHeader  = 1280;
constexpr int kGrowth      = 15;   // weights are at most 2^kGrowth ...
constexpr int kStart       = 10;   // ... and 2^kStart where a group begins

// TMEM columns: two buffers of S, over which both parts of P are written; Q's parts; two buffers of O
constexpr uint32_t kColS = 0, kColQ = 128, kColO = 256, kTmemCols = 512;

__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {  // K-major rows of 128 bytes, 8-row atoms
    return (uint64_t) ((saddr >> 4) & 0x3fffu) | (uint64_t) 1u << 16 | (uint64_t) (1024u >> 4) << 32 |
           (uint64_t) 1u << 46 | (uint64_t) 2u << 61;
}

// f16 x f16 -> f32, both K-major, M = 128
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n) {
    return (1u << 4) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (128 >> 4) << 24);
}

// d (+)= a * b, a in TMEM: two fp16 a column
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    const uint32_t z = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%4, %4, %4, %4}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(z), "r"(add)
        : "memory");
}

__device__ __forceinline__ void tc_commit(uint64_t * bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

__device__ __forceinline__ void tc_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tc_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 columns of this warp's TMEM lanes (a row a thread).
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t (&v)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t (&v)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// Named barrier of n threads; whether any of them brought true.
__device__ __forceinline__ bool bar_any(int id, int n, bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(id), "r"(n), "r"((uint32_t) mine)
        : "memory");
    return any != 0;
}

__device__ __forceinline__ void fence_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ float pow2(int e) {  // |e| <= 126
    return __uint_as_float((uint32_t) (127 + e) << 23);
}

// Which of 32 cells from c0 on a row sees that sees positions (low, pos] and the sinks.
__device__ __forceinline__ uint32_t seen_bits(const AttendTile & t, int c0, int pos, int low) {
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };  // bits 0 .. n - 1
    const int p0 = t.position(c0), p1 = t.position(c0 + 31);
    // one run of positions (a ring's newest lap may begin right behind the sinks)
    const bool one_kind = t.ring == 1u << 30 || c0 >= t.sinks || c0 + 31 < t.sinks;
    if (one_kind && p1 != kNever && p1 - p0 == 31) {
        return below(pos - p0 + 1) & (~below(low - p0 + 1) | below(t.sinks - p0));
    }
    uint32_t bits = 0u;
#pragma unroll 1
    for (int j = 0; j < 32; ++j) {
        const int p = t.position(c0 + j);
        bits |= (uint32_t) (p <= pos && (p > low || p < t.sinks)) << j;
    }
    return bits;
}

// One look at a phase, suspended for up to about ns.
__device__ __forceinline__ void mbar_try_wait_for(uint64_t * bar, uint32_t parity, uint32_t ns) {
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1, %2;\n\t}" ::"r"(smem_addr(bar)),
                 "r"(parity), "r"(ns)
                 : "memory");
}

template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

constexpr int kMaxKv = 3;  // operand tiles
constexpr int kScans = 8;  // tiles ahead of the rows' that may be looked at: stages + operand tiles + 1 are less

struct ManyHeader {
    uint64_t raw_full[4], raw_free[4];
    uint64_t k_full[kMaxKv], v_full[kMaxKv];  // operand tiles written
    uint64_t kv_free[kMaxKv];                 // the tile's second product is done (operands and P may be rewritten)
    uint64_t s_full[2], p_full[2];
    uint64_t o_free[2];                       // a group's sums have been read
    uint64_t done;                            // every MMA issued has completed
    uint32_t tmem;
    int      stop;
    int      new_group[2];                    // tile begins a group
    // what was found out about a tile: powers of two on its key and value scales; every row sees every cell;
    // a seen value scale is not finite, and whose blocks; cells some row sees
    uint64_t scan_full[kScans];
    int      k_exp[kScans], v_exp[kScans], all[kScans], odd[kScans];
    uint32_t seen[kScans][2];
    uint8_t  bad[kScans][kManyCells];
};
static_assert(sizeof(ManyHeader) <= kManyHeader, "header");

template <int NB>
struct ManyLayout {
    static constexpr int kAtoms  = NB / 2;                 // 64 values (128 bytes) of a row
    static constexpr int kKAtom  = kManyCells * 128;
    static constexpr int kKBytes = 2 * kAtoms * kKAtom;
    static constexpr int kVPart  = NB * 32 * 128;          // a row of 64 cells a value
    static constexpr int kTile   = kKBytes + 2 * kVPart;
    static constexpr int kQRow   = NB * 64 + 16;           // a row of q on its way to TMEM
};

template <int NB, bool K4, bool V4>
struct ManyShape {
    static constexpr int kRaw    = kManyCells * NB * ((K4 ? 16 : 32) + (V4 ? 16 : 32) + 4);
    static constexpr int kSmem   = 227 * 1024;
    static constexpr int kPair   = 4 * kManyRows;  // exchange between a row's two threads
    static constexpr int kKv     = 3 * ManyLayout<NB>::kTile + 2 * kRaw + kPair + kManyHeader <= kSmem ? 3 : 2;
    static constexpr int kStages = kKv * ManyLayout<NB>::kTile + 3 * kRaw + kPair + kManyHeader <= kSmem ? 3 : 2;
    static constexpr int kBytes  = kKv * ManyLayout<NB>::kTile + kStages * kRaw + kPair + kManyHeader;
    static_assert(kBytes <= kSmem && kManyRows * (128 * NB + 16) <= kKv * ManyLayout<NB>::kTile && 2 * kManyRows * ManyLayout<NB>::kQRow <= kKv * ManyLayout<NB>::kTile, "shared memory");
};

template <int NB, bool K4, bool V4, int PARTS>
__global__ void __launch_bounds__(kManyThreads, 1) kv_attend_many_kernel(const KvAttendArgs a) {
    using L               = ManyLayout<NB>;
    using Shape           = ManyShape<NB, K4, V4>;
    constexpr int hd      = 32 * NB;
    constexpr int krow    = (K4 ? 16 : 32) * NB, vrow = (V4 ? 16 : 32) * NB, drow = 2 * NB;
    constexpr int kRawV   = kManyCells * krow, kRawKd = kRawV + kManyCells * vrow, kRawVd = kRawKd + kManyCells * drow;
    constexpr int kRaw = Shape::kRaw, kStages = Shape::kStages, kKv = Shape::kKv;
    constexpr int kCols   = hd / 2;  // O columns a thread
    extern __shared__ __align__(1024) uint8_t many_smem[];
    uint8_t * const    smem = many_smem;
    uint8_t * const    raw  = smem + kKv * L::kTile;
    int * const        pair = reinterpret_cast<int *>(raw + kStages * kRaw);
    ManyHeader * const h    = reinterpret_cast<ManyHeader *>(pair + kManyRows);
    const int          warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_wait_primary();
    if ((smem_addr(smem) & 1023u) != 0u) {  // the swizzle's atoms need it
        if (threadIdx.x == 0) {
            kv_report(B200Q8_ERR_INTERNAL);
        }
        return;
    }
    AttendTile t;
    // blocks: the last tile of rows (it sees most) of every kv head first
    if (!attend_tile(a, NB, kManyRows, (int) gridDim.x / a.c.n_kv - 1 - (int) blockIdx.x / a.c.n_kv,
                     (int) blockIdx.x % a.c.n_kv, kManyCells, 0, 1, t)) {
        return;
    }
    const int mine = t.mine;
    const int pos_lo = t.r.pos + t.row / a.group, pos_hi = t.r.pos + t.last / a.group;
    const int low_lo = a.window ? pos_lo - a.window : -1, low_hi = a.window ? pos_hi - a.window : -1;
    const int es = a.type == kSrcF32 ? 4 : 2;

    auto copy = [&](int i) {  // tile i into its stage, by one thread
        uint8_t *    to   = raw + i % kStages * kRaw;
        uint64_t *   bar  = &h->raw_full[i % kStages];
        const size_t cell = (size_t) t.cell(i);
        mbar_arrive_expect_tx(bar, kRaw);
        bulk_copy_g2s(to, t.kc + cell * krow, kManyCells * krow, bar);
        bulk_copy_g2s(to + kRawKd, t.kd + cell * drow, kManyCells * drow, bar);
        bulk_copy_g2s(to + kRawV, t.vc + cell * vrow, kManyCells * vrow, bar);
        bulk_copy_g2s(to + kRawVd, t.vd + cell * drow, kManyCells * drow, bar);
    };
    if (threadIdx.x == 32 * kCopyWarp) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&h->raw_full[i], 1);
            mbar_init(&h->raw_free[i], kCodeWarps);
        }
        for (int i = 0; i < kScans; ++i) {
            mbar_init(&h->scan_full[i], 1);
        }
        for (int i = 0; i < kKv; ++i) {
            mbar_init(&h->k_full[i], kCodeWarps);
            mbar_init(&h->v_full[i], kCodeWarps);
            mbar_init(&h->kv_free[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&h->s_full[i], 1);
            mbar_init(&h->p_full[i], kRowWarps);
            mbar_init(&h->o_free[i], kRowWarps);
        }
        mbar_init(&h->done, 1);
        h->stop = 0;
        fence_mbar_init();
        for (int i = 0; i < min(mine, kStages); ++i) {
            copy(i);
        }
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&h->tmem)),
                     "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    // ---- q as operands: row-wise scaled, in the order of values that the key operands have; by way of
    // shared memory (the operand tiles' place) to TMEM
    if (warp < kRowWarps) {
        constexpr int kPer = hd / 4, kSide = 32 / kPer;  // lanes a row, rows at a time
        const int     part = lane % kPer;                // values 4 * part .. + 3
        constexpr int kMine = kManyRows / kRowWarps / kSide;  // rounds; all rows are asked for before one is used
        uint4         raws[kMine];
        const int     row0  = t.row + warp * (kManyRows / kRowWarps) + lane / kPer;
        int           token = row0 / a.group, head = row0 % a.group;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const uint8_t * src = static_cast<const uint8_t *>(a.q) + (size_t) (t.r.row + token) * a.q_stride +
                                  (size_t) ((t.kvh * a.group + head) * hd + 4 * part) * es;
            raws[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row0 + i * kSide < t.n_rows) {
                raws[i] = load4_raw(src, es, a.wide);
            }
            for (head += kSide; head >= a.group; head -= a.group) {
                ++token;
            }
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int    in = warp * (kManyRows / kRowWarps) + i * kSide + lane / kPer;
            const float4 x  = widen4(raws[i], a.type);
            float top = max_nan(max_nan(fabsf(x.x), fabsf(x.y)), max_nan(fabsf(x.z), fabsf(x.w)));
#pragma unroll
            for (int off = 1; off < kPer; off <<= 1) {
                top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
            }
            float up, unscale;
            row_scale(top, a.scale, 15, up, unscale);
            if (!(top <= 3.40282347e38f)) {
                up = 0.0f;  // a row that is not finite: all its scores are NaN
                unscale = NAN;
            }
            if (part == 0) {
                pair[in] = __float_as_int(unscale);
            }
            // two words of two values: neighbours (bytes), or k and k + 4 of an octet (nibbles), which
            // takes two values of the lane beside
            float v[4] = { x.x * up, x.y * up, x.z * up, x.w * up };
            if (up == 0.0f) {
                v[0] = v[1] = v[2] = v[3] = 0.0f;
            }
            if (K4) {
                const bool  odd = part & 1;
                const float g0  = __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[2], 1);
                const float g1  = __shfl_xor_sync(0xffffffffu, odd ? v[1] : v[3], 1);
                const float w0 = odd ? g0 : v[0], w1 = odd ? v[2] : g0, w2 = odd ? g1 : v[1], w3 = odd ? v[3] : g1;
                v[0] = w0;
                v[1] = w1;
                v[2] = w2;
                v[3] = w3;
            }
            uint2 hi, lo;
            split_half(v[0], v[1], hi.x, lo.x);
            split_half(v[2], v[3], hi.y, lo.y);
            uint8_t * to = smem + in * L::kQRow + 8 * part;
            *reinterpret_cast<uint2 *>(to) = hi;
            if (PARTS == 2) {
                *reinterpret_cast<uint2 *>(to + kManyRows * L::kQRow) = lo;
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = h->tmem;
    if (warp < kRowWarps && (PARTS == 2 || warp < 4)) {  // warps 0 .. 3 the first parts, 4 .. 7 the second
        const uint8_t * from = smem + (warp >> 2) * kManyRows * L::kQRow + (32 * (warp & 3) + lane) * L::kQRow;
#pragma unroll
        for (int c = 0; c < hd / 2; c += 16) {
            uint32_t v[16];
            load_words<16>(from + 4 * c, v);
            tc_st16(tmem + ((uint32_t) (32 * (warp & 3)) << 16) + kColQ + (uint32_t) ((warp >> 2) * 64 + c), v);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    auto           fail = [&]() {
        kv_report(B200Q8_ERR_DEVICE_TIMEOUT);
        *(volatile int *) &h->stop = 1;
    };
    // a bounded wait; false once it, or any other of the CTA, ran out
    auto wait = [&](uint64_t * bar, uint32_t parity) {
        if (mbar_wait_bounded_or_flag(bar, parity, &h->stop)) {
            return true;
        }
        if (*(volatile int *) &h->stop == 0) {
            fail();
        }
        return false;
    };

    // 16 warps start with 128 registers a thread: 8 * 144 + 8 * 112 = 16 * 128
    if (warp < kRowWarps) {
        more_registers<144>();
        // ---------------------------------------------------------------- weights
        const int      in    = 32 * (warp & 3) + lane, side = warp >> 2;  // row of the tile; which half of the columns
        const int      row   = t.row + in;
        const bool     valid = row < t.n_rows;
        const int      prow = valid ? t.r.pos + row / a.group : -1, lrow = valid && a.window ? prow - a.window : -1;
        const uint32_t lanes = tmem + ((uint32_t) (32 * (warp & 3)) << 16);
        const float    unscale = __int_as_float(pair[in]);
        constexpr int  kBar = 32 * kRowWarps;
        bar_any(2, kBar, false);  // everyone has read its scale: the exchange is free
        float    o[kCols], sum = 0.0f, top = -INFINITY, ref = 0.0f;
        float    o_ref = 0.0f;  // exponent that o is relative to (value power - reference), once something was folded
        int      v_exp = 0, group = 0, tiles = 0;
        uint32_t lost = 0u;     // blocks that a value scale which is not finite spoils
        bool     folded = false, alive = true;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            o[c] = 0.0f;
        }
        // group n, which ended with tile last, into the plain sums; its sums are relative to at
        auto fold = [&](int n, int last, float at) {
            const bool ok = wait(&h->kv_free[last % kKv], (uint32_t) (last / kKv & 1));
            if (bar_any(2, kBar, !ok)) {
                return false;
            }
            tc_after();
            const float f = folded ? exp2_approx(fminf(at - o_ref, 126.0f)) : 0.0f;  // (no cells yet: 0 times it)
#pragma unroll
            for (int c = 0; c < kCols; c += 32) {
                uint32_t v[32];
                tc_ld32(lanes + kColO + (uint32_t) ((n & 1) * 128 + side * kCols + c), v);
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    o[c + k] = fmaf(o[c + k], f, __uint_as_float(v[k]));
                }
            }
            tc_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&h->o_free[n & 1]);
            }
            o_ref  = at;
            folded = true;
            return true;
        };
        for (int i = 0; i < mine; ++i) {
            const int  b = i & 1, kb = i % kKv, sc = i % kScans;
            const bool ok = wait(&h->k_full[kb], (uint32_t) (i / kKv & 1)) && wait(&h->s_full[b], (uint32_t) (i >> 1 & 1));
            tc_after();
            uint32_t s[32];
            tc_ld32(lanes + kColS + (uint32_t) (b * 64 + side * 32), s);
            tc_before();
            const float f = max_nan(unscale * pow2(-h->k_exp[sc]), 1.17549435e-38f);  // not 0: -inf stays -inf
            const bool odd = h->odd[sc] != 0;
            if (!h->all[sc] || odd) {
                const uint32_t seen = seen_bits(t, t.cell(i) + 32 * side, prow, lrow);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    s[j] = seen >> j & 1u ? s[j] : 0xff800000u;
                }
                if (odd) {
                    for (int j = 0; j < 32; ++j) {
                        lost |= seen >> j & 1u ? h->bad[sc][32 * side + j] : 0u;
                    }
                }
            }
            float m = __uint_as_float(s[0]);
#pragma unroll
            for (int j = 1; j < 32; ++j) {
                m = fmaxf(m, __uint_as_float(s[j]));
            }
            m *= f;
            // a group begins: at its time, where a weight would grow too large, where a row sees its
            // first cells, where the values' power of two changes
            const int  v_now = h->v_exp[sc];
            // (once all are here, everyone has read S, and P may go over it)
            const bool vote = bar_any(2, kBar, !ok || (valid && (m > ref + (float) kGrowth || (top == -INFINITY && m > -INFINITY))));
            if (vote && bar_any(2, kBar, !ok)) {
                alive = false;
                break;
            }
            const bool begin = vote || i == 0 || tiles == kFoldTiles || v_now != v_exp;
            const float at = (float) v_exp - ref;
            if (begin) {
                // the row's largest score of this tile, over both threads
                if (side) {
                    pair[in] = __float_as_int(m);
                }
                bar_any(2, kBar, false);
                if (!side) {
                    top         = fmaxf(top, fmaxf(m, __int_as_float(pair[in])));
                    pair[in] = __float_as_int(top);
                }
                bar_any(2, kBar, false);
                top             = __int_as_float(pair[in]);
                const float now = top == -INFINITY ? 0.0f : top - (float) kStart;
                sum *= i == 0 ? 0.0f : exp2_approx(fminf(ref - now, 126.0f));
                ref   = now;
                v_exp = v_now;
                tiles = 0;
            }
            ++tiles;
            uint32_t hi[16], lo[16];
            float    add = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float p0 = exp2_approx(fmaf(__uint_as_float(s[j]), f, -ref));
                const float p1 = exp2_approx(fmaf(__uint_as_float(s[j + 1]), f, -ref));
                add += p0 + p1;
                split_half(p0, p1, hi[j / 2], lo[j / 2]);
            }
            sum += add;
            tc_after();
            const uint32_t pa = lanes + kColS + (uint32_t) (b * 64 + side * 16);
            tc_st16(pa, hi);
            tc_st16(pa + 32, lo);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            if (threadIdx.x == 0) {
                h->new_group[b] = begin;
            }
            tc_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&h->p_full[b]);
            }
            if (begin) {
                if (group > 0 && !fold(group - 1, i - 1, at)) {
                    alive = false;
                    break;
                }
                ++group;
            }
        }
        if (alive) {
            alive = fold(group - 1, mine - 1, (float) v_exp - ref);
        }
        // ---- both threads' sums of weights, and the row
        if (alive) {
            if (side) {
                pair[in] = __float_as_int(sum);
            }
            bar_any(2, kBar, false);
            if (!side) {
                sum += __int_as_float(pair[in]);
                pair[in] = __float_as_int(sum);
            }
            bar_any(2, kBar, false);
            sum = __int_as_float(pair[in]);
            if (bar_any(2, kBar, lost != 0u)) {
                pair[in] = 0;
                bar_any(2, kBar, false);
                atomicOr(&pair[in], (int) lost);
                bar_any(2, kBar, false);
                lost = (uint32_t) pair[in];
            }
            // by way of shared memory (no product or copy is left), so that a row is written by lanes side by side
            constexpr int kRow = 4 * hd + 16;
            const float   f    = sum != 0.0f ? pow2(-v_exp) / sum : 0.0f;
            uint8_t *     to   = smem + in * kRow + 4 * side * kCols;
#pragma unroll
            for (int c = 0; c < kCols; c += 4) {
                float4 v = make_float4(o[c] * f, o[c + 1] * f, o[c + 2] * f, o[c + 3] * f);
                if (lost >> ((side * kCols + c) >> 5) & 1u) {
                    v = make_float4(NAN, NAN, NAN, NAN);
                }
                *reinterpret_cast<float4 *>(to + 4 * c) = v;
            }
            bar_any(2, kBar, false);
            constexpr int kPer = hd / 4, kSide = 32 / kPer;
            const int row0  = t.row + warp * (kManyRows / kRowWarps) + lane / kPer;
            int       token = row0 / a.group, head = row0 % a.group;
#pragma unroll 4
            for (int i = 0; i < kManyRows / kRowWarps; i += kSide) {
                if (row0 + i < t.n_rows) {
                    uint8_t * dst = static_cast<uint8_t *>(a.out) + (size_t) (t.r.row + token) * a.out_stride +
                                    (size_t) ((t.kvh * a.group + head) * hd + 4 * (lane % kPer)) * es;
                    store4(dst, a.type, a.wide,
                           *reinterpret_cast<const float4 *>(smem + (row0 - t.row + i) * kRow + 16 * (lane % kPer)));
                }
                for (head += kSide; head >= a.group; head -= a.group) {
                    ++token;
                }
            }
        }
    } else {
        fewer_registers<112>();
        if (warp == kCopyWarp) {
            // -------------------------------------- copies, and a look at each tile
            int  v_exp = 0, i = 0, copied = min(mine, kStages);
            bool v_set = false;
            for (; i < mine; ++i) {
                const int s = i % kStages, sc = i % kScans;
                if (!__all_sync(0xffffffffu, wait(&h->raw_full[s], (uint32_t) (i / kStages & 1)))) {
                    break;
                }
                // what is seen of two cells a lane, and the largest scales of that
                const uint8_t * r = raw + s * kRaw;
                uint32_t        seen[2], ktop = 0u, vtop = 0u;
                bool            all = true, odd = false;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int  cell = 32 * x + lane;
                    const int  p    = t.position(t.cell(i) + cell);
                    const bool sink = p < t.sinks;
                    const bool any  = p <= pos_hi && (p > low_lo || sink);
                    all             = all && p <= pos_lo && (p > low_hi || sink);
                    seen[x]         = __ballot_sync(0xffffffffu, any);
                    uint32_t kd[NB / 2], vd[NB / 2], bad = 0u;
                    load_words<NB / 2>(r + kRawKd + cell * drow, kd);
                    load_words<NB / 2>(r + kRawVd + cell * drow, vd);
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        const uint32_t k = (n & 1 ? kd[n / 2] >> 16 : kd[n / 2]) & 0x7fffu;
                        const uint32_t v = (n & 1 ? vd[n / 2] >> 16 : vd[n / 2]) & 0x7fffu;
                        ktop             = max(ktop, any && k < 0x7c00u ? k : 0u);
                        vtop             = max(vtop, any && v < 0x7c00u ? v : 0u);
                        bad |= (uint32_t) (any && v >= 0x7c00u) << n;
                    }
                    h->bad[sc][cell] = (uint8_t) bad;
                    odd              = odd || bad != 0u;
                }
                ktop = __reduce_max_sync(0xffffffffu, ktop);
                vtop = __reduce_max_sync(0xffffffffu, vtop);
                all  = __all_sync(0xffffffffu, all);
                odd  = __any_sync(0xffffffffu, odd);
                // largest key operand below 2^15; a tile's values lie up to 2^6 below that, and a new
                // power (which begins a group: a fold) is taken only where they would not
                const int kmax = ktop ? (int) (__float_as_uint(half_float((unsigned short) ktop)) >> 23) - 127 : 0;
                const int vmax = vtop ? (int) (__float_as_uint(half_float((unsigned short) vtop)) >> 23) - 127 : -100;
                constexpr int kHigh = V4 ? 11 : 7;  // scale below 2^(kHigh + 1), code up to 8 or 127
                if (vtop != 0u && (!v_set || vmax + v_exp > kHigh || vmax + v_exp < kHigh - 6)) {
                    v_exp = kHigh - 3 - vmax;
                    v_set = true;
                }
                __syncwarp();
                if (lane == 0) {
                    h->k_exp[sc]   = min(30, (K4 ? 11 : 7) - kmax);  // (2^15 twice is what fp16 can multiply by)
                    h->v_exp[sc]   = v_exp;
                    h->all[sc]     = all;
                    h->odd[sc]     = odd;
                    h->seen[sc][0] = seen[0];
                    h->seen[sc][1] = seen[1];
                    mbar_arrive(&h->scan_full[sc]);
                }
                // the next tile to look at, if it is not on its way yet
                if (copied < mine && copied == i + 1) {
                    if (!__all_sync(0xffffffffu, wait(&h->raw_free[copied % kStages], (uint32_t) ((copied / kStages - 1) & 1)))) {
                        break;
                    }
                    if (lane == 0) {
                        copy(copied);
                    }
                    ++copied;
                }
            }
            // what is in flight lands before the CTA leaves
            for (int k = max(0, copied - kStages); k < copied; ++k) {
                (void) mbar_wait_bounded(&h->raw_full[k % kStages], (uint32_t) (k / kStages & 1));
            }
        } else if (warp == kMmaWarp) {
            // ------------------------------------------------------------------ MMAs
            if (lane == 0) {
                const uint32_t kv0   = smem_addr(smem);
                int            group = 0;           // groups begun
                int            first = 0, second = 0;  // products issued
                bool           ok    = true;
                long long      since = clock64();
                while (second < mine && ok) {
                    // S = Q K^T of the next tile, once its keys are there and its S buffer's P is used
                    if (first < mine && first < second + 2 && mbar_test_wait(&h->k_full[first % kKv], (uint32_t) (first / kKv & 1)) &&
                        (first < 2 || mbar_test_wait(&h->kv_free[(first - 2) % kKv], (uint32_t) ((first - 2) / kKv & 1)))) {
                        tc_after();
                        const uint32_t s = tmem + kColS + (uint32_t) ((first & 1) * 64), k0 = kv0 + first % kKv * L::kTile;
                        uint32_t       add = 0u;
#pragma unroll
                        for (int x = 2 - PARTS; x < 3; ++x) {  // lo*hi, hi*lo, hi*hi
                            const uint32_t qa = tmem + kColQ + (x == 0 ? 64u : 0u);
                            const uint32_t ka = k0 + (x == 1 ? (uint32_t) (L::kAtoms * L::kKAtom) : 0u);
#pragma unroll
                            for (int k = 0; k < hd / 16; ++k) {
                                tc_mma_ts(s, qa + 8 * k, desc_sw128(ka + (k >> 2) * L::kKAtom + 32 * (k & 3)),
                                          idesc_f16(kManyCells), add);
                                add = 1u;
                            }
                        }
                        tc_commit(&h->s_full[first & 1]);
                        ++first;
                        since = clock64();
                        continue;
                    }
                    // O += P V of the tile whose weights are ready
                    const int b = second & 1, kvb = second % kKv;
                    if (second < first && mbar_test_wait(&h->p_full[b], (uint32_t) (second >> 1 & 1)) &&
                        mbar_test_wait(&h->v_full[kvb], (uint32_t) (second / kKv & 1))) {
                        const bool begin = *(volatile int *) &h->new_group[b] != 0;
                        if (begin) {
                            if (group >= 2 && !wait(&h->o_free[group & 1], (uint32_t) ((group / 2 - 1) & 1))) {
                                ok = false;
                                break;
                            }
                            ++group;
                        }
                        tc_after();
                        const uint32_t o = tmem + kColO + (uint32_t) (((group - 1) & 1) * 128);
                        const uint32_t pc = tmem + kColS + (uint32_t) (b * 64), v = kv0 + kvb * L::kTile + L::kKBytes;
                        uint32_t       add = begin ? 0u : 1u;
#pragma unroll
                        for (int x = 0; x < 3; ++x) {
                            const uint32_t pa = pc + (x == 0 ? 32u : 0u);
                            const uint32_t va = v + (x == 1 ? (uint32_t) L::kVPart : 0u);
#pragma unroll
                            for (int k = 0; k < kManyCells / 16; ++k) {
                                tc_mma_ts(o, pa + 8 * k, desc_sw128(va + 32 * k), idesc_f16(hd), add);
                                add = 1u;
                            }
                        }
                        tc_commit(&h->kv_free[kvb]);
                        ++second;
                        since = clock64();
                        continue;
                    }
                    // nothing is ready: a short sleep on what comes next leaves the issue slots to the others
                    if (second < first) {
                        mbar_try_wait_for(&h->p_full[b], (uint32_t) (second >> 1 & 1), 200u);
                    } else {
                        mbar_try_wait_for(&h->k_full[first % kKv], (uint32_t) (first / kKv & 1), 200u);
                    }
                    if (*(volatile int *) &h->stop != 0) {
                        ok = false;
                    } else if (clock64() - since > kWaitLimitCycles) {
                        fail();
                        ok = false;
                    }
                }
                // every MMA completes before TMEM and shared memory are given up
                tc_commit(&h->done);
                (void) mbar_wait_bounded(&h->done, 0);
            }
        } else {
            // ------------------------------------------------------- codes to operands
            const int tid = threadIdx.x - 32 * kRowWarps;
            for (int i = 0; i < mine; ++i) {
                const int  s = i % kStages, b = i % kKv, sc = i % kScans;
                const bool ok = wait(&h->scan_full[sc], (uint32_t) (i / kScans & 1)) &&
                                wait(&h->raw_full[s], (uint32_t) (i / kStages & 1)) &&
                                (i < kKv || wait(&h->kv_free[b], (uint32_t) ((i / kKv - 1) & 1)));
                if (!__all_sync(0xffffffffu, ok)) {
                    break;
                }
                const uint8_t * r       = raw + s * kRaw;
                const uint32_t  seen_lo = h->seen[sc][0], seen_hi = h->seen[sc][1];
                const int       k_exp = h->k_exp[sc], v_exp = h->v_exp[sc];
                uint8_t * const kv = smem + b * L::kTile;
                // -- keys: 256 (cell, chunk) pairs, the last 64 by the threads that have no values to do
                {
                    const __half2 ka = __float2half2_rn(pow2(k_exp / 2)), kb = __float2half2_rn(pow2(k_exp - k_exp / 2));
                    const int     cell = tid & 63;
#pragma unroll 1
                    for (int c = tid >> 6; c < 4; c = tid < 64 ? c + 3 : 4) {
                        constexpr int kW = K4 ? 1 : 2;
                        uint32_t      w[NB * kW], d[NB / 2];
                        load_words<NB * kW>(r + cell * krow + c * (krow / 4), w);
                        load_words<NB / 2>(r + kRawKd + cell * drow, d);
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            uint32_t f[4];
                            key_operands<K4>(w[kW * n], w[kW * n + kW - 1], f);
                            const __half2 both = __hmul2(__hmul2(bits_h2(d[n / 2]), ka), kb);
                            const __half2 sc   = n & 1 ? __high2half2(both) : __low2half2(both);
                            uint4         hi, lo;
                            uint32_t *    ph = &hi.x, * pl = &lo.x;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const __half2 x = __hmul2(bits_h2(f[e]), sc);
                                ph[e]           = h2_bits(x);
                                pl[e]           = h2_bits(__hfma2(bits_h2(f[e]), sc, __hneg2(x)));
                            }
                            const int o  = 4 * n + c;
                            uint8_t * to = kv + (o >> 3) * L::kKAtom + cell * 128 + (((o & 7) ^ (cell & 7)) << 4);
                            *reinterpret_cast<uint4 *>(to)                         = hi;
                            *reinterpret_cast<uint4 *>(to + L::kAtoms * L::kKAtom) = lo;
                        }
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&h->k_full[b]);
                }
                // -- values, transposed: eight cells of a lane group's four values of half the blocks
                if (tid >= 64) {
                    constexpr int kN = NB / 2;  // blocks a thread
                    const __half2 va = __float2half2_rn(pow2(v_exp / 2)), vb = __float2half2_rn(pow2(v_exp - v_exp / 2));
                    const int     k8 = tid & 7, g = tid >> 3 & 7, half = (tid >> 6) - 1;
                    uint32_t      w[8][kN], d[8];  // d: scales of the half's blocks, two at a time
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int cell = 8 * k8 + x;
                        const uint8_t * vp = r + kRawV + cell * vrow + g * (vrow / 8) + half * (kN * (V4 ? 2 : 4));
                        const uint8_t * dp = r + kRawVd + cell * drow + half * (2 * kN);
                        const bool seen = (cell < 32 ? seen_lo >> cell : seen_hi >> (cell - 32)) & 1u;
                        if (V4) {
                            const uint32_t both = kN == 2 ? *reinterpret_cast<const uint32_t *>(vp)
                                                          : *reinterpret_cast<const unsigned short *>(vp);
#pragma unroll
                            for (int n = 0; n < kN; ++n) {
                                w[x][n] = both >> (16 * n);
                            }
                        } else {
                            load_words<kN>(vp, w[x]);
                        }
                        uint32_t e = kN == 2 ? *reinterpret_cast<const uint32_t *>(dp) : *reinterpret_cast<const unsigned short *>(dp);
                        // cells no row sees, and scales that are not finite, must not count
                        e = seen ? e : 0u;
                        e = (e & 0x7c00u) == 0x7c00u ? e & 0xffff0000u : e;
                        e = (e & 0x7c000000u) == 0x7c000000u ? e & 0xffffu : e;
                        d[x] = h2_bits(__hmul2(__hmul2(bits_h2(e), va), vb));
                    }
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        uint4 hi[4], lo[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {  // pairs of cells
                            uint32_t f[4];
                            value_operands<V4>(w[2 * y][n], w[2 * y + 1][n], false, f);
                            const __half2 sc = bits_h2(prmt(d[2 * y], d[2 * y + 1], n ? 0x7632u : 0x5410u));
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const __half2 x = __hmul2(bits_h2(f[e]), sc);
                                (&hi[e].x)[y]   = h2_bits(x);
                                (&lo[e].x)[y]   = h2_bits(__hfma2(bits_h2(f[e]), sc, __hneg2(x)));
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int row = 32 * (half * kN + n) + 4 * g + e;
                            uint8_t * to  = kv + L::kKBytes + row * 128 + ((k8 ^ (row & 7)) << 4);
                            *reinterpret_cast<uint4 *>(to)             = hi[e];
                            *reinterpret_cast<uint4 *>(to + L::kVPart) = lo[e];
                        }
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&h->v_full[b]);
                    mbar_arrive(&h->raw_free[s]);
                }
            }
        }
    }
    pdl_launch_dependents();
    tc_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

template <int NB, int PARTS>
KvAttendMany attend_many(int k4, int v4) {
    KvAttendMany m;
    if (k4 && v4) {
        m.fn   = (const void *) kv_attend_many_kernel<NB, true, true, PARTS>;
        m.smem = ManyShape<NB, true, true>::kBytes;
    } else if (k4) {
        m.fn   = (const void *) kv_attend_many_kernel<NB, true, false, PARTS>;
        m.smem = ManyShape<NB, true, false>::kBytes;
    } else if (v4) {
        m.fn   = (const void *) kv_attend_many_kernel<NB, false, true, PARTS>;
        m.smem = ManyShape<NB, false, true>::kBytes;
    } else {
        m.fn   = (const void *) kv_attend_many_kernel<NB, false, false, PARTS>;
        m.smem = ManyShape<NB, false, false>::kBytes;
    }
    m.rows    = kManyRows;
    m.threads = kManyThreads;
    return m;
}

}  // namespace

KvAttendMany kv_attend_many(int nb, int k4, int v4, int type) {
    const bool one = type == kSrcBF16;
    return nb == 2   ? (one ? attend_many<2, 1>(k4, v4) : attend_many<2, 2>(k4, v4))
           : nb == 4 ? (one ? attend_many<4, 1>(k4, v4) : attend_many<4, 2>(k4, v4))
                     : KvAttendMany{};
}

}  // namespace b200q8
