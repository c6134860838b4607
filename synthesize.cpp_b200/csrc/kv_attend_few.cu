// kv_attend_few.cu -- attention over the quantised cache for few query rows: (tokens x heads of a kv head) x blocks
// of a head <= 8, which is a decode step of the talker (2 heads of 4 blocks).
//
// With 2 rows, two thirds of what a warp does for 8 is thrown away.  Here an
// operand row is a (query row, block) pair: row (h, b) of q's operand holds q
// in block b and zeros elsewhere, so one chain of products over the whole
// head gives every block's sum in a row - a lane - of its own.  A lane scales
// its one block's sums, the blocks are added by shuffles, and each lane then
// forms the weights times its own block's value scales, once, instead of
// every lane doing so for every block.  q is scaled by a power of two to 30
// bits and sign and enters as four signed bytes: the keys' codes are bytes as
// they lie (nibbles: a mask), the sums are exact integers.  (Fixed point: three
// bytes would hold a value 2^10 below the row's largest to 12 bits.)  The
// second product, in fp16, gives row (h, b) the values of all blocks; those of
// block b count.  Rows 8 .. 15 hold the weights' second fp16 parts (of q: the
// third and first bytes).
//
// The reference of the weights moves only when the largest weight times the
// largest value scale of a lane's cells would pass 2^15, or a weight
// kMostWeight (the weights of cells whose values are zero must not overflow
// either).  It is set so that the largest product of both is below 2^8, as far
// as weights stay below 2^-kZero: 7 bits to grow, and a product's fp16 parts
// hold it to 2^-22 of itself or 2^-32 of the largest.  So products add up in
// the tensor cores' accumulators; they are moved to plain fp32 sums every kFold
// steps, because the tensor cores cut their sums off where fp32 addition
// rounds.
//
// 64 streams of 698 to 8100 positions (keys in 8 bits, values in 4; 519 MB):
// 142 us, 3.7 TB/s; its copies alone take 85 us.  It is bound by instructions
// with fixed latencies: a step of 32 cells is about 850, at 2.6 warps a
// scheduler or fewer.  A stream alone (32701 positions, Q4_0): 34 us, because
// its 128 CTAs do not fill the SMs.
#include "kv_attend.cuh"

namespace b200q8 {
namespace {

constexpr int   kFold       = 8;
constexpr float kMostWeight = 1.2379400392853803e27f;  // 2^90: sums over 2^30 cells stay below 2^120
constexpr int   kZero       = -73;     // log2 of what a value scale of zero counts as
constexpr int   kBias       = 0x4b400000;  // an integer sum on top of it is the bits of 1.5 * 2^23 + sum

// REGS: 168 with four warps a CTA (three CTAs an SM), 128 with eight (two, so that a cluster of 16 finds room)
template <int NB, bool EXACT, bool K4, bool V4, int REGS>
__global__ void __maxnreg__(REGS) kv_attend_few_kernel(const KvAttendArgs a, const int n_split, const int n_stages) {
    constexpr int kRows = 8 / NB;  // query rows a CTA
    extern __shared__ __align__(128) uint8_t smem[];
    const AttendShared sh = attend_shared(smem);
    const int nb   = EXACT ? NB : a.c.nb;
    const int hd   = nb * 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
    const int g = lane >> 2, c4 = lane & 3;
    uint64_t * const full = sh.full + warp * kMaxStages;  // each warp has stages of its own
    if (lane == 0) {
        for (int i = 0; i < n_stages; ++i) {
            mbar_init(&full[i], 1);
        }
        fence_mbar_init();
    }
    __syncwarp();
    pdl_wait_primary();
    AttendTile t;
    if (!attend_tile(a, nb, kRows, row_tile(n_split), blockIdx.y, kStep, (int) (blockIdx.x % n_split) * n_warps + warp, n_split * n_warps, t)) {
        return;
    }
    // bytes a cell, and where a stage keeps its arrays (as t has them, but constants)
    const int krow = (K4 ? 16 : 32) * nb, vrow = (V4 ? 16 : 32) * nb, drow = 2 * nb;
    const int off_v = kStep * krow, off_kd = off_v + kStep * vrow, off_vd = off_kd + kStep * drow;
    const int stage_bytes = off_vd + kStep * drow;
    uint8_t * const stages = sh.stages + (size_t) warp * n_stages * stage_bytes;
    // lanes 0 .. 3 copy one of a step's arrays each
    const uint8_t * from     = lane == 0 ? t.kc : lane == 1 ? t.vc : lane == 2 ? t.kd : t.vd;
    const int       from_row = lane == 0 ? krow : lane == 1 ? vrow : drow;
    const int       to       = lane == 0 ? 0 : lane == 1 ? off_v : lane == 2 ? off_kd : off_vd;
    auto            issue    = [&](int i, int stage) {
        if (lane == 0) {
            mbar_arrive_expect_tx(&full[stage], (uint32_t) stage_bytes);
        }
        if (lane < 4) {
            bulk_copy_g2s(stages + stage * stage_bytes + to, from + (size_t) t.cell(i) * from_row,
                          (uint32_t) (kStep * from_row), &full[stage]);
        }
    };
    for (int i = 0; i < min(t.mine, n_stages); ++i) {
        issue(i, i);
    }

    // ---- this lane's operand row: query row t.row + g / NB, block g % NB, as
    // q * 2^x in four signed bytes (30 bits and sign)
    const int  block = g % NB;
    const int  row   = t.row + g / NB;
    const bool valid = row < t.n_rows && block < nb;
    const int  token = row < t.n_rows ? row / a.group : 0;
    const int  es    = a.type == kSrcF32 ? 4 : 2;
    const int  prow = row < t.n_rows ? t.r.pos + token : -1, lrow = a.window ? prow - a.window : -1;
    uint32_t   qhi[NB][4], qlo[NB][4];  // rows g: parts 3 | 1, rows g + 8: parts 2 | 0
    int        chi[4], clo[4];          // what the sums start from
    float      unscale;
    {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
        if (valid) {
            const uint8_t * src = static_cast<const uint8_t *>(a.q) + (size_t) (t.r.row + token) * a.q_stride +
                                  (size_t) ((t.kvh * a.group + row % a.group) * hd + 32 * block + 8 * c4) * es;
            x = load4(src, a.type, a.wide);
            y = load4(src + 4 * es, a.type, a.wide);
        }
        const float q[8] = { x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w };
        float       top  = 0.0f;
        bool        bad  = false;  // not finite
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            top = fmaxf(top, fabsf(q[e]));
            bad = bad || !(fabsf(q[e]) <= 3.40282347e38f);
        }
#pragma unroll
        for (int off = 1; off < 4 * NB; off <<= 1) {  // over the row's lanes: 4 a block
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            bad = __shfl_xor_sync(0xffffffffu, (int) bad, off) != 0 || bad;
        }
        float up;
        row_scale(top, a.scale, 30, up, unscale);
        if (bad) {
            unscale = NAN;  // every score of the row
        }
        uint32_t part[4][2] = {};
        int      total[4]   = {};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // the lane's codes: even and odd nibbles of a word, or two words of bytes
            const int reg = K4 ? e & 1 : e >> 2, byte = K4 ? e >> 1 : e & 3;
            int       v   = bad ? 0 : __float2int_rn(q[e] * up);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int digit = k == 3 ? v : (int) (signed char) (v & 0xff);
                part[k][reg] |= (uint32_t) (digit & 0xff) << (8 * byte);
                total[k] += digit;
                v = (v - digit) >> 8;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            total[k] += __shfl_xor_sync(0xffffffffu, total[k], 1);
            total[k] += __shfl_xor_sync(0xffffffffu, total[k], 2);
        }
        const int off = K4 ? 8 : 0;  // Q4_0 codes are stored as code + 8
        chi[0] = chi[1] = kBias - off * total[3];
        chi[2] = chi[3] = kBias - off * total[2];
        clo[0] = clo[1] = kBias - off * total[1];
        clo[2] = clo[3] = kBias - off * total[0];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            qhi[b][0] = b == block ? part[3][0] : 0u;
            qhi[b][1] = b == block ? part[2][0] : 0u;
            qhi[b][2] = b == block ? part[3][1] : 0u;
            qhi[b][3] = b == block ? part[2][1] : 0u;
            qlo[b][0] = b == block ? part[1][0] : 0u;
            qlo[b][1] = b == block ? part[0][0] : 0u;
            qlo[b][2] = b == block ? part[1][1] : 0u;
            qlo[b][3] = b == block ? part[0][1] : 0u;
        }
    }
    const int pos_lo = t.r.pos + t.row / a.group, pos_hi = t.r.pos + t.last / a.group;
    const int low_lo = a.window ? pos_lo - a.window : -1, low_hi = a.window ? pos_hi - a.window : -1;

    float ref = valid ? -INFINITY : 0.0f, sum = 0.0f;
    float acc[4][4], o[4][2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        o[e][0] = o[e][1] = 0.0f;
        acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.0f;
    }
    auto fold = [&]() {  // both parts to the plain sums
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[e][0] += acc[e][0] + acc[e][2];
            o[e][1] += acc[e][1] + acc[e][3];
            acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.0f;
        }
    };

    int i = 0, stage = 0, phase = 0, done = 0;
    for (; i < t.mine; ++i) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[stage], phase))) {
            break;
        }
        uint8_t * const s  = stages + stage * stage_bytes;
        const int       c0 = t.cell(i);
        // which of the step's cells some row, and every row, sees
        const int      p    = t.position(c0 + lane);
        const bool     sink = p < t.sinks;
        const uint32_t any  = __ballot_sync(0xffffffffu, p <= pos_hi && (p > low_lo || sink));
        const bool     all  = __all_sync(0xffffffffu, p <= pos_lo && (p > low_hi || sink));
        if (any != 0) {
            const uint8_t * sk = s, * sv = s + off_v, * skd = s + off_kd, * svd = s + off_vd;

            // ---- every block's share of the scores of four 8-column tiles, two
            // at a time; scaled and added over the blocks: scores of cells 4x + c
            constexpr int          kW = K4 ? 1 : 2;  // words a block
            const unsigned short * kd = reinterpret_cast<const unsigned short *>(skd) + (EXACT || block < nb ? block : 0);
            const unsigned short * vd = reinterpret_cast<const unsigned short *>(svd) + (EXACT || block < nb ? block : 0);
            float                  sc[8], dv[8];
            unsigned short         vbits[8];
#pragma unroll
            for (int u0 = 0; u0 < 4; u0 += 2) {
                uint32_t w[2][NB * kW];
                int      hi[2][4], lo[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    load_chunk<NB * kW, EXACT>(sk + (8 * (u0 + u) + 4 * (g & 1) + (g >> 1)) * krow + c4 * (krow / 4),
                                               2 * kW * nb, w[u]);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (!EXACT && b >= nb) {
                        break;
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t b0 = K4 ? w[u][b] & 0x0f0f0f0fu : w[u][kW * b];
                        const uint32_t b1 = K4 ? w[u][b] >> 4 & 0x0f0f0f0fu : w[u][kW * b + kW - 1];
                        mma_i8(hi[u], qhi[b], b0, b1, b == 0 ? chi : hi[u]);
                        mma_i8(lo[u], qlo[b], b0, b1, b == 0 ? clo : lo[u]);
                    }
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int   u = y >> 1, j = y & 1, x = 2 * u0 + y;
                    const float s3 = __int_as_float(hi[u][j]) - 12582912.0f, s2 = __int_as_float(hi[u][j + 2]) - 12582912.0f;
                    const float s1 = __int_as_float(lo[u][j]) - 12582912.0f, s0 = __int_as_float(lo[u][j + 2]) - 12582912.0f;
                    float       v  = fmaf(fmaf(s3, 256.0f, s2), 65536.0f, fmaf(s1, 256.0f, s0)) * half_float(kd[(4 * x + c4) * nb]);
                    v              = EXACT || block < nb ? v : 0.0f;
#pragma unroll
                    for (int off = 4; off < 4 * NB; off <<= 1) {
                        v += __shfl_xor_sync(0xffffffffu, v, off);
                    }
                    sc[x]    = fmaf(v, 0.0f, v);  // an infinite scale: values of both signs, so not a number
                    vbits[x] = vd[(4 * x + c4) * nb];
                }
            }
            if (!EXACT && block >= nb) {
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    vbits[x] = 0;
                }
            }
            uint32_t seen = 0xffu;
            if (!all) {
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const int pc = __shfl_sync(0xffffffffu, p, 4 * x + c4);
                    if (!(pc <= prow && (pc > lrow || pc < t.sinks))) {
                        seen &= ~(1u << x);
                        sc[x] = -INFINITY;
                    }
                    if (!(any >> (4 * x + c4) & 1u)) {
                        vbits[x] = 0;  // no row sees the cell: whatever it holds must not count
                    }
                }
            }
            float top = 0.0f;  // largest magnitude of the value scales; NaN if one is
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                dv[x] = half_float(vbits[x]);
                top   = max_nan(top, fabsf(dv[x]));
            }
            // a scale that is not finite: the block of a row that sees it is lost, others must not be
            bool poison = false;
            if (__any_sync(0xffffffffu, !(top <= 65504.0f))) {
                top = 0.0f;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    if (!(fabsf(dv[x]) <= 65504.0f)) {
                        poison = poison || (seen >> x & 1u);
                        dv[x]  = 0.0f;
                    }
                    top = fmaxf(top, fabsf(dv[x]));
                }
            }
            // ---- weights relative to the reference, which moves if they grow too large
            float    pw[8], add = 0.0f, peak = 0.0f;
            uint32_t ah[2][4];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                pw[x] = exp2_approx(fmaf(sc[x], unscale, -ref));
                peak  = fmaxf(peak, pw[x]);
            }
            if (__any_sync(0xffffffffu, valid && (peak * top > 32768.0f || peak > kMostWeight || (ref == -INFINITY && seen)))) {
                float m = -INFINITY;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const int e = max(kZero, (int) (__float_as_uint(fabsf(dv[x])) >> 23) - 127);
                    m           = fmaxf(m, fmaf(sc[x], unscale, (float) e));
                }
                m                = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m                = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const float next = fmaxf(ref, m - 7.0f);
                if (valid && next > -INFINITY) {
                    const float alpha = exp2_approx(ref - next);  // 0 before the first cell
                    ref               = next;
                    sum *= alpha;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        o[k][0] *= alpha;
                        o[k][1] *= alpha;
#pragma unroll
                        for (int l = 0; l < 4; ++l) {
                            acc[k][l] *= alpha;
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const float z = sc[x] * unscale;
                    pw[x]         = ref > -INFINITY ? exp2_approx(fmaf(sc[x], unscale, -ref)) : isnan(z) ? z : 0.0f;
                }
            }
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                add += pw[x];
            }
            sum += add;
            if (poison) {
                o[0][0] = o[0][1] = o[1][0] = o[1][1] = o[2][0] = o[2][1] = o[3][0] = o[3][1] = NAN;
            }
#pragma unroll
            for (int x = 0; x < 8; x += 2) {
                split_half(pw[x] * dv[x], pw[x + 1] * dv[x + 1], ah[x >> 2][x & 2], ah[x >> 2][(x & 2) + 1]);
            }
            // ---- weighted values of all blocks
            constexpr int kVW = V4 ? (NB + 1) / 2 : NB;  // words of a value chunk
            uint32_t      vw[8][kVW];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                load_chunk<kVW, EXACT>(sv + (4 * x + c4) * vrow + g * (vrow / 8), V4 ? nb : 2 * nb, vw[x]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (!EXACT && b >= nb) {
                    break;
                }
                const uint32_t own = b == block ? 0xffffffffu : 0u;
#pragma unroll
                for (int grp = 0; grp < 2; ++grp) {
                    const int      x = 4 * grp, k = V4 ? b / 2 : b;
                    const uint32_t am[4] = { ah[grp][0] & own, ah[grp][1] & own, ah[grp][2] & own, ah[grp][3] & own };
                    uint32_t       f0[4], f1[4];
                    value_operands<V4>(vw[x][k], vw[x + 1][k], b & 1, f0);
                    value_operands<V4>(vw[x + 2][k], vw[x + 3][k], b & 1, f1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        mma_f16(acc[e], am, f0[e], f1[e]);
                    }
                }
            }
            if (++done == kFold) {
                done = 0;
                fold();
            }
        }
        __syncwarp();
        if (i + n_stages < t.mine) {
            issue(i + n_stages, stage);
        }
        stage = stage + 1 == n_stages ? 0 : stage + 1;
        phase ^= stage == 0;
    }
    if (i < t.mine) {
        attend_abandon(a, full, t.mine, n_stages, i);
    }
    __syncthreads();  // the stages' memory is free
    fold();
    pdl_launch_dependents();  // here, not first: CTAs that wait would take slots where it suits them, not evenly
    // ---- to shared memory: [warp][row][value], statistics of (row, block)
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (c4 == 0) {
        sh.ref[warp * kStats + g] = ref;
        sh.sum[warp * kStats + g] = sum;
    }
    if (block < nb) {
        float * to = reinterpret_cast<float *>(sh.stages) + (size_t) (warp * kRows + g / NB) * hd + 32 * block + 8 * c4;
        *reinterpret_cast<float4 *>(to)     = make_float4(o[0][0], o[1][0], o[2][0], o[3][0]);
        *reinterpret_cast<float4 *>(to + 4) = make_float4(o[0][1], o[1][1], o[2][1], o[3][1]);
    }
    __syncthreads();
    attend_join<kRows, NB>(a, t, sh, hd, 1, n_split);
}

template <int NB, bool EXACT, int REGS>
const void * attend_few(int k4, int v4) {
    return k4 ? (v4 ? (const void *) kv_attend_few_kernel<NB, EXACT, true, true, REGS> : (const void *) kv_attend_few_kernel<NB, EXACT, true, false, REGS>)
              : (v4 ? (const void *) kv_attend_few_kernel<NB, EXACT, false, true, REGS> : (const void *) kv_attend_few_kernel<NB, EXACT, false, false, REGS>);
}

template <int REGS>
const void * attend_few_of(int nb, int k4, int v4) {
    return nb == 2   ? attend_few<2, true, REGS>(k4, v4)
           : nb == 4 ? attend_few<4, true, REGS>(k4, v4)
           : nb == 1 ? attend_few<2, false, REGS>(k4, v4)
                     : attend_few<4, false, REGS>(k4, v4);
}

}  // namespace

int kv_attend_few_rows(int nb) {
    return nb <= 2 ? 4 : nb <= 4 ? 2 : 0;
}

const void * kv_attend_few(int nb, int warps, int k4, int v4) {
    return warps == 8 ? attend_few_of<128>(nb, k4, v4) : attend_few_of<168>(nb, k4, v4);
}

}  // namespace b200q8
