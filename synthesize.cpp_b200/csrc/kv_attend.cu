// kv_attend.cu -- attention over the quantised cache on the tensor cores.
//
// Mathematics.  With codes c (small integers) and one scale d per 32-value
// block, a score is  s_j = sum_b dk[j][b] * (sum_{i in b} q_i ck[j][i])  and an
// output  o_i = sum_j (w_j dv[j][b(i)]) cv[j][i].  Both inner sums are matrix
// products whose cache operand is the integer codes themselves, exact in fp16,
// so nothing of the cache is rounded: block scales multiply the fp32 sums of
// the first product and the weights of the second.  The other operand (q,
// and w * dv) is split into an fp16 value and the fp16 value of what that
// leaves over, 22 bits together, which makes the products as good as fp32
// ones.  q is first scaled by a power of two per row so that its largest
// value lies in [2^14, 2^15), and weights are taken relative to a running
// reference  ref = max_j s_j + e - 14  with 2^e <= max dv < 2^(e+1)  (log2
// units; the score's maximum runs, the scales' is a step's own, because large
// scales at small weights would cost all later steps bits), so that w * dv is
// below 2^15 and held to 2^-22 of itself or 2^-38 of the largest weight times
// the step's largest scale.  The sum of weights uses the same reference, so the
// result is their plain quotient.
//
// Work split.  A CTA takes a tile of query rows (tokens x heads of one kv
// head, token major) of one run; a cluster of CTAs splits the tile's visible
// cells and joins its partial results through distributed shared memory
// (fixed order: the same call gives the same bits).  Tiles of tc
// cells arrive by bulk copies (one contiguous run per array) in a ring of
// stages.  The CTA's warps are wr row groups times cell groups; a warp takes
// 32 cells at a time.  Few rows have a form of their own (kv_attend_few.cu),
// long prompts one on tcgen05 (kv_attend_many.cu); here are STACKED, 8 rows a
// warp, q's two parts in the upper and lower half of one 16-row operand (no
// second product), and TALL, 16 rows a warp, a product for each part (half the
// conversions of codes per row).
//
// Fragments.  A key row's chunk c holds, of each block, values 8c .. 8c+7:
// what lane c of a quad feeds to the block's two products.  A value row's
// chunk g holds values 4g .. 4g+3 of each block: what lane group g feeds to
// the block's four 8-column products.  The 32 cells of a step are dealt so
// that the columns a thread has scores of are the cells whose values it loads:
// column 2c + i of 8-column tile u of 16-cell group s is cell 16s+8u+4i+c.
//
// 24 streams, 24 heads over 4 of 64 values, 8-bit, bf16 (38 MB): 25 us a call,
// 1.5 TB/s; one wave of clusters, bound by the chain of a step (codes to fp16,
// two products with a reduction between them) rather than by the copies.
#include "kv_attend.cuh"

#include <algorithm>
#include <atomic>

namespace b200q8 {
namespace {

// NB: the most blocks a head has (EXACT: all of them).  K4, V4: 4-bit codes.
// PARTS (TALL): fp16 parts of q; 1 for bf16 rows, whose 8 bits one fp16 value
// holds.  Weights have two parts for every type.
template <int NB, bool EXACT, bool K4, bool V4, bool TALL, int PARTS>
__global__ void __launch_bounds__(128)
    kv_attend_kernel(const KvAttendArgs a, const int wr, const int n_split, const int n_stages, const int tc) {
    constexpr int kRows = TALL ? 16 : 8;
    constexpr int kHalf = TALL ? 2 : 1;       // rows a thread has scores of: g (and g + 8)
    constexpr int kQ    = TALL ? PARTS : 1;   // q operands
    extern __shared__ __align__(128) uint8_t smem[];
    const AttendShared sh = attend_shared(smem);
    const int nb   = EXACT ? NB : a.c.nb;
    const int hd   = nb * 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c4 = lane & 3;
    attend_init(sh, n_stages);
    pdl_wait_primary();
    AttendTile t;
    if (!attend_tile(a, nb, kRows * wr, row_tile(n_split), blockIdx.y, tc, blockIdx.x % n_split, n_split, t)) {
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < min(t.mine, n_stages); ++i) {
            t.issue(a.c.n_ctx, sh.stages + i * t.stage_bytes, &sh.full[i], i);
        }
    }
    const KvRun & r = t.r;
    const int     es = a.type == kSrcF32 ? 4 : 2, krow = t.krow, vrow = t.vrow, drow = t.drow;

    // ---- this thread's query rows, as fp16 parts of q * 2^x
    const int rg = warp % wr, pg = warp / wr, n_pg = (int) (blockDim.x >> 5) / wr;
    const int warp_row = t.row + rg * kRows, n_rows = t.n_rows;
    uint32_t  qf[NB][2][kQ][4];
    float     unscale[kHalf];
    int       prow[kHalf], lrow[kHalf];  // a row sees positions in (lrow, prow], and sinks
#pragma unroll
    for (int h = 0; h < kHalf; ++h) {
        const int  row   = warp_row + g + 8 * h;
        const bool valid = row < n_rows;
        const int  token = valid ? row / a.group : 0;
        const int  head  = t.kvh * a.group + (valid ? row % a.group : 0);
        const uint8_t * src = static_cast<const uint8_t *>(a.q) + (size_t) (r.row + token) * a.q_stride +
                              (size_t) (head * hd + 8 * c4) * es;
        prow[h] = valid ? r.pos + token : -1;
        lrow[h] = a.window ? prow[h] - a.window : -1;
        float q[NB][8];
        float top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
            if (b < nb && valid) {
                x = load4(src + (size_t) (32 * b) * es, a.type, a.wide);
                y = load4(src + (size_t) (32 * b + 4) * es, a.type, a.wide);
            }
            const float v[8] = { x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w };
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[b][e] = v[e];
                top     = fmaxf(top, fabsf(v[e]));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float up;
        row_scale(top, a.scale, 15, up, unscale[h]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                uint32_t h0, l0, h1, l1;
                split_half(q[b][key_value<K4>(kk, 0, 0)] * up, q[b][key_value<K4>(kk, 0, 1)] * up, h0, l0);
                split_half(q[b][key_value<K4>(kk, 1, 0)] * up, q[b][key_value<K4>(kk, 1, 1)] * up, h1, l1);
                if (TALL) {
                    qf[b][kk][0][h]     = h0;
                    qf[b][kk][0][2 + h] = h1;
                    if (PARTS == 2) {
                        qf[b][kk][kQ - 1][h]     = l0;
                        qf[b][kk][kQ - 1][2 + h] = l1;
                    }
                } else {
                    qf[b][kk][0][0] = h0;
                    qf[b][kk][0][1] = l0;
                    qf[b][kk][0][2] = h1;
                    qf[b][kk][0][3] = l1;
                }
            }
        }
    }
    // positions of the warp's first and last row (its rows are consecutive tokens)
    const bool has_rows = warp_row < n_rows;
    const int  wpos_lo  = r.pos + min(warp_row, n_rows - 1) / a.group;
    const int  wpos_hi  = r.pos + min(warp_row + kRows - 1, n_rows - 1) / a.group;
    const int  wlow_lo = a.window ? wpos_lo - a.window : -1, wlow_hi = a.window ? wpos_hi - a.window : -1;

    float ref_m[kHalf], sum[kHalf], o[NB][4][2 * kHalf];
    int   ref_e = -25;
#pragma unroll
    for (int h = 0; h < kHalf; ++h) {
        ref_m[h] = -INFINITY;
        sum[h]   = 0.0f;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int i = 0; i < 2 * kHalf; ++i) {
                o[b][e][i] = 0.0f;
            }
        }
    }

    int i = 0, stage = 0, phase = 0;
    for (; i < t.mine; ++i) {
        if (!mbar_wait_bounded(&sh.full[stage], phase)) {
            *sh.dead = 1;
        }
        uint8_t * const s    = sh.stages + stage * t.stage_bytes;
        const int       cell = t.cell(i);
        for (int st = pg; st < tc / kStep && has_rows; st += n_pg) {
            const int c0 = cell + st * kStep;
            // which of the step's cells some row, and every row, sees
            const int      p    = c0 + lane < a.c.n_ctx ? t.position(c0 + lane) : kNever;
            const bool     sink = p < a.c.sinks;
            const uint32_t any  = __ballot_sync(0xffffffffu, p <= wpos_hi && (p > wlow_lo || sink));
            const bool     all  = __all_sync(0xffffffffu, p <= wpos_lo && (p > wlow_hi || sink));
            if (any == 0) {
                continue;
            }
            const uint8_t * sk = s + st * kStep * krow, * sv = s + t.off_v + st * kStep * vrow;
            const uint8_t * skd = s + t.off_kd + st * kStep * drow, * svd = s + t.off_vd + st * kStep * drow;

            // ---- scores of the step's four 8-column tiles
            float sc[4][2 * kHalf];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int       at = 8 * n + 4 * (g & 1) + (g >> 1);  // the cell this lane loads keys of
                const uint8_t * kp = sk + at * krow + c4 * (krow / 4);
                constexpr int   kW = K4 ? 1 : 2;                      // words a block
                uint32_t        w[NB * kW];
                if (EXACT) {
                    load_words<NB * kW>(kp, w);
                } else {
#pragma unroll
                    for (int j = 0; j < NB * kW; ++j) {
                        w[j] = j < nb * kW ? *reinterpret_cast<const uint32_t *>(kp + 4 * j) : 0u;
                    }
                }
                uint32_t dw[2][(NB + 1) / 2];  // scales of cells 8n + c, 8n + 4 + c
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint8_t * dp = skd + (8 * n + 4 * j + c4) * drow;
                    if (EXACT) {
                        load_words<(NB + 1) / 2>(dp, dw[j]);
                    } else {
#pragma unroll
                        for (int b = 0; b < NB; b += 2) {
                            const unsigned short * dh = reinterpret_cast<const unsigned short *>(dp) + b;
                            dw[j][b / 2] = (b < nb ? dh[0] : 0u) | (b + 1 < nb ? (uint32_t) dh[1] << 16 : 0u);
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2 * kHalf; ++h) {
                    sc[n][h] = 0.0f;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (!EXACT && b >= nb) {
                        break;
                    }
                    uint32_t f[4];
                    key_operands<K4>(w[kW * b], w[kW * b + kW - 1], f);
                    float acc[4];
                    mma_f16_first(acc, qf[b][0][kQ - 1], f[0], f[1]);
                    mma_f16(acc, qf[b][1][kQ - 1], f[2], f[3]);
                    if (kQ > 1) {
                        mma_f16(acc, qf[b][0][0], f[0], f[1]);
                        mma_f16(acc, qf[b][1][0], f[2], f[3]);
                    }
                    const float2 d0 = __half22float2(bits_h2(dw[0][b / 2])), d1 = __half22float2(bits_h2(dw[1][b / 2]));
                    const float  da = b & 1 ? d0.y : d0.x, db = b & 1 ? d1.y : d1.x;
                    if (TALL) {
                        sc[n][0] = fmaf(acc[0], da, sc[n][0]);
                        sc[n][1] = fmaf(acc[1], db, sc[n][1]);
                        sc[n][2 * kHalf - 2] = fmaf(acc[2], da, sc[n][2 * kHalf - 2]);
                        sc[n][2 * kHalf - 1] = fmaf(acc[3], db, sc[n][2 * kHalf - 1]);
                    } else {
                        sc[n][0] = fmaf(acc[0] + acc[2], da, sc[n][0]);
                        sc[n][1] = fmaf(acc[1] + acc[3], db, sc[n][1]);
                    }
                }
            }

            // an infinite scale: values of both signs, so the score is not a number
#pragma unroll
            for (int n = 0; n < 4; ++n) {
#pragma unroll
                for (int h = 0; h < 2 * kHalf; ++h) {
                    sc[n][h] = fmaf(sc[n][h], 0.0f, sc[n][h]);
                }
            }

            // ---- which of this thread's cells its rows see
            uint32_t seen[kHalf];  // bit 2n + j: cell 8n + 4j + c
#pragma unroll
            for (int h = 0; h < kHalf; ++h) {
                seen[h] = 0xffu;
            }
            if (!all) {
#pragma unroll
                for (int n = 0; n < 4; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int pc = __shfl_sync(0xffffffffu, p, 8 * n + 4 * j + c4);
#pragma unroll
                        for (int h = 0; h < kHalf; ++h) {
                            if (!(pc <= prow[h] && (pc > lrow[h] || pc < a.c.sinks))) {
                                seen[h] &= ~(1u << (2 * n + j));
                                sc[n][2 * h + j] = -INFINITY;
                            }
                        }
                    }
                }
            }

            // ---- scales of this thread's cells' values, their largest exponent
            uint32_t dv[8][(NB + 1) / 2];
            __half2  top = bits_h2(0u);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const uint8_t * dp = svd + (4 * x + c4) * drow;
                if (EXACT) {
                    load_words<(NB + 1) / 2>(dp, dv[x]);
                } else {
#pragma unroll
                    for (int b = 0; b < NB; b += 2) {
                        const unsigned short * dh = reinterpret_cast<const unsigned short *>(dp) + b;
                        dv[x][b / 2] = (b < nb ? dh[0] : 0u) | (b + 1 < nb ? (uint32_t) dh[1] << 16 : 0u);
                    }
                }
#pragma unroll
                for (int b = 0; b < (NB + 1) / 2; ++b) {
                    if (NB == 1) {
                        dv[x][b] &= 0xffffu;
                    }
                    if (!all && !(any >> (4 * x + c4) & 1u)) {
                        dv[x][b] = 0u;  // no row sees it: whatever it holds must not count
                    }
                    top = __hmax2_nan(top, __habs2(bits_h2(dv[x][b])));
                }
            }
            float dmax = __half2float(__hmax_nan(__low2half(top), __high2half(top)));
            {
                const float d1 = __shfl_xor_sync(0xffffffffu, dmax, 1);
                dmax           = isnan(dmax) || isnan(d1) ? NAN : fmaxf(dmax, d1);
                const float d2 = __shfl_xor_sync(0xffffffffu, dmax, 2);
                dmax           = isnan(dmax) || isnan(d2) ? NAN : fmaxf(dmax, d2);
            }
            uint32_t poison[kHalf];  // bit b: a row sees a scale of block b that is not finite
#pragma unroll
            for (int h = 0; h < kHalf; ++h) {
                poison[h] = 0u;
            }
            const bool odd = !(dmax <= 65504.0f);  // the same for the whole warp
            if (odd) {
                dmax = 0.0f;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t bits = b & 1 ? dv[x][b / 2] >> 16 : dv[x][b / 2] & 0xffffu;
                        if ((bits & 0x7c00u) == 0x7c00u) {
#pragma unroll
                            for (int h = 0; h < kHalf; ++h) {
                                poison[h] |= (seen[h] >> x & 1u) << b;
                            }
                            dv[x][b / 2] &= b & 1 ? 0x0000ffffu : 0xffff0000u;
                        } else {
                            dmax = fmaxf(dmax, fabsf(__half2float(__ushort_as_half((unsigned short) bits))));
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < kHalf; ++h) {
                    poison[h] |= __shfl_xor_sync(0xffffffffu, poison[h], 1);
                    poison[h] |= __shfl_xor_sync(0xffffffffu, poison[h], 2);
                }
                dmax = fmaxf(dmax, __shfl_xor_sync(0xffffffffu, dmax, 1));
                dmax = fmaxf(dmax, __shfl_xor_sync(0xffffffffu, dmax, 2));
            }
            const int e_new = max(-25, (int) (__float_as_uint(dmax) >> 23) - 127);

            // ---- weights relative to the new reference
            float alpha[kHalf];
#pragma unroll
            for (int h = 0; h < kHalf; ++h) {
                float m = ref_m[h];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    m = fmaxf(m, fmaxf(sc[n][2 * h] * unscale[h], sc[n][2 * h + 1] * unscale[h]));
                }
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const float ref = (m == -INFINITY ? 0.0f : m) + (float) (e_new - 14);
                alpha[h]        = exp2_approx(ref_m[h] + (float) (ref_e - 14) - ref);  // 0 before the first cell
                ref_m[h]        = m;
                float add       = 0.0f;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        sc[n][2 * h + j] = exp2_approx(fmaf(sc[n][2 * h + j], unscale[h], -ref));
                        add += sc[n][2 * h + j];
                    }
                }
                sum[h] = fmaf(sum[h], alpha[h], add);
            }
            ref_e = e_new;

            // ---- weighted values, block after block
            constexpr int kVW = V4 ? (NB + 1) / 2 : NB;  // words of a value chunk
            uint32_t      vw[8][kVW];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const uint8_t * vp = sv + (4 * x + c4) * vrow + g * (vrow / 8);
                if (EXACT) {
                    load_words<kVW>(vp, vw[x]);
                } else {
#pragma unroll
                    for (int j = 0; j < kVW; ++j) {
                        if (V4) {
                            const unsigned short * vh = reinterpret_cast<const unsigned short *>(vp) + 2 * j;
                            vw[x][j] = (2 * j < nb ? vh[0] : 0u) | (2 * j + 1 < nb ? (uint32_t) vh[1] << 16 : 0u);
                        } else {
                            vw[x][j] = j < nb ? *reinterpret_cast<const uint32_t *>(vp + 4 * j) : 0u;
                        }
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (!EXACT && b >= nb) {
                    break;
                }
                float acc[4][4];
#pragma unroll
                for (int grp = 0; grp < 2; ++grp) {  // 16 cells
                    uint32_t f[2][4];                // [cells c, 4 + c | 8 + c, 12 + c][value of the chunk]
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int x = 4 * grp + 2 * u;
                        const int k = V4 ? b / 2 : b;
                        value_operands<V4>(vw[x][k], vw[x + 1][k], b & 1, f[u]);
                    }
                    uint32_t ahi[4], alo[4];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int    n  = 2 * grp + u;
                        const float2 d0 = __half22float2(bits_h2(dv[2 * n][b / 2])), d1 = __half22float2(bits_h2(dv[2 * n + 1][b / 2]));
                        const float  da = b & 1 ? d0.y : d0.x, db = b & 1 ? d1.y : d1.x;
#pragma unroll
                        for (int h = 0; h < kHalf; ++h) {
                            uint32_t hi, lo;
                            split_half(sc[n][2 * h] * da, sc[n][2 * h + 1] * db, hi, lo);
                            if (TALL) {
                                ahi[2 * u + h] = hi;
                                alo[2 * u + h] = lo;
                            } else {
                                ahi[2 * u]     = hi;
                                ahi[2 * u + 1] = lo;
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (grp == 0) {
                            mma_f16_first(acc[e], TALL ? alo : ahi, f[0][e], f[1][e]);
                        } else {
                            mma_f16(acc[e], TALL ? alo : ahi, f[0][e], f[1][e]);
                        }
                        if (TALL) {
                            mma_f16(acc[e], ahi, f[0][e], f[1][e]);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (TALL) {
#pragma unroll
                        for (int h = 0; h < kHalf; ++h) {
                            o[b][e][2 * h]     = fmaf(o[b][e][2 * h], alpha[h], acc[e][2 * h]);
                            o[b][e][2 * h + 1] = fmaf(o[b][e][2 * h + 1], alpha[h], acc[e][2 * h + 1]);
                        }
                    } else {
                        o[b][e][0] = fmaf(o[b][e][0], alpha[0], acc[e][0] + acc[e][2]);
                        o[b][e][1] = fmaf(o[b][e][1], alpha[0], acc[e][1] + acc[e][3]);
                    }
                }
            }
            if (odd) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
#pragma unroll
                    for (int h = 0; h < kHalf; ++h) {
                        if (poison[h] >> b & 1u) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                o[b][e][2 * h] = o[b][e][2 * h + 1] = NAN;
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();
        if (*sh.dead) {
            break;
        }
        if (threadIdx.x == 0 && i + n_stages < t.mine) {
            t.issue(a.c.n_ctx, s, &sh.full[stage], i + n_stages);
        }
        stage = stage + 1 == n_stages ? 0 : stage + 1;
        phase ^= stage == 0;
    }
    if (i < t.mine) {
        attend_abandon(a, sh.full, t.mine, n_stages, i);
        __syncthreads();
    }
    pdl_launch_dependents();  // here, not first: CTAs that wait would take slots where it suits them, not evenly
    // ---- to shared memory: [warp][row][value]
    float * part = reinterpret_cast<float *>(sh.stages);
#pragma unroll
    for (int h = 0; h < kHalf; ++h) {
        float l = sum[h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int row = g + 8 * h;
        if (c4 == 0) {
            sh.ref[warp * kStats + row] = ref_m[h] + (float) (ref_e - 14);
            sh.sum[warp * kStats + row] = l;
        }
        float * to = part + (size_t) (warp * kRows + row) * hd + 8 * c4;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (b < nb) {
                *reinterpret_cast<float4 *>(to + 32 * b) =
                    make_float4(o[b][0][2 * h], o[b][1][2 * h], o[b][2][2 * h], o[b][3][2 * h]);
                *reinterpret_cast<float4 *>(to + 32 * b + 4) =
                    make_float4(o[b][0][2 * h + 1], o[b][1][2 * h + 1], o[b][2][2 * h + 1], o[b][3][2 * h + 1]);
            }
        }
    }
    __syncthreads();
    attend_join<kRows, 1>(a, t, sh, hd, wr, n_split);
}

template <int NB, bool EXACT, bool TALL, int PARTS>
const void * attend_fn(int k4, int v4) {
    return k4 ? (v4 ? (const void *) kv_attend_kernel<NB, EXACT, true, true, TALL, PARTS> : (const void *) kv_attend_kernel<NB, EXACT, true, false, TALL, PARTS>)
              : (v4 ? (const void *) kv_attend_kernel<NB, EXACT, false, true, TALL, PARTS> : (const void *) kv_attend_kernel<NB, EXACT, false, false, TALL, PARTS>);
}

// Shared-memory and cluster attributes, once a kernel and device.
cudaError_t prepare_kernel(const void * fn) {
    constexpr int               kSlots = 128;
    static std::atomic<const void *> ready[64][kSlots];
    int                         dev = 0;
    cudaError_t                 e   = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
        return e;
    }
    const bool known = dev >= 0 && dev < 64;
    int        i     = 0;
    for (; known && i < kSlots; ++i) {
        const void * k = ready[dev][i].load(std::memory_order_acquire);
        if (k == fn) {
            return cudaSuccess;
        }
        if (k == nullptr) {
            break;
        }
    }
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e == cudaSuccess) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    }
    for (; e == cudaSuccess && known && i < kSlots; ++i) {
        const void * none = nullptr;
        if (ready[dev][i].compare_exchange_strong(none, fn) || none == fn) {
            break;
        }
    }
    return e;
}

// Which kernel a call launches, and how.
struct AttendPlan {
    const void * fn;
    bool         few, many;
    int          threads;
    int          wr, split, tc, n_stages;
    int64_t      tiles;
    size_t       smem;
};

AttendPlan attend_plan(const KvAttendArgs & a, int sm_count) {
    AttendPlan    p  = {};
    const int     nb = a.c.nb, k4 = a.c.four[0], v4 = a.c.four[1];
    const int64_t rows = (int64_t) a.b.max_len * a.group;
    // Prompts: the 128-row kernel, where its CTAs (one an SM) take 3 of 8 SMs
    // or more; fewer leave too much idle, and the others can split the cells.
    // 512 tokens after 4000 (64 CTAs) 189 us against 284 us, 512 after none 33
    // against 55 us; 256 after 8000 (32 CTAs) 325 against 261 us.
    const KvAttendMany m = kv_attend_many(nb, k4, v4, a.type);
    if (m.fn != nullptr && rows >= m.rows) {
        p.tiles = (rows + m.rows - 1) / m.rows;
        if (8 * p.tiles * a.c.n_kv * a.b.n_seqs >= 3 * (int64_t) sm_count) {
            p.fn      = m.fn;
            p.many    = true;
            p.threads = m.threads;
            p.split   = 1;
            p.smem    = m.smem;
            return p;
        }
    }
    p.few = rows <= kv_attend_few_rows(nb);
    const bool tall  = !p.few && rows > 8 && (nb == 2 || nb == 4);
    const int  high  = p.few ? kv_attend_few_rows(nb) : tall ? 16 : 8;
    p.wr             = 1;
    if (!p.few) {
        p.wr           = rows <= high ? 1 : rows <= 2 * high ? 2 : 4;
        const bool one = a.type == kSrcBF16;
        p.fn = tall ? (nb == 2 ? (one ? attend_fn<2, true, true, 1>(k4, v4) : attend_fn<2, true, true, 2>(k4, v4))
                               : (one ? attend_fn<4, true, true, 1>(k4, v4) : attend_fn<4, true, true, 2>(k4, v4)))
               : nb == 2 ? attend_fn<2, true, false, 2>(k4, v4)
               : nb == 4 ? attend_fn<4, true, false, 2>(k4, v4)
               : nb == 8 ? attend_fn<8, true, false, 2>(k4, v4)
                         : attend_fn<8, false, false, 2>(k4, v4);
    }
    p.tiles = (rows + high * p.wr - 1) / (high * p.wr);
    const int64_t base  = p.tiles * a.c.n_kv * a.b.n_seqs;
    const int64_t reach = a.window ? std::min((int64_t) a.c.n_ctx, (int64_t) a.window + a.b.max_len + a.c.sinks) : a.c.n_ctx;
    // Slots are counted as three CTAs of four warps an SM, which is what fits at
    // 168 registers a thread or fewer (the few-row kernel, heads of 64).  Of the
    // forms with up to 255 two fit (heads of 128 in 16-row tiles, heads of more
    // blocks), of heads of 256 in 8 bits one (139 KB of stages); there a call
    // near the count takes a second wave.
    // While the rows leave slots free the cells are split over a cluster: 8 kv
    // heads of one stream over 32701 cells take 420 us unsplit and 41 us over
    // 16 CTAs, 32 streams over 2000 cells 37 us unsplit (256 CTAs) and 43 us
    // over 2.  More rows than slots: two parts even out streams of different
    // length (64 streams of 698 to 8100 cells: 154 to 146 us).  A part is at
    // least a warp step for each warp.
    // Where a cluster of 16 is all there is and few of them, eight warps a CTA
    // (one stream over 32701 cells in 4 bits: 37 to 35 us, two 55 to 47; heads
    // of 128 in 8 bits have room for one stage a warp then).
    const int64_t slots = 3 * (int64_t) sm_count;
    const int     warps = p.few && 2 * base * 16 <= slots && reach >= kStep * 8 * 16 ? 8 : 4;
    const int64_t most  = std::min<int64_t>(16, std::max<int64_t>(1, reach / (kStep * warps)));
    if (p.few) {
        p.fn = kv_attend_few(nb, warps, k4, v4);
    }
    p.threads           = 32 * warps;
    p.split             = (int) std::min(most, base <= slots ? slots / base : p.few ? 2 : 1);
    p.tc                = kStep * warps;  // cells a stage holds
    const int stage     = p.tc * nb * ((k4 ? 16 : 32) + (v4 ? 16 : 32) + 4);
    const int budget    = warps == 8 ? 113 * 1024 : 75 * 1024;  // shared memory: two CTAs an SM, or three
    p.n_stages          = stage * 4 <= budget ? 4 : stage * 3 <= budget ? 3 : stage * 2 <= budget || warps == 4 ? 2 : 1;
    p.smem              = kHeadBytes + std::max(p.n_stages * stage, warps * high * nb * 32 * 4);
    return p;
}

}  // namespace

cudaError_t prepare_kv_attend(const KvAttendArgs & a, int sm_count) {
    return prepare_kernel(attend_plan(a, sm_count).fn);
}

cudaError_t launch_kv_attend(const KvAttendArgs & args, cudaStream_t stream, int sm_count) {
    KvAttendArgs a = args;
    AttendPlan   p = attend_plan(a, sm_count);
    cudaError_t  e = prepare_kernel(p.fn);
    if (e != cudaSuccess) {
        return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = p.many ? dim3((unsigned) (p.tiles * a.c.n_kv), 1, (unsigned) a.b.n_seqs)
                                    : dim3((unsigned) (p.tiles * p.split), (unsigned) a.c.n_kv, (unsigned) a.b.n_seqs);
    cfg.blockDim           = dim3((unsigned) p.threads);
    cfg.dynamicSmemBytes   = p.smem;
    cfg.stream             = stream;
    // programmatic dependent launch: the kernels may start while the one before
    // them in the stream ends, and touch memory after griddepcontrol.wait
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id                                         = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x                           = (unsigned) p.split;
    attr[1].val.clusterDim.y                           = 1;
    attr[1].val.clusterDim.z                           = 1;
    cfg.attrs                                          = attr;
    cfg.numAttrs                                       = p.split > 1 ? 2 : 1;
    if (p.many) {
        void * params[] = { &a };
        return cudaLaunchKernelExC(&cfg, p.fn, params);
    }
    if (p.few) {
        void * params[] = { &a, &p.split, &p.n_stages };
        return cudaLaunchKernelExC(&cfg, p.fn, params);
    }
    void * params[] = { &a, &p.wr, &p.split, &p.n_stages, &p.tc };
    return cudaLaunchKernelExC(&cfg, p.fn, params);
}

}  // namespace b200q8
