// Attention of each sequence's last rows over its pages.
//
// o = sum_t p_t v_t with p = softmax over the positions t that a row sees, in one pass with the running
// maximum and sum of the softmax in 32 bits.  The product's sides are swapped, S^T = K Q^T and
// O^T = V^T P^T: the scores of v_mfma_f32_16x16x32_f16 then leave each lane the probabilities of four
// positions of a tile for its own column, and those of two tiles are, as they stand, the second
// product's operand.  Nothing passes through LDS or between lanes but the rare new maximum.
#include <algorithm>

#include "paged.h"
#include "paged_device.h"

namespace bh {
namespace {

constexpr int kWaves = 4;
constexpr int kPair = 32;        // positions of two tiles, one product's
constexpr int kColumns = 16;     // (row, head) pairs of a key/value head that share a pass
// Pairs of tiles that a wave takes at a time: two where its registers hold their loads.
constexpr int pairs_at_once(int nb) { return nb <= 2 ? 2 : 1; }
// Waves a SIMD holds at once, by the registers that a head size takes (a workgroup is one wave a SIMD).  Held to one
// more the kernels of 128 values take 32 us for 60001 4-bit positions instead of 22 (registers spilled); those of
// 64 with four, a pair of tiles at a time, 70 us for 64 sequences instead of 66.
constexpr int resident(int nb) { return nb <= 4 ? 2 : 1; }
constexpr int kMergeRow = 132;   // LDS floats a column, for 128 values: 16-byte rows, shifted over the banks

// What a wave holds of two tiles: keys, values and, of 4-bit tiles, their scales.
template <int NB, bool Q4>
struct TilePair {
    static constexpr int GS = NB < 4 ? NB : 4, NG = NB / GS;
    uint32_t k[2][NG][Q4 ? GS : 4 * GS], v[2][NG][Q4 ? 1 : 4][GS];
    uint32_t ks[2][NG][Q4 ? 2 * GS : 1], vs[2][NG][Q4 ? 2 * GS : 1];

    __device__ inline void load_keys(const uint8_t* tile, int x, int lane) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if constexpr (Q4) {
                load_words<GS>(tile + (n * 64 + lane) * GS * 4, k[x][n]);
                load_words<2 * GS>(tile + tile_key_scales_at(NB) + (lane / 16 * NB + n * GS) * 8, ks[x][n]);
            } else {
#pragma unroll
                for (int j = 0; j < GS; ++j) {
                    const word4v w = *reinterpret_cast<const word4v*>(tile + ((n * GS + j) * 64 + lane) * 16);
                    for (int e = 0; e < 4; ++e) k[x][n][4 * j + e] = w[e];
                }
            }
        }
    }
    __device__ inline void load_values(const uint8_t* tile, int x, int n, int lane) {
        const uint8_t* at = tile + tile_values_at(Q4, NB);
        if constexpr (Q4) {
            load_words<GS>(at + (n * 64 + lane) * GS * 4, v[x][n][0]);
            load_words<2 * GS>(tile + tile_value_scales_at(NB) + (lane / 16 * NB + n * GS) * 8, vs[x][n]);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) load_words<GS>(at + ((r * NG + n) * 64 + lane) * GS * 4, v[x][n][r]);
        }
    }
    // Leaves out the values of positions whose bit 4 x + r of `seen` is not set, whatever lies there.
    __device__ inline void keep_seen(int n, uint32_t seen) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if constexpr (Q4) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t b = seen >> (4 * x + 2 * j), mask = (b & 1 ? 0xFFFF : 0) | (b & 2 ? 0xFFFF0000 : 0);
                    for (int k = 0; k < GS; ++k) vs[x][n][2 * k + j] &= mask;
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t mask = seen >> (4 * x + r) & 1 ? 0xFFFFFFFF : 0;
                    for (int k = 0; k < GS; ++k) v[x][n][r][k] &= mask;
                }
            }
        }
    }
    // Whether infinities or NaN are among a group of blocks' values.
    __device__ inline bool any_ill(int n) const {
        uint32_t found = 0;
        for (int x = 0; x < 2; ++x) {
            if constexpr (Q4) {
                for (int j = 0; j < 2 * GS; ++j) found |= ill<true>(vs[x][n][j]);
            } else {
                for (int r = 0; r < 4; ++r)
                    for (int j = 0; j < GS; ++j) found |= ill<false>(v[x][n][r][j]);
            }
        }
        return __any((found & kIll) != 0);
    }
};

// Where the statistics of a row's head's part are.
template <int HD>
__device__ inline float* part_stats(const PagedAttnArgs& a, uint32_t row, uint32_t head, uint32_t split) {
    return a.part + static_cast<size_t>(a.b.rows) * a.heads * a.splits * HD + ((static_cast<size_t>(row) * a.heads + head) * a.splits + split) * 2;
}

// A workgroup takes up to 16 columns, the (row, head) pairs of one key/value head, and one part of the
// positions they see; its waves take pairs of tiles in turn.  EXACT: queries and probabilities as sums
// of two halves, and 4-bit values as sums of two: 32-bit results.
//
// Over fp16 pages bound by memory: 16 tokens at up to 4000, 8 heads of 128 for 16, 43 us, 4.3 TB/s (a copy moves 5.1 in and out).  Over
// 4 bits by vector issue, 318 instructions for 64 positions of heads of 64, most of them unpacking: 64 tokens at up to 8000, 8 heads of 64
// for 32, 63 us (3.1 TB/s); one at 60001, 8 of 128, 23 (3.0 TB/s), 4 of them the join.  16 columns use half of the products' rate at most, and
// the products do not bound it: with fewer than 16 (row, head) pairs the rest are multiplied for nothing.
template <int NB, bool Q4, bool EXACT>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(resident(NB)))) void k_paged_attn(PagedAttnArgs a) {
    constexpr int GS = NB < 4 ? NB : 4, NG = NB / GS, HD = 32 * NB, QROW = HD + 8, TP = pairs_at_once(NB), STEP = TP * kPair;
    constexpr bool kEarly = NB <= 8;  // all of a pair's loads ahead of its products (the widest heads have no registers for it)
    constexpr bool kHeldQ = NB * (EXACT ? 2 : 1) <= 8;  // queries in registers, otherwise read from LDS for each product
    __shared__ union {
        _Float16 q[EXACT ? 2 : 1][kColumns][QROW];
        float merge[kWaves][kColumns][kMergeRow];
    } lds;
    __shared__ float qfactor[kColumns], stats[kWaves][kColumns][2];
    const int lane = static_cast<int>(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int i = lane % 16, g = lane / 16;
    const uint32_t first_tile = over(blockIdx.y, a.kv_heads), h = blockIdx.y - first_tile * a.kv.kv_heads;
    const int32_t window = a.window > static_cast<uint32_t>(kMaxLength) ? 0 : static_cast<int32_t>(a.window);

    for (uint32_t s = blockIdx.z; s < a.b.seqs; s += gridDim.z) {
        const SeqRows sr = seq_rows(a.b, s);
        const uint32_t cols = (sr.end - sr.begin) * a.group.d;
        for (uint32_t c0 = first_tile * kColumns; c0 < cols; c0 += over(gridDim.y, a.kv_heads) * kColumns) {
            const uint32_t c_last = std::min<uint32_t>(c0 + kColumns, cols) - 1;
            const int32_t pos_lo = sr.first + static_cast<int32_t>(over(c0, a.group)), pos_hi = sr.first + static_cast<int32_t>(over(c_last, a.group));
            const int32_t t_lo = window != 0 && pos_lo - window + 1 > 0 ? pos_lo - window + 1 : 0;
            const int32_t t_hi = static_cast<int32_t>(std::min<int64_t>(static_cast<int64_t>(pos_hi) + 1, static_cast<int64_t>(a.b.page_stride) << a.kv.page_shift));
            const int32_t step_lo = t_lo / STEP, steps = t_hi > t_lo ? (t_hi + STEP - 1) / STEP - step_lo : 0;
            // A part's steps, as the longest sequence would have them: a shorter one has fewer parts, and its workgroups
            // without steps make room.
            const int32_t per = std::max<int32_t>(a.per, steps <= a.per * static_cast<int32_t>(a.splits) ? 0 : (steps + static_cast<int32_t>(a.splits) - 1) / static_cast<int32_t>(a.splits));
            const int32_t first = static_cast<int32_t>(std::min<int64_t>(steps, static_cast<int64_t>(per) * blockIdx.x));
            const int32_t step_end = step_lo + std::min<int32_t>(steps, first + per);
            int32_t step = step_lo + first + wave;
            if (a.splits != 1 && first == steps) {
                const uint32_t c = c0 + threadIdx.x, row = over(c, a.group);
                if (threadIdx.x < kColumns && c < cols) {
                    float* ml = part_stats<HD>(a, sr.begin + row, h * a.group.d + (c - row * a.group.d), blockIdx.x);
                    ml[0] = -__builtin_inff();
                    ml[1] = 0;
                }
                continue;
            }
            // The wave's first pair of tiles is on its way while the queries are made ready.  In the loop the next pair's
            // keys are fetched once these have been multiplied, and its values once these have.
            TilePair<NB, Q4> kv[TP];
            const WavePages pages(a.kv, a.b, s, h);
            const uint8_t* tile[2 * TP] = {};
            uint32_t there = 0, page[2 * TP] = {};
            const auto find = [&](int32_t st) {
#pragma unroll
                for (int x = 0; x < 2 * TP; ++x) page[x] = pages.page(st * STEP + 16 * x);
            };
            const auto locate = [&](int32_t st) {
                there = 0;
#pragma unroll
                for (int x = 0; x < 2 * TP; ++x) {
                    there |= pages.there(page[x]) ? 1u << x : 0;
                    tile[x] = pages.tile(page[x], st * STEP + 16 * x, tile_bytes(Q4, NB));
                }
            };
            const auto fetch_keys = [&] {
#pragma unroll
                for (int x = 0; x < 2 * TP; ++x) kv[x / 2].load_keys(tile[x], x % 2, lane);
            };
            const auto fetch_values = [&] {
#pragma unroll
                for (int n = 0; n < NG; ++n) {
#pragma unroll
                    for (int x = 0; x < 2 * TP; ++x) kv[x / 2].load_values(tile[x], x % 2, n, lane);
                }
            };
            if (steps > 0) find(step);
            locate(step);
            if constexpr (kEarly) {
                fetch_keys();
                fetch_values();
            }
            if (steps > 0) find(step + kWaves);

            // the columns' queries, as halves in LDS: 16 threads a column, scaled by a power of two where
            // the type has more range than a half
            {
                const uint32_t qc = threadIdx.x / 16, sub = threadIdx.x % 16, c = c0 + qc, row = over(c, a.group);
                constexpr int K = (HD + 127) / 128;
                float x[K][8], top = 0;
                const char* qp = row_ptr(a.q, sr.begin + row, h * a.group.d + (c - row * a.group.d));
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    for (int j = 0; j < 8; ++j) x[k][j] = 0;
                    const int d = (k * 16 + sub) * 8;
                    if (c < cols && d < HD) load8(qp, a.q.type, (reinterpret_cast<uintptr_t>(qp) & 15) == 0, d, x[k]);
                    for (int j = 0; j < 8; ++j) top = __builtin_fmaxf(top, __builtin_fabsf(x[k][j]));
                }
                for (int m = 1; m < 16; m *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, m));
                const int e = a.q.type != kTypeF16 && top > 0 && top <= 3.402823466e38f ? __builtin_amdgcn_frexp_expf(top) : 9;
                // (never 0: scores of 0 and of minus infinity, what is not seen, stay what they are)
                if (sub == 0) qfactor[qc] = __builtin_fmaxf(__builtin_ldexpf(__builtin_fabsf(a.scale) * 1.44269504088896f, e - 9), 1.17549435e-38f);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int d = (k * 16 + sub) * 8;
                    half8v hi, lo;
                    for (int j = 0; j < 8; ++j) {
                        const float y = __builtin_ldexpf(a.scale < 0 ? -x[k][j] : x[k][j], 9 - e);
                        hi[j] = static_cast<_Float16>(y);
                        lo[j] = static_cast<_Float16>(y - static_cast<float>(hi[j]));
                    }
                    if (d < HD) {
                        *reinterpret_cast<half8v*>(&lds.q[0][qc][d]) = hi;
                        if constexpr (EXACT) *reinterpret_cast<half8v*>(&lds.q[1][qc][d]) = lo;
                    }
                }
            }
            __syncthreads();
            half8v held[EXACT ? 2 : 1][kHeldQ ? NB : 1];
            if constexpr (kHeldQ) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    for (int e = 0; e < (EXACT ? 2 : 1); ++e) held[e][b] = *reinterpret_cast<const half8v*>(&lds.q[e][i][32 * b + 8 * g]);
                }
            }
            const auto query = [&](int part, int b) -> half8v {
                if constexpr (kHeldQ) return held[part][b];
                else return *reinterpret_cast<const half8v*>(&lds.q[part][i][32 * b + 8 * g]);
            };
            const float qscale = qfactor[i];
            const int32_t pos = c0 + i < cols ? sr.first + static_cast<int32_t>(over(c0 + i, a.group)) : pos_lo;

            Maximum mx;
            float l = 0;
            float4v acc[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b][0] = acc[b][1] = float4v{0, 0, 0, 0};

            for (; step < step_end; step += kWaves) {
                const int32_t t0 = step * STEP;
                const uint32_t here = there;
                const bool more = step + kWaves < step_end;
                float4v sc[2 * TP];
#pragma unroll
                for (int x = 0; x < 2 * TP; ++x) {
                    sc[x] = float4v{0, 0, 0, 0};
                    if constexpr (!kEarly) kv[x / 2].load_keys(tile[x], x % 2, lane);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int n = b / GS, k = b % GS;
                        if constexpr (Q4) {
                            const uint32_t w = kv[x / 2].k[x % 2][n][k], w8 = w >> 8;
                            const half8v kx = operand(bits(codes(w, false)), bits(codes(w, true)), bits(codes(w8, false)), bits(codes(w8, true)));
                            float4v d{0, 0, 0, 0};
                            if constexpr (EXACT) d = mfma(kx, query(1, b), d);
                            d = mfma(kx, query(0, b), d);
                            const half2v s01 = halves(kv[x / 2].ks[x % 2][n][2 * k]), s23 = halves(kv[x / 2].ks[x % 2][n][2 * k + 1]);
                            sc[x][0] = __builtin_fmaf(d[0], static_cast<float>(s01[0]), sc[x][0]);
                            sc[x][1] = __builtin_fmaf(d[1], static_cast<float>(s01[1]), sc[x][1]);
                            sc[x][2] = __builtin_fmaf(d[2], static_cast<float>(s23[0]), sc[x][2]);
                            sc[x][3] = __builtin_fmaf(d[3], static_cast<float>(s23[1]), sc[x][3]);
                        } else {
                            const uint32_t* w = &kv[x / 2].k[x % 2][n][4 * k];
                            const half8v kx = operand(w[0], w[1], w[2], w[3]);
                            if constexpr (EXACT) sc[x] = mfma(kx, query(1, b), sc[x]);
                            sc[x] = mfma(kx, query(0, b), sc[x]);
                        }
                    }
                }
                if constexpr (kEarly) {  // (after the last pair that one again: a branch would keep two sets of registers)
                    if (more) {
                        locate(step + kWaves);
                        find(step + 2 * kWaves);
                    }
                    fetch_keys();
                }
                // positions that every column sees need no masks
                const bool full = here == (1u << 2 * TP) - 1 && t0 + STEP - 1 <= pos_lo && (window == 0 || t0 > pos_hi - window);
                uint32_t seen = 0xFFFF, anyones = 0xFFFF;  // of the lane's positions, by its column and by any
                if (!full) {
                    seen = anyones = 0;
#pragma unroll
                    for (int j = 0; j < 8 * TP; ++j) {
                        const int32_t t = t0 + 16 * (j / 4) + 4 * g + j % 4;
                        const bool is = here >> (j / 4) & 1;
                        if (is && t >= t_lo && t <= pos_hi) anyones |= 1u << j;
                        if (is && t <= pos && (window == 0 || t > pos - window)) seen |= 1u << j;
                        else sc[j / 4][j % 4] = -__builtin_inff();
                    }
                }
                float tops[2 * TP];
#pragma unroll
                for (int x = 0; x < 2 * TP; ++x) tops[x] = __builtin_fmaxf(__builtin_fmaxf(sc[x][0], sc[x][1]), __builtin_fmaxf(sc[x][2], sc[x][3]));
                float top = __builtin_fmaxf(tops[0], tops[1]);
                if constexpr (TP == 2) top = __builtin_fmaxf(top, __builtin_fmaxf(tops[2], tops[3]));
                if (__any(top * qscale > mx.m + kLazy)) {
                    top = __builtin_fmaxf(top, __shfl_xor(top, 16));
                    top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                    const float f = mx.renew(top, qscale);
                    l *= f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        acc[b][0] *= f;
                        acc[b][1] *= f;
                    }
                }
                if (mx.far) {
                    for (int j = 0; j < 8 * TP; ++j) sc[j / 4][j % 4] -= mx.shift;
                }
                half8v ph[TP], pl[EXACT ? TP : 1];
#pragma unroll
                for (int j = 0; j < 8 * TP; j += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j / 4][j % 4], qscale, -mx.base));
                    const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j / 4][j % 4 + 1], qscale, -mx.base));
                    const half2v e{static_cast<_Float16>(e0), static_cast<_Float16>(e1)};
                    ph[j / 8][j % 8] = e[0];
                    ph[j / 8][j % 8 + 1] = e[1];
                    if constexpr (EXACT) {
                        pl[j / 8][j % 8] = static_cast<_Float16>(e0 - static_cast<float>(e[0]));
                        pl[j / 8][j % 8 + 1] = static_cast<_Float16>(e1 - static_cast<float>(e[1]));
                        l += e0;
                        l += e1;
                    } else {
                        l = __builtin_amdgcn_fdot2(e, half2v{1, 1}, l, false);  // (the sum of what is multiplied)
                    }
                }
#pragma unroll
                for (int yn = 0; yn < TP * NG; ++yn) {
                    const int y = yn / NG, n = yn % NG;
                    TilePair<NB, Q4>& kv_ = kv[y];
                    if constexpr (!kEarly) {
                        kv_.load_values(tile[2 * y], 0, n, lane);
                        kv_.load_values(tile[2 * y + 1], 1, n, lane);
                    }
                    if (!full) kv_.keep_seen(n, anyones >> (8 * y));
                    // (in 4 bits a whole block is NaN, which only columns that do not see it need kept from)
                    if ((!full || !Q4) && __builtin_expect(kv_.any_ill(n), 0)) {
                        half8v sees;
                        for (int j = 0; j < 8; ++j) sees[j] = static_cast<_Float16>(seen >> (8 * y + j) & 1 ? 1.0f : 0.0f);
#pragma unroll
                        for (int k = 0; k < GS; ++k) {
                            const int b = n * GS + k;
                            uint32_t up[2][4], down[2][4];  // of the lane's two columns
                            for (int x = 0; x < 2; ++x) {
                                if constexpr (Q4) {
                                    for (int j = 0; j < 2; ++j) {
                                        const Marks mk = scale_marks(kv_.vs[x][n][2 * k + j]);
                                        kv_.vs[x][n][2 * k + j] = mk.rest;
                                        up[0][2 * x + j] = up[1][2 * x + j] = mk.up;
                                        down[0][2 * x + j] = down[1][2 * x + j] = mk.down;
                                    }
                                } else {
                                    for (int j = 0; j < 2; ++j) {
                                        const Marks m0 = marks(kv_.v[x][n][2 * j][k]), m1 = marks(kv_.v[x][n][2 * j + 1][k]);
                                        kv_.v[x][n][2 * j][k] = m0.rest;
                                        kv_.v[x][n][2 * j + 1][k] = m1.rest;
                                        for (int c2 = 0; c2 < 2; ++c2) {
                                            const uint32_t sel = c2 ? 0x07060302 : 0x05040100;
                                            up[c2][2 * x + j] = __builtin_amdgcn_perm(m1.up, m0.up, sel);
                                            down[c2][2 * x + j] = __builtin_amdgcn_perm(m1.down, m0.down, sel);
                                        }
                                    }
                                }
                            }
#pragma unroll
                            for (int c2 = 0; c2 < 2; ++c2) {
                                const float4v none{0, 0, 0, 0};
                                const float4v u = mfma(operand(up[c2][0], up[c2][1], up[c2][2], up[c2][3]), sees, none);
                                const float4v d = mfma(operand(down[c2][0], down[c2][1], down[c2][2], down[c2][3]), sees, none);
                                for (int r = 0; r < 4; ++r) acc[b][c2][r] += ill_sum(u[r], d[r]);
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < GS; ++k) {
                        const int b = n * GS + k;
#pragma unroll
                        for (int c2 = 0; c2 < 2; ++c2) {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                if constexpr (Q4) {
                                    const uint32_t w = kv_.v[x][n][0][k];
                                    const half2v c01 = codes(w, c2), c23 = codes(w >> 8, c2);
                                    const half2v d01 = halves(kv_.vs[x][n][2 * k]), d23 = halves(kv_.vs[x][n][2 * k + 1]);
                                    const half2v v01 = c01 * d01, v23 = c23 * d23;
                                    hi[2 * x] = bits(v01);
                                    hi[2 * x + 1] = bits(v23);
                                    // the product has 15 bits at most and its rounding error is a multiple of d's last place: exact
                                    if constexpr (EXACT) {
                                        lo[2 * x] = bits(__builtin_elementwise_fma(c01, d01, -v01));
                                        lo[2 * x + 1] = bits(__builtin_elementwise_fma(c23, d23, -v23));
                                    }
                                } else {
                                    const uint32_t sel = c2 ? 0x07060302 : 0x05040100;
                                    hi[2 * x] = __builtin_amdgcn_perm(kv_.v[x][n][1][k], kv_.v[x][n][0][k], sel);
                                    hi[2 * x + 1] = __builtin_amdgcn_perm(kv_.v[x][n][3][k], kv_.v[x][n][2][k], sel);
                                }
                            }
                            const half8v vh = operand(hi[0], hi[1], hi[2], hi[3]);
                            if constexpr (EXACT) {
                                if constexpr (Q4) acc[b][c2] = mfma(operand(lo[0], lo[1], lo[2], lo[3]), ph[y], acc[b][c2]);
                                acc[b][c2] = mfma(vh, pl[y], acc[b][c2]);
                            }
                            acc[b][c2] = mfma(vh, ph[y], acc[b][c2]);
                        }
                    }
                }
                if constexpr (kEarly) {
                    fetch_values();
                } else if (more) {
                    locate(step + kWaves);
                    find(step + 2 * kWaves);
                }
            }
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);

            // the waves' parts are joined, 128 values at a time, in their order
            if (g == 0) {
                stats[wave][i][0] = mx.m;
                stats[wave][i][1] = l;
            }
            __syncthreads();  // (and all have their queries: their place is taken)
            const int oc = static_cast<int>(threadIdx.x) / 16, od = static_cast<int>(threadIdx.x) % 16 * 8;
            const uint32_t out_c = c0 + oc, out_j = over(out_c, a.group), out_head = h * a.group.d + (out_c - out_j * a.group.d);
            float top = -__builtin_inff(), mine_top = -__builtin_inff(), sum = 0;
            for (int w = 0; w < kWaves; ++w) {
                top = __builtin_fmaxf(top, stats[w][oc][0]);
                mine_top = __builtin_fmaxf(mine_top, stats[w][i][0]);
            }
            for (int w = 0; w < kWaves; ++w) sum += stats[w][oc][1] * weight(stats[w][oc][0], top);
            const float f = weight(mx.m, mine_top);
            const float inv = sum == 0 ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                if (n != 0) __syncthreads();
#pragma unroll
                for (int k = 0; k < GS; ++k) {
                    const int b = n * GS + k;
                    float4v lo, hi;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        lo[2 * r] = acc[b][0][r] * f;
                        lo[2 * r + 1] = acc[b][1][r] * f;
                        hi[2 * r] = acc[b][0][r + 2] * f;
                        hi[2 * r + 1] = acc[b][1][r + 2] * f;
                    }
                    *reinterpret_cast<float4v*>(&lds.merge[wave][i][32 * k + 8 * g]) = lo;
                    *reinterpret_cast<float4v*>(&lds.merge[wave][i][32 * k + 8 * g + 4]) = hi;
                }
                __syncthreads();
                if (od < 32 * GS && out_c < cols) {
                    float y[8];
                    for (int j = 0; j < 8; ++j) {
                        y[j] = lds.merge[0][oc][od + j];
                        for (int w = 1; w < kWaves; ++w) y[j] += lds.merge[w][oc][od + j];
                    }
                    const int d = 128 * n + od;
                    if (a.splits == 1) {
                        for (int j = 0; j < 8; ++j) y[j] = sum == 0 ? 0.0f : y[j] * inv;
                        char* op = row_ptr(a.out, sr.begin + out_j, out_head);
                        store8(op, a.out.type, (reinterpret_cast<uintptr_t>(op) & 15) == 0, d, y);
                    } else {
                        const size_t u = (static_cast<size_t>(sr.begin + out_j) * a.heads + out_head) * a.splits + blockIdx.x;
                        store8(a.part + u * HD, kTypeF32, true, d, y);
                        if (d == 0) {
                            float* ml = part_stats<HD>(a, sr.begin + out_j, out_head, blockIdx.x);
                            ml[0] = top;
                            ml[1] = sum;
                        }
                    }
                }
            }
            __syncthreads();  // the next columns' queries and statistics
        }
    }
}

// Joins few parts of a row's head: a wave for each.
constexpr uint32_t kFewSplits = 8;
__global__ __launch_bounds__(256) void k_paged_join_few(PagedAttnArgs a) {
    const uint32_t lane = threadIdx.x % 64, hd = a.kv.head_dim, splits = a.splits;
    const float* stats = a.part + static_cast<size_t>(a.b.rows) * a.heads * splits * hd;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        const uint32_t total = (sr.end - sr.begin) * a.heads;
        for (uint32_t u = blockIdx.x * 4 + threadIdx.x / 64; u < total; u += gridDim.x * 4) {
            const uint32_t row = over(u, a.per_row), head = u - row * a.heads;
            const size_t at = (static_cast<size_t>(sr.begin + row) * a.heads + head) * splits;
            float m[kFewSplits], l[kFewSplits], top = -__builtin_inff(), sum = 0;
#pragma unroll
            for (uint32_t p = 0; p < kFewSplits; ++p) {
                m[p] = p < splits ? stats[(at + p) * 2] : -__builtin_inff();
                l[p] = p < splits ? stats[(at + p) * 2 + 1] : 0.0f;
                top = __builtin_fmaxf(top, m[p]);
            }
#pragma unroll
            for (uint32_t p = 0; p < kFewSplits; ++p) {
                m[p] = m[p] == -__builtin_inff() && l[p] == 0 ? 0.0f : weight(m[p], top);
                sum += l[p] * m[p];
            }
            const float inv = 1.0f / sum;
            char* op = row_ptr(a.out, sr.begin + row, head);
            for (uint32_t d = lane; d < hd; d += 64) {
                float y = 0;
#pragma unroll
                for (uint32_t p = 0; p < kFewSplits; ++p) {
                    if (m[p] != 0) y += a.part[(at + p) * hd + d] * m[p];
                }
                y = sum == 0 ? 0.0f : y * inv;
                if (a.out.type == kTypeF32) reinterpret_cast<float*>(op)[d] = y;
                else reinterpret_cast<uint16_t*>(op)[d] = static_cast<uint16_t>(a.out.type == kTypeF16 ? to_half(y) : to_bf16(y));
            }
        }
    }
}

// Joins the parts of a row's head: a workgroup for each 32 dimensions, eight threads for each 32nd part, all of whose loads
// are on their way at once.  Parts without positions are not looked at.
constexpr uint32_t kMaxSplits = 256;
__global__ __launch_bounds__(256) void k_paged_join(PagedAttnArgs a) {
    constexpr uint32_t kParts = kMaxSplits / 32;
    __shared__ float tops[4], sums[4];
    __shared__ float4v joined[4][8];
    const uint32_t t = threadIdx.x, g = t / 8, wave = t / 64, hd = a.kv.head_dim, splits = a.splits;
    const uint32_t chunk = blockIdx.z, d = chunk * 32 + t % 8 * 4;
    const float* stats = a.part + static_cast<size_t>(a.b.rows) * a.heads * splits * hd;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        const uint32_t total = (sr.end - sr.begin) * a.heads;
        for (uint32_t u = blockIdx.x; u < total; u += gridDim.x) {
            const uint32_t row = over(u, a.per_row), head = u - row * a.heads;
            const size_t at = (static_cast<size_t>(sr.begin + row) * a.heads + head) * splits;
            float m[kParts], l[kParts], top = -__builtin_inff();
            float4v part[kParts];
#pragma unroll
            for (uint32_t k = 0; k < kParts; ++k) {
                const uint32_t p = g + 32 * k;
                m[k] = -__builtin_inff();
                l[k] = 0;
                part[k] = float4v{0, 0, 0, 0};
                if (p < splits) {
                    m[k] = stats[(at + p) * 2];
                    l[k] = stats[(at + p) * 2 + 1];
                    part[k] = *reinterpret_cast<const float4v*>(a.part + (at + p) * hd + d);
                }
                top = __builtin_fmaxf(top, m[k]);
            }
            for (int x = 8; x < 64; x *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, x));
            if (t % 64 == 0) tops[wave] = top;
            __syncthreads();
            for (int w = 0; w < 4; ++w) top = __builtin_fmaxf(top, tops[w]);
            float sum = 0;
            float4v y{0, 0, 0, 0};
#pragma unroll
            for (uint32_t k = 0; k < kParts; ++k) {
                if (m[k] == -__builtin_inff() && l[k] == 0) continue;
                const float f = weight(m[k], top);
                sum += l[k] * f;
                y += part[k] * f;
            }
            for (int x = 8; x < 64; x *= 2) {
                sum += __shfl_xor(sum, x);
                for (int j = 0; j < 4; ++j) y[j] += __shfl_xor(y[j], x);
            }
            if (t % 64 == 0) sums[wave] = sum;
            if (t % 64 < 8) joined[wave][t % 8] = y;
            __syncthreads();
            if (t < 8) {
                sum = sums[0] + sums[1] + sums[2] + sums[3];
                y = joined[0][t] + joined[1][t] + joined[2][t] + joined[3][t];
                const float inv = 1.0f / sum;
                char* op = row_ptr(a.out, sr.begin + row, head);
                for (int j = 0; j < 4; ++j) {
                    const float z = sum == 0 ? 0.0f : y[j] * inv;
                    if (a.out.type == kTypeF32) reinterpret_cast<float*>(op)[d + j] = z;
                    else reinterpret_cast<uint16_t*>(op)[d + j] = static_cast<uint16_t>(a.out.type == kTypeF16 ? to_half(z) : to_bf16(z));
                }
            }
            __syncthreads();
        }
    }
}

// Positions of a wave's step.
uint64_t step_of(const PagedKv& kv) { return static_cast<uint64_t>(kPair) * pairs_at_once(static_cast<int>(kv.head_dim / 32)); }

uint32_t most_rows(const PagedBatch& b) { return b.max_rows == 0 || b.max_rows > b.rows ? b.rows : b.max_rows; }

uint64_t column_tiles(const PagedKv& kv, const PagedBatch& b, uint32_t heads) {
    const uint64_t cols = static_cast<uint64_t>(most_rows(b)) * (heads / kv.kv_heads);
    return std::max<uint64_t>(1, (cols + kColumns - 1) / kColumns);
}

template <int NB, bool Q4>
hipError_t launch_typed(const PagedAttnArgs& a, dim3 grid, hipStream_t st) {
    if (a.q.type == kTypeF32 || a.out.type == kTypeF32) k_paged_attn<NB, Q4, true><<<grid, dim3(64 * kWaves), 0, st>>>(a);
    else k_paged_attn<NB, Q4, false><<<grid, dim3(64 * kWaves), 0, st>>>(a);
    return hipGetLastError();
}

template <int NB>
hipError_t launch_sized(const PagedAttnArgs& a, dim3 grid, hipStream_t st) {
    return a.kv.q4 ? launch_typed<NB, true>(a, grid, st) : launch_typed<NB, false>(a, grid, st);
}

}  // namespace

// The longest stretch of positions that a row's columns may see, as far as the host knows.
uint64_t longest(const PagedKv& kv, const PagedBatch& b, uint32_t window) {
    const uint64_t capacity = static_cast<uint64_t>(b.page_stride) * kv.page_tokens;
    const uint64_t length = b.max_length == 0 ? capacity : std::min<uint64_t>(b.max_length, capacity);
    return window == 0 ? length : std::min<uint64_t>(length, static_cast<uint64_t>(window) + most_rows(b));
}

// Prompts go to the kernel of many columns where those of a sequence fill half of its workgroup and there is enough to
// do: its workgroups start slowly (25 to 50 us), and 16 columns' fill the card at once.  Measured here and there, in us
// (without a window, since the workspace is sized before it is known): 128 rows of 8000 positions, 16 heads of 128
// in 4 bits 57 and 40, 300 rows 95 and 106; 100 rows of 20000, 32 heads of 64 64 and 90; 1500 rows of 1500 57 and 51;
// 1000 rows of 4000, 8 heads of 256 93 and 93; 32-bit, 1000 rows of 3000, 16 heads of 128 88 and 71.
bool is_prompt(const PagedKv& kv, const PagedBatch& b, uint32_t heads, bool exact) {
    const uint64_t length = longest(kv, b, 0), seen = length - std::min<uint64_t>(length, most_rows(b)) / 2;  // on average
    const double work = static_cast<double>(b.rows) * heads * kv.head_dim * static_cast<double>(seen);
    return prompt_fits(kv.head_dim, exact) && work >= (exact ? 7e9 : 3.5e9) &&
           static_cast<uint64_t>(most_rows(b)) * (heads / kv.kv_heads) * 2 >= prompt_columns(kv.head_dim, exact);
}

uint32_t paged_splits(const PagedKv& kv, const PagedBatch& b, uint32_t heads, bool exact, uint32_t window) {
    const bool prompt = is_prompt(kv, b, heads, exact);
    const uint64_t wide = prompt_columns(kv.head_dim, exact), cols = static_cast<uint64_t>(most_rows(b)) * (heads / kv.kv_heads);
    const uint64_t blocks = static_cast<uint64_t>(b.seqs) * kv.kv_heads * (prompt ? (cols + wide - 1) / wide : column_tiles(kv, b, heads));
    // As many workgroups as are resident at once: each costs about 9 us before and after its positions.  Where there are
    // that many without, one for each 8192 positions, so that a long sequence among short ones does not run alone, of
    // 256 MB at most.
    const uint64_t target = 256 * resident(static_cast<int>(kv.head_dim / 32)), most = longest(kv, b, window);
    const uint64_t least = prompt ? 512 : kWaves * step_of(kv), useful = (most + least - 1) / least;
    const uint64_t room = (uint64_t{1} << 26) / (std::max<uint64_t>(b.rows, 1) * heads * (kv.head_dim + 2));
    // Prompts: one workgroup a CU, or, where those of 128 columns see more and more, two: 5000 rows of 5000 positions,
    // 4 heads of 256, 146 us for 256, and 2000 of 4000 146 for 138.
    const uint64_t cus = wide == 128 && window == 0 ? 512 : 256;
    const uint64_t wanted = prompt ? cus / blocks : std::max<uint64_t>(target / blocks, std::min<uint64_t>((most + 8191) / 8192, room));
    // A few steps of a wave cost less than the join (a token of 16 heads of 128 at 333: 9.6 us a call in one part, 11.5 in three, at 500 10 and 11,
    // at 1000 13 and 11; heads of 256 in 4 bits at 200 12 and 13, at 500 15.5 and 13.4).
    if (!prompt && useful <= (kv.head_dim <= 128 ? 4 : 2)) return 1;
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(std::min(useful, wanted), kMaxSplits)));
}

size_t paged_workspace(const PagedKv& kv, const PagedBatch& b, uint32_t heads) {
    const size_t splits = std::max(paged_splits(kv, b, heads, false, 0), paged_splits(kv, b, heads, true, 0));
    return splits == 1 ? 0 : static_cast<size_t>(b.rows) * heads * splits * (kv.head_dim + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttnArgs& args, hipStream_t st) {
    PagedAttnArgs a = args;
    const bool exact = a.q.type == kTypeF32 || a.out.type == kTypeF32, prompt = is_prompt(a.kv, a.b, a.heads, exact);
    a.splits = paged_splits(a.kv, a.b, a.heads, exact, a.window);
    const uint64_t steps = longest(a.kv, a.b, a.window) / step_of(a.kv) + 1;
    a.per = static_cast<int32_t>(std::min<uint64_t>((steps + a.splits - 1) / a.splits, kMaxLength / kPair / a.splits));
    const uint64_t tiles = std::min<uint64_t>(column_tiles(a.kv, a.b, a.heads), 65535 / a.kv.kv_heads);
    const dim3 grid(a.splits, static_cast<uint32_t>(tiles * a.kv.kv_heads), std::min<uint32_t>(a.b.seqs, 65535));
    hipError_t e = hipErrorInvalidValue;
    if (prompt) e = launch_paged_prompt(a, exact, most_rows(a.b), st);
    else switch (a.kv.head_dim / 32) {
        case 2: e = launch_sized<2>(a, grid, st); break;
        case 3: e = launch_sized<3>(a, grid, st); break;
        case 4: e = launch_sized<4>(a, grid, st); break;
        case 8: e = launch_sized<8>(a, grid, st); break;
        case 16: e = launch_sized<16>(a, grid, st); break;
    }
    if (e != hipSuccess || a.splits == 1) return e;
    const uint64_t y = std::min<uint64_t>(a.b.seqs, 65535), x = static_cast<uint64_t>(most_rows(a.b)) * a.heads;
    const uint64_t most = std::max<uint64_t>(1, 65536 / y);
    // (a token's 16 heads in five parts: 5.8 us by workgroups, 8.8 by waves; 2048 in two: 12.5 and 5.2)
    if (a.splits <= kFewSplits && x * y >= 1024) {
        k_paged_join_few<<<dim3(static_cast<uint32_t>(std::min((x + 3) / 4, most)), static_cast<uint32_t>(y)), dim3(256), 0, st>>>(a);
    } else {
        k_paged_join<<<dim3(static_cast<uint32_t>(std::min(x, most)), static_cast<uint32_t>(y), a.kv.head_dim / 32), dim3(256), 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace bh
