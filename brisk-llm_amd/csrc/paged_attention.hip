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
constexpr int kStep = 32;        // positions a wave takes at a time: two tiles
constexpr int kColumns = 16;     // (row, head) pairs of a key/value head that share a pass
// Probabilities are held as 2^kLift p relative to a maximum that is renewed once it is passed by
// 2^kLazy: at most 2^15 as halves, and those of a half's smallest steps 2^-31 of the largest.
constexpr float kLazy = 8.0f, kLift = 7.0f;
constexpr int kMergeRow = 132;   // LDS floats a column, for 128 values: 16-byte rows, shifted over the banks

__device__ inline half8v operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(half8v, word4v{a, b, c, d}); }
__device__ inline float4v mfma(half8v a, half8v b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline uint32_t bits(half2v x) { return __builtin_bit_cast(uint32_t, x); }
__device__ inline half2v halves(uint32_t x) { return __builtin_bit_cast(half2v, x); }

// Codes less 8 of nibbles 0 and 4 (of 1 and 5, when `high`) of a word: a code in the low bits of a
// half's significand is 1024 + n, four bits up it is 64 + n; taking the rest off is exact.
__device__ inline half2v codes(uint32_t w, bool high) {
    return high ? halves((w & 0x00F000F0) | 0x54005400) - half2v{72, 72} : halves((w & 0x000F000F) | 0x64006400) - half2v{1032, 1032};
}

// Whether halves of a word are infinities or NaN, or as 4-bit scales past kMaxScale: then bit 15 or 31 of the
// result is set, by the carry out of the exponent (exponents of 31 all ones, of 28 on for a scale).
template <bool SCALE>
__device__ inline uint32_t ill(uint32_t w) { return (w & 0x7FFF7FFF) + (SCALE ? 0x10001000 : 0x04000400); }
constexpr uint32_t kIll = 0x80008000;
template <bool SCALE>
__device__ inline uint32_t without_ill(uint32_t w) {
    const uint32_t x = ill<SCALE>(w);
    return w & ((x & 0x8000 ? 0 : 0xFFFF) | (x & 0x80000000 ? 0 : 0xFFFF0000));
}

template <int N>
struct alignas(N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4) Words {
    uint32_t w[N];
};
template <int N>
__device__ inline void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    const Words<N> x = *reinterpret_cast<const Words<N>*>(p);
    for (int k = 0; k < N; ++k) w[k] = x.w[k];
}

// EXACT: queries and probabilities as sums of two halves, and 4-bit values as sums of two: 32-bit results.
template <int NB, bool Q4, bool EXACT>
__global__ __launch_bounds__(64 * kWaves) void k_paged_attn(PagedAttnArgs a) {
    constexpr int GS = NB < 4 ? NB : 4, NG = NB / GS, HD = 32 * NB;
    __shared__ float merge[kWaves][kColumns][kMergeRow];
    __shared__ float stats[kWaves][kColumns][2];
    const int lane = static_cast<int>(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int i = lane % 16, g = lane / 16;
    const uint32_t h = blockIdx.y % a.kv.kv_heads, first_tile = blockIdx.y / a.kv.kv_heads, tiles = gridDim.y / a.kv.kv_heads;
    const int64_t window = a.window;

    for (uint32_t s = blockIdx.z; s < a.b.seqs; s += gridDim.z) {
        const SeqRows sr = seq_rows(a.b, s);
        const int64_t cols = (sr.end - sr.begin) * a.group;
        for (int64_t ct = first_tile; ct * kColumns < cols; ct += tiles) {
            const int64_t c = ct * kColumns + i, last = std::min<int64_t>(ct * kColumns + kColumns, cols) - 1;
            const bool mine = c < cols;
            const int64_t row = sr.begin + (mine ? c / a.group : 0);
            const int64_t head = static_cast<int64_t>(h) * a.group + (mine ? c % a.group : 0);
            const int64_t pos_lo = sr.first + ct * kColumns / a.group, pos_hi = sr.first + last / a.group;
            const int64_t pos = mine ? sr.first + (row - sr.begin) : pos_lo;
            const int64_t t_lo = window != 0 && pos_lo - window + 1 > 0 ? pos_lo - window + 1 : 0;
            const int64_t t_hi = std::min<int64_t>(pos_hi + 1, static_cast<int64_t>(a.b.page_stride) << a.kv.page_shift);
            const int64_t step_lo = t_lo / kStep, steps = t_hi > t_lo ? (t_hi + kStep - 1) / kStep - step_lo : 0;
            const int64_t per = (steps + a.splits - 1) / a.splits;
            const int64_t step_end = step_lo + std::min<int64_t>(steps, per * (blockIdx.x + 1));

            // the column's query, scaled by a power of two where its type has more range than a half
            half8v qh[NB], ql[EXACT ? NB : 1];
            float qscale = a.scale * 1.44269504088896f;
            {
                const char* qp = row_ptr(a.q, row, head);
                const bool vec = (reinterpret_cast<uintptr_t>(qp) & 15) == 0;
                float top = 0;
                float x[NB][8];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    load8(qp, a.q.type, vec, 32 * b + 8 * g, x[b]);
                    for (int j = 0; j < 8; ++j) {
                        if (!mine) x[b][j] = 0;
                        top = __builtin_fmaxf(top, __builtin_fabsf(x[b][j]));
                    }
                }
                int e = 9;
                if (a.q.type != kTypeF16) {
                    top = __builtin_fmaxf(top, __shfl_xor(top, 16));
                    top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                    if (top > 0 && top <= 3.402823466e38f) e = __builtin_amdgcn_frexp_expf(top);
                }
                qscale = __builtin_ldexpf(qscale, e - 9);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    for (int j = 0; j < 8; ++j) {
                        const float y = __builtin_ldexpf(x[b][j], 9 - e);
                        qh[b][j] = static_cast<_Float16>(y);
                        if constexpr (EXACT) ql[b][j] = static_cast<_Float16>(y - static_cast<float>(qh[b][j]));
                    }
                }
            }

            float m = -__builtin_inff(), l = 0;
            float4v acc[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b][0] = acc[b][1] = float4v{0, 0, 0, 0};

            for (int64_t step = step_lo + per * blockIdx.x + wave; step < step_end; step += kWaves) {
                const int64_t t0 = step * kStep;
                const uint8_t* tile[2];
                bool there[2];
                float4v sc[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int64_t page = page_of(a.kv, a.b, s, t0 + 16 * x);
                    there[x] = page >= 0;
                    tile[x] = a.kv.data + tile_at(a.kv, page < 0 ? 0 : page, h, t0 + 16 * x);
                    float4v sum{0, 0, 0, 0};
                    if constexpr (Q4) {
#pragma unroll
                        for (int n = 0; n < NG; ++n) {
                            uint32_t w[GS];
                            load_words<GS>(tile[x] + (n * 64 + lane) * GS * 4, w);
#pragma unroll
                            for (int k = 0; k < GS; ++k) {
                                const int b = n * GS + k;
                                const half8v kx = operand(bits(codes(w[k], false)), bits(codes(w[k], true)), bits(codes(w[k] >> 8, false)),
                                                          bits(codes(w[k] >> 8, true)));
                                float4v d{0, 0, 0, 0};
                                if constexpr (EXACT) d = mfma(kx, ql[b], d);
                                d = mfma(kx, qh[b], d);
                                const word2v ks = *reinterpret_cast<const word2v*>(tile[x] + tile_key_scales_at(NB) + (g * NB + b) * 8);
                                sum[0] = __builtin_fmaf(d[0], from_half(ks[0] & 0xFFFF), sum[0]);
                                sum[1] = __builtin_fmaf(d[1], from_half(ks[0] >> 16), sum[1]);
                                sum[2] = __builtin_fmaf(d[2], from_half(ks[1] & 0xFFFF), sum[2]);
                                sum[3] = __builtin_fmaf(d[3], from_half(ks[1] >> 16), sum[3]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const half8v kx = __builtin_bit_cast(half8v, *reinterpret_cast<const word4v*>(tile[x] + (b * 64 + lane) * 16));
                            if constexpr (EXACT) sum = mfma(kx, ql[b], sum);
                            sum = mfma(kx, qh[b], sum);
                        }
                    }
                    sc[x] = sum;
                }
                // positions t0 .. t0 + 31 that every column sees need no masks
                const bool full = there[0] && there[1] && t0 + kStep - 1 <= pos_lo && (window == 0 || t0 > pos_hi - window);
                float p[8];
                uint32_t seen = 0xFF;
                float top = -__builtin_inff();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = sc[j / 4][j % 4] * qscale;
                    if (!full) {
                        const int64_t t = t0 + 16 * (j / 4) + 4 * g + j % 4;
                        if (!(there[j / 4] && t <= pos && (window == 0 || t > pos - window))) {
                            p[j] = -__builtin_inff();
                            seen &= ~(1u << j);
                        }
                    }
                    top = __builtin_fmaxf(top, p[j]);
                }
                if (__any(top > m + kLazy)) {
                    top = __builtin_fmaxf(top, __shfl_xor(top, 16));
                    top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                    const float next = __builtin_fmaxf(m, top);
                    const float f = __builtin_amdgcn_exp2f(m - (next == -__builtin_inff() ? 0.0f : next));
                    m = next;
                    l *= f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        acc[b][0] *= f;
                        acc[b][1] *= f;
                    }
                }
                const float base = m == -__builtin_inff() ? 0.0f : m - kLift;
                half8v ph, pl;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = __builtin_amdgcn_exp2f(p[j] - base);
                    l += p[j];
                    ph[j] = static_cast<_Float16>(p[j]);
                    if constexpr (EXACT) pl[j] = static_cast<_Float16>(p[j] - static_cast<float>(ph[j]));
                }
                // a value that is not finite, at a position that some column does not see: the product
                // is taken without it, and the columns that see it get it afterwards (4-bit: its whole block is NaN)
                bool poison = false;
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    uint32_t v[2][Q4 ? 1 : 4][GS], vs[2][Q4 ? 2 * GS : 1];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint8_t* at = tile[x] + tile_values_at(Q4, NB);
                        if constexpr (Q4) {
                            load_words<GS>(at + (n * 64 + lane) * GS * 4, v[x][0]);
                            load_words<2 * GS>(tile[x] + tile_value_scales_at(NB) + (g * NB + n * GS) * 8, vs[x]);
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r) load_words<GS>(at + ((r * NG + n) * 64 + lane) * GS * 4, v[x][r]);
                        }
                    }
                    // (with 32-bit results everywhere: an infinity times a probability's second part is of any sign)
                    if (!full || (EXACT && !Q4)) {
                        uint32_t found = 0;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if constexpr (Q4) {
                                for (int k = 0; k < 2 * GS; ++k) found |= ill<true>(vs[x][k]);
                            } else {
                                for (int r = 0; r < 4; ++r)
                                    for (int k = 0; k < GS; ++k) found |= ill<false>(v[x][r][k]);
                            }
                        }
                        if (__any((found & kIll) != 0)) {
                            poison = true;
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                if constexpr (Q4) {
                                    for (int k = 0; k < 2 * GS; ++k) vs[x][k] = without_ill<true>(vs[x][k]);
                                } else {
                                    for (int r = 0; r < 4; ++r)
                                        for (int k = 0; k < GS; ++k) v[x][r][k] = without_ill<false>(v[x][r][k]);
                                }
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
                                    const half2v c01 = codes(v[x][0][k], c2), c23 = codes(v[x][0][k] >> 8, c2);
                                    const half2v d01 = halves(vs[x][2 * k]), d23 = halves(vs[x][2 * k + 1]);
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
                                    hi[2 * x] = __builtin_amdgcn_perm(v[x][1][k], v[x][0][k], sel);
                                    hi[2 * x + 1] = __builtin_amdgcn_perm(v[x][3][k], v[x][2][k], sel);
                                }
                            }
                            const half8v vh = operand(hi[0], hi[1], hi[2], hi[3]);
                            if constexpr (EXACT) {
                                if constexpr (Q4) acc[b][c2] = mfma(operand(lo[0], lo[1], lo[2], lo[3]), ph, acc[b][c2]);
                                acc[b][c2] = mfma(vh, pl, acc[b][c2]);
                            }
                            acc[b][c2] = mfma(vh, ph, acc[b][c2]);
                        }
                    }
                }
                if (poison) {
                    for (int j = 0; j < 8; ++j) {
                        for (int gg = 0; gg < 4; ++gg) {
                            const float pt = __shfl(p[j], i + 16 * gg);
                            const bool sees = __shfl(seen, i + 16 * gg) >> j & 1;
                            const uint32_t token = 4 * gg + j % 4;
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                float x[8];
                                read8(tile[j / 4], Q4, NB, true, token, 32 * b + 8 * g, x);
#pragma unroll
                                for (int y = 0; y < 8; ++y) {
                                    if (sees && !(__builtin_fabsf(x[y]) <= 3.402823466e38f)) acc[b][y % 2][y / 2] += pt * x[y];
                                }
                            }
                        }
                    }
                }
            }
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);

            // the waves' parts are joined, 128 values at a time, in their order
            if (g == 0) {
                stats[wave][i][0] = m;
                stats[wave][i][1] = l;
            }
            __syncthreads();
            const int oc = static_cast<int>(threadIdx.x) / 16, od = static_cast<int>(threadIdx.x) % 16 * 8;
            const int64_t out_c = ct * kColumns + oc;
            float top = -__builtin_inff(), mine_top = -__builtin_inff(), sum = 0;
            for (int w = 0; w < kWaves; ++w) {
                top = __builtin_fmaxf(top, stats[w][oc][0]);
                mine_top = __builtin_fmaxf(mine_top, stats[w][i][0]);
            }
            const float base = top == -__builtin_inff() ? 0.0f : top;
            for (int w = 0; w < kWaves; ++w) sum += stats[w][oc][1] * __builtin_amdgcn_exp2f(stats[w][oc][0] - base);
            const float f = __builtin_amdgcn_exp2f(m - (mine_top == -__builtin_inff() ? 0.0f : mine_top));
            const int64_t out_row = sr.begin + out_c / a.group, out_head = static_cast<int64_t>(h) * a.group + out_c % a.group;
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
                    *reinterpret_cast<float4v*>(&merge[wave][i][32 * k + 8 * g]) = lo;
                    *reinterpret_cast<float4v*>(&merge[wave][i][32 * k + 8 * g + 4]) = hi;
                }
                __syncthreads();
                if (od < 32 * GS && out_c < cols) {
                    float y[8];
                    for (int j = 0; j < 8; ++j) {
                        y[j] = merge[0][oc][od + j];
                        for (int w = 1; w < kWaves; ++w) y[j] += merge[w][oc][od + j];
                    }
                    const int d = 128 * n + od;
                    if (a.splits == 1) {
                        const float inv = sum == 0 ? 0.0f : 1.0f / sum;
                        for (int j = 0; j < 8; ++j) y[j] = sum == 0 ? 0.0f : y[j] * inv;
                        char* op = row_ptr(a.out, out_row, out_head);
                        store8(op, a.out.type, (reinterpret_cast<uintptr_t>(op) & 15) == 0, d, y);
                    } else {
                        const size_t u = (static_cast<size_t>(out_row) * a.heads + out_head) * a.splits + blockIdx.x;
                        store8(a.part + u * HD, kTypeF32, true, d, y);
                        if (d == 0) {
                            float* ml = a.part + static_cast<size_t>(a.b.rows) * a.heads * a.splits * HD + u * 2;
                            ml[0] = top;
                            ml[1] = sum;
                        }
                    }
                }
            }
            __syncthreads();  // the next columns' statistics
        }
    }
}

// Joins the parts of a row's head, in their order: one wave each.
__global__ __launch_bounds__(256) void k_paged_join(PagedAttnArgs a) {
    const int lane = static_cast<int>(threadIdx.x) % 64, wave = static_cast<int>(threadIdx.x) / 64, hd = static_cast<int>(a.kv.head_dim);
    const float* stats = a.part + static_cast<size_t>(a.b.rows) * a.heads * a.splits * hd;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        const int64_t total = (sr.end - sr.begin) * a.heads;
        for (int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + wave; u < total; u += static_cast<int64_t>(gridDim.x) * 4) {
            const int64_t row = sr.begin + u / a.heads, head = u % a.heads;
            const size_t at = (static_cast<size_t>(row) * a.heads + head) * a.splits;
            float top = -__builtin_inff();
            for (uint32_t p = 0; p < a.splits; ++p) top = __builtin_fmaxf(top, stats[(at + p) * 2]);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            float sum = 0;
            for (uint32_t p = 0; p < a.splits; ++p) sum += stats[(at + p) * 2 + 1] * __builtin_amdgcn_exp2f(stats[(at + p) * 2] - base);
            for (int d = lane; d < hd; d += 64) {
                float y = 0;
                for (uint32_t p = 0; p < a.splits; ++p) y += a.part[(at + p) * hd + d] * __builtin_amdgcn_exp2f(stats[(at + p) * 2] - base);
                y = sum == 0 ? 0.0f : y / sum;
                char* op = row_ptr(a.out, row, head);
                if (a.out.type == kTypeF32) reinterpret_cast<float*>(op)[d] = y;
                else reinterpret_cast<uint16_t*>(op)[d] = static_cast<uint16_t>(a.out.type == kTypeF16 ? to_half(y) : to_bf16(y));
            }
        }
    }
}

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

uint32_t paged_splits(const PagedKv& kv, const PagedBatch& b, uint32_t heads) {
    const uint64_t blocks = static_cast<uint64_t>(b.seqs) * kv.kv_heads * column_tiles(kv, b, heads);
    const uint64_t capacity = static_cast<uint64_t>(b.page_stride) * kv.page_tokens;
    const uint64_t length = b.max_length == 0 ? capacity : std::min<uint64_t>(b.max_length, capacity);
    const uint64_t useful = (length + kWaves * kStep - 1) / (kWaves * kStep);
    const uint64_t wanted = (1024 + blocks - 1) / blocks;
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(std::min(useful, wanted), 256)));
}

size_t paged_workspace(const PagedKv& kv, const PagedBatch& b, uint32_t heads) {
    const size_t splits = paged_splits(kv, b, heads);
    return splits == 1 ? 0 : static_cast<size_t>(b.rows) * heads * splits * (kv.head_dim + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t st) {
    const uint64_t tiles = std::min<uint64_t>(column_tiles(a.kv, a.b, a.heads), 65535 / a.kv.kv_heads);
    const dim3 grid(a.splits, static_cast<uint32_t>(tiles * a.kv.kv_heads), std::min<uint32_t>(a.b.seqs, 65535));
    hipError_t e = hipErrorInvalidValue;
    switch (a.kv.head_dim / 32) {
        case 2: e = launch_sized<2>(a, grid, st); break;
        case 3: e = launch_sized<3>(a, grid, st); break;
        case 4: e = launch_sized<4>(a, grid, st); break;
        case 8: e = launch_sized<8>(a, grid, st); break;
        case 16: e = launch_sized<16>(a, grid, st); break;
    }
    if (e != hipSuccess || a.splits == 1) return e;
    const uint64_t y = std::min<uint64_t>(a.b.seqs, 65535), x = (static_cast<uint64_t>(most_rows(a.b)) * a.heads + 3) / 4;
    const uint64_t most = std::max<uint64_t>(1, 65536 / y);
    k_paged_join<<<dim3(static_cast<uint32_t>(std::min(x, most)), static_cast<uint32_t>(y)), dim3(256), 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace bh
