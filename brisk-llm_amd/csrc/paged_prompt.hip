// Attention of prompts over their pages: many rows of a sequence at once.
//
// As in paged_attention.hip the product's sides are swapped, S^T = K Q^T and O^T = V^T P^T, here with
// v_mfma_f32_32x32x16_f16 (twice the rate of the 16-wide one: 2.08 against 1.14 PFLOP/s measured), and
// a lane's probabilities are its second product's operand as they stand.  Keys and values pass through
// LDS, 64 positions at a time, as halves in operand order: a tile is unpacked once for the workgroup's
// columns, and an operand is one conflict-free 16-byte read of a lane.
#include <algorithm>

#include "paged.h"
#include "paged_device.h"

namespace bh {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = 64;  // positions in LDS at a time: a tile for each wave to unpack
constexpr int kWide = 32;   // columns of a product

// What a thread holds of its wave's tile until it goes to LDS.
template <int NB, bool Q4>
struct RawTile {
    static constexpr int GS = NB < 4 ? NB : 4, NG = NB / GS;
    uint32_t k[NG][Q4 ? GS : 4 * GS], v[NG][Q4 ? 1 : 4][GS], vs[NG][Q4 ? 2 * GS : 1];
    uint16_t ks[Q4 ? NB : 1];

    __device__ inline void load(const uint8_t* tile, int lane) {
        const uint8_t* at = tile + tile_values_at(Q4, NB);
        const int i = lane % 16, g = lane / 16;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if constexpr (Q4) {
                load_words<GS>(tile + (n * 64 + lane) * GS * 4, k[n]);
                load_words<GS>(at + (n * 64 + lane) * GS * 4, v[n][0]);
                load_words<2 * GS>(tile + tile_value_scales_at(NB) + (g * NB + n * GS) * 8, vs[n]);
            } else {
#pragma unroll
                for (int j = 0; j < GS; ++j) {
                    const word4v w = *reinterpret_cast<const word4v*>(tile + ((n * GS + j) * 64 + lane) * 16);
                    for (int e = 0; e < 4; ++e) k[n][4 * j + e] = w[e];
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) load_words<GS>(at + ((r * NG + n) * 64 + lane) * GS * 4, v[n][r]);
            }
        }
        if constexpr (Q4) {
#pragma unroll
            for (int b = 0; b < NB; ++b) ks[b] = *reinterpret_cast<const uint16_t*>(tile + tile_key_scales_at(NB) + ((i / 4 * NB + b) * 4 + i % 4) * 2);
        }
    }

    // The values of positions 4 g + r whose bit r of `keep` is not set become zeros.
    __device__ inline void keep_values(uint32_t keep) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if constexpr (Q4) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t b = keep >> (2 * j), mask = (b & 1 ? 0xFFFF : 0) | (b & 2 ? 0xFFFF0000 : 0);
                    for (int e = 0; e < GS; ++e) vs[n][2 * e + j] &= mask;
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t mask = keep >> r & 1 ? 0xFFFFFFFF : 0;
                    for (int e = 0; e < GS; ++e) v[n][r][e] &= mask;
                }
            }
        }
    }
    // Whether an infinity or NaN is among the values.
    __device__ inline bool any_ill() const {
        uint32_t found = 0;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if constexpr (Q4) {
                for (int e = 0; e < 2 * GS; ++e) found |= ill<true>(vs[n][e]);
            } else {
                for (int r = 0; r < 4; ++r)
                    for (int e = 0; e < GS; ++e) found |= ill<false>(v[n][r][e]);
            }
        }
        return __any((found & kIll) != 0);
    }
    __device__ inline void drop_ill() {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if constexpr (Q4) {
                for (int e = 0; e < 2 * GS; ++e) vs[n][e] = scale_marks(vs[n][e]).rest;
            } else {
                for (int r = 0; r < 4; ++r)
                    for (int e = 0; e < GS; ++e) v[n][r][e] = marks(v[n][r][e]).rest;
            }
        }
    }
};

template <int NB>
struct BlockLds {
    // operands [32 positions][16 dimensions] and [32 dimensions][16 positions], 64 lanes x 16 bytes each
    word4v k[kBlock / 32][2 * NB][64];
    word4v v[NB][kBlock / 16][64];
    int there[kWaves], poison[kWaves];  // whether a tile is there, and holds values that are not finite (here they are zeros)
};

// Unpacks tile x of the block.  4-bit values are rounded to halves as codes times scales: 2^-11 of a
// value at most, as the probabilities are.
template <int NB, bool Q4>
__device__ inline void unpack(const RawTile<NB, Q4>& raw, BlockLds<NB>& out, int x, int lane) {
    constexpr int GS = NB < 4 ? NB : 4;
    const int i = lane % 16, g = lane / 16;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int n = b / GS, e = b % GS;
        word4v key;
        if constexpr (Q4) {
            const uint32_t w = raw.k[n][e], w8 = w >> 8;
            const half2v d = halves(raw.ks[b] | static_cast<uint32_t>(raw.ks[b]) << 16);
            key = word4v{bits(codes(w, false) * d), bits(codes(w, true) * d), bits(codes(w8, false) * d), bits(codes(w8, true) * d)};
        } else {
            key = word4v{raw.k[n][4 * e], raw.k[n][4 * e + 1], raw.k[n][4 * e + 2], raw.k[n][4 * e + 3]};
        }
        out.k[x / 2][2 * b + g / 2][g % 2 * 32 + x % 2 * 16 + i] = key;
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
            word2v val;
            if constexpr (Q4) {
                const uint32_t w = raw.v[n][0][e];
                val[0] = bits(codes(w, c2) * halves(raw.vs[n][2 * e]));
                val[1] = bits(codes(w >> 8, c2) * halves(raw.vs[n][2 * e + 1]));
            } else {
                const uint32_t sel = c2 ? 0x07060302 : 0x05040100;
                val[0] = __builtin_amdgcn_perm(raw.v[n][1][e], raw.v[n][0][e], sel);
                val[1] = __builtin_amdgcn_perm(raw.v[n][3][e], raw.v[n][2][e], sel);
            }
            reinterpret_cast<word2v*>(&out.v[b][x][g % 2 * 32 + 2 * i + c2])[g / 2] = val;
        }
    }
}

// A workgroup of four waves takes CT x 128 columns, (row, head) pairs of one key/value head, each wave
// CT x 32 of them, and one part of the positions.  Without a window a wave's two sets of columns are one from the
// front of the prompt and its mirror image from the back: what two sets see adds up to the same for all.
template <int NB, int CT, bool Q4>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(1))) void k_paged_prompt(PagedAttnArgs a) {
    constexpr int HD = 32 * NB;
    __shared__ union {
        BlockLds<NB> block[2];
        _Float16 q[kWaves][kWide][HD + 8];
        float out[kWaves][kWide][HD + 4];
    } lds;
    const int lane = static_cast<int>(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int col = lane % 32, half = lane / 32;
    const uint32_t h = blockIdx.x, split = blockIdx.y % a.splits, first_set = blockIdx.y / a.splits, set_step = gridDim.y / a.splits;
    const int32_t window = a.window > static_cast<uint32_t>(kMaxLength) ? 0 : static_cast<int32_t>(a.window);
    const int32_t capacity = static_cast<int32_t>(std::min<int64_t>(kMaxLength, static_cast<int64_t>(a.b.page_stride) << a.kv.page_shift));

    for (uint32_t s = blockIdx.z; s < a.b.seqs; s += gridDim.z) {
        const SeqRows sr = seq_rows(a.b, s);
        const uint32_t cols = (sr.end - sr.begin) * a.group.d, tiles = (cols + kWide - 1) / kWide;
        const bool mirrored = CT == 2 && window == 0;
        const uint32_t halves_of = mirrored ? (tiles + 1) / 2 : (tiles + CT - 1) / CT;  // pairs of sets
        for (uint32_t set = first_set; set * kWaves < halves_of; set += set_step) {
            // the wave's columns
            const uint32_t pair = set * kWaves + wave;
            uint32_t tile[CT];
            int32_t pos_lo[CT], pos_hi[CT], t_lo[CT], t_hi[CT], pos[CT];
            const auto range = [&](uint32_t t, int32_t& plo, int32_t& phi, int32_t& tlo, int32_t& thi) {
                const uint32_t last = std::min<uint32_t>((t + 1) * kWide, cols) - 1;
                plo = sr.first + static_cast<int32_t>(over(t * kWide, a.group));
                phi = sr.first + static_cast<int32_t>(over(last, a.group));
                tlo = window != 0 && plo - window + 1 > 0 ? plo - window + 1 : 0;
                thi = std::min(phi + 1, capacity);
            };
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                tile[c] = mirrored && c == 1 ? tiles - 1 - pair : CT * pair * (mirrored ? 0 : 1) + (mirrored ? pair : c);
                const bool live = pair < halves_of && tile[c] < tiles && !(c == 1 && tile[c] == tile[0]);
                pos_lo[c] = pos_hi[c] = t_lo[c] = t_hi[c] = 0;
                if (live) range(tile[c], pos_lo[c], pos_hi[c], t_lo[c], t_hi[c]);
                else tile[c] = tiles;
                const uint32_t cc = tile[c] * kWide + col;
                pos[c] = cc < cols ? sr.first + static_cast<int32_t>(over(cc, a.group)) : pos_lo[c];
            }
            // the workgroup's positions: from its first set's to its last one's
            int32_t wg_lo, wg_plo, wg_phi, wg_hi, unused_lo, unused_hi, unused;
            {
                const uint32_t p0 = set * kWaves, p1 = std::min(p0 + kWaves, halves_of) - 1;
                const uint32_t front = mirrored ? p0 : CT * p0, back = mirrored ? tiles - 1 - p0 : std::min<uint32_t>(CT * p1 + CT - 1, tiles - 1);
                range(front, wg_plo, unused, wg_lo, unused_hi);
                range(back, unused, wg_phi, unused_lo, wg_hi);
            }
            const int32_t blk_lo = wg_lo / kBlock, blocks = wg_hi > wg_lo ? (wg_hi + kBlock - 1) / kBlock - blk_lo : 0;
            const int32_t per = (blocks + static_cast<int32_t>(a.splits) - 1) / static_cast<int32_t>(a.splits);
            const int32_t blk_begin = blk_lo + static_cast<int32_t>(std::min<int64_t>(blocks, static_cast<int64_t>(per) * split));
            const int32_t blk_end = blk_lo + static_cast<int32_t>(std::min<int64_t>(blocks, static_cast<int64_t>(per) * (split + 1)));

            RawTile<NB, Q4> raw;
            bool there = false;
            const auto fetch = [&](int32_t blk) {
                const int32_t t = blk * kBlock + 16 * wave, page = page_of(a.kv, a.b, s, t);
                there = page >= 0;
                raw.load(a.kv.data + tile_at(a.kv, there ? page : 0, h, t), lane);
            };
            const auto put = [&](int32_t blk) {
                const int32_t t = blk * kBlock + 16 * wave + 4 * (lane / 16);
                // some column does not see all of the block: what none sees is left out
                if (!there || (blk + 1) * kBlock - 1 > wg_plo || (window != 0 && blk * kBlock <= wg_phi - window)) {
                    uint32_t keep = 0;
                    for (int r = 0; r < 4; ++r) keep |= there && t + r >= wg_lo && t + r <= wg_phi ? 1u << r : 0;
                    raw.keep_values(keep);
                }
                const bool poison = raw.any_ill();
                if (__builtin_expect(poison, 0)) raw.drop_ill();
                BlockLds<NB>& out = lds.block[blk & 1];
                unpack<NB, Q4>(raw, out, wave, lane);
                if (lane == 0) {
                    out.there[wave] = there;
                    out.poison[wave] = poison;
                }
            };
            if (blk_begin < blk_end) fetch(blk_begin);

            // the columns' queries, through the wave's part of LDS: 16 lanes a column, scaled by a power of two where the
            // type has more range than a half
            __syncthreads();  // the blocks of the columns before
            half8v q[CT][2 * NB];
            float qscale[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const int sub = lane % 16;
#pragma unroll 1
                for (int r = lane / 16; r < kWide; r += 4) {
                    constexpr int K = (HD + 127) / 128;
                    const uint32_t cc = tile[c] * kWide + r;
                    const bool live = cc < cols;
                    const uint32_t row = live ? over(cc, a.group) : 0;
                    const char* qp = row_ptr(a.q, sr.begin + row, h * a.group.d + (live ? cc - row * a.group.d : 0));
                    float x[K][8], top = 0;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        for (int j = 0; j < 8; ++j) x[k][j] = 0;
                        const int d = (k * 16 + sub) * 8;
                        if (live && d < HD) load8(qp, a.q.type, (reinterpret_cast<uintptr_t>(qp) & 15) == 0, d, x[k]);
                        for (int j = 0; j < 8; ++j) top = __builtin_fmaxf(top, __builtin_fabsf(x[k][j]));
                    }
                    for (int n = 1; n < 16; n *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, n));
                    const int e = a.q.type != kTypeF16 && top > 0 && top <= 3.402823466e38f ? __builtin_amdgcn_frexp_expf(top) : 9;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const int d = (k * 16 + sub) * 8;
                        half8v y;
                        for (int j = 0; j < 8; ++j) y[j] = static_cast<_Float16>(__builtin_ldexpf(x[k][j], 9 - e));
                        if (d < HD) *reinterpret_cast<half8v*>(&lds.q[wave][r][d]) = y;
                    }
                    if (sub == 0) *reinterpret_cast<float*>(&lds.q[wave][r][HD]) = __builtin_ldexpf(a.scale * 1.44269504088896f, e - 9);
                }
#pragma unroll
                for (int k = 0; k < 2 * NB; ++k) q[c][k] = *reinterpret_cast<const half8v*>(&lds.q[wave][col][16 * k + 8 * half]);
                qscale[c] = *reinterpret_cast<const float*>(&lds.q[wave][col][HD]);
            }
            __syncthreads();  // (the queries' place is taken by the blocks)

            float m[CT], l[CT];
            float16v acc[CT][NB];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                m[c] = -__builtin_inff();
                l[c] = 0;
                for (int b = 0; b < NB; ++b)
                    for (int r = 0; r < 16; ++r) acc[c][b][r] = 0;
            }

            // 32 positions from t0 on, for the sets of columns from FIRST on
            const auto sub = [&](auto from, const BlockLds<NB>& in, int32_t t0, int tt) {
                constexpr int FIRST = decltype(from)::value;
                const bool here[2] = {in.there[2 * tt] != 0, in.there[2 * tt + 1] != 0};
                const bool poison = (in.poison[2 * tt] | in.poison[2 * tt + 1]) != 0;
                float16v sc[CT];
                half8v p[CT][2];
                uint32_t seen[CT];
#pragma unroll
                for (int c = FIRST; c < CT; ++c) sc[c] = float16v{};
#pragma unroll
                for (int k = 0; k < 2 * NB; ++k) {
                    const half8v kx = __builtin_bit_cast(half8v, in.k[tt][k][lane]);
#pragma unroll
                    for (int c = FIRST; c < CT; ++c) sc[c] = mfma(kx, q[c][k], sc[c]);
                }
#pragma unroll
                for (int c = FIRST; c < CT; ++c) {
                    const bool full = here[0] && here[1] && t0 + 31 <= pos_lo[c] && (window == 0 || t0 > pos_hi[c] - window);
                    seen[c] = 0xFFFF;
                    if (!full) {
                        seen[c] = 0;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int32_t t = t0 + 8 * (r / 4) + 4 * half + r % 4;
                            if (here[r / 8] && t <= pos[c] && (window == 0 || t > pos[c] - window)) seen[c] |= 1u << r;
                            else sc[c][r] = qscale[c] < 0 ? __builtin_inff() : -__builtin_inff();
                        }
                    }
                    float top = -__builtin_inff();
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        sc[c][r] *= qscale[c];
                        top = __builtin_fmaxf(top, sc[c][r]);
                    }
                    if (__any(top > m[c] + kLazy)) {
                        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                        const float next = __builtin_fmaxf(m[c], top);
                        const float f = weight(m[c], next);
                        m[c] = next;
                        l[c] *= f;
#pragma unroll
                        for (int b = 0; b < NB; ++b) acc[c][b] *= f;
                    }
                    const float base = m[c] == -__builtin_inff() ? 0.0f : m[c] - kLift;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float e = __builtin_amdgcn_exp2f(sc[c][r] - base);
                        l[c] += e;
                        p[c][r / 8][r % 8] = static_cast<_Float16>(e);
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const half8v vx = __builtin_bit_cast(half8v, in.v[b][2 * tt + u][lane]);
#pragma unroll
                        for (int c = FIRST; c < CT; ++c) acc[c][b] = mfma(vx, p[c][u], acc[c][b]);
                    }
                }
                if (__builtin_expect(poison, 0)) {  // the values that are not finite, from the tiles themselves
#pragma unroll 1
                    for (int u = 0; u < 2; ++u) {
                        const int32_t t = t0 + 16 * u, page = page_of(a.kv, a.b, s, t);
                        const uint8_t* tile_ = a.kv.data + tile_at(a.kv, page < 0 ? 0 : page, h, t);
                        half8v sees[CT];
                        for (int c = FIRST; c < CT; ++c)
                            for (int e = 0; e < 8; ++e) sees[c][e] = static_cast<_Float16>(seen[c] >> (8 * u + e) & 1 ? 1.0f : 0.0f);
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            uint32_t up[4] = {}, down[4] = {};
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const uint32_t token = e / 4 * 8 + 4 * half + e % 4, d = 32 * b + col;
                                const uint32_t x = *reinterpret_cast<const uint16_t*>(
                                    tile_ + (Q4 ? scale_offset(NB, true, token, b) : value_offset(false, NB, token, d & ~1) + (d & 1) * 2));
                                const Marks mk = Q4 ? scale_marks(x) : marks(x);
                                up[e / 2] |= mk.up << (16 * (e % 2));
                                down[e / 2] |= mk.down << (16 * (e % 2));
                            }
#pragma unroll
                            for (int c = FIRST; c < CT; ++c) {
                                const float16v f = mfma(operand(up[0], up[1], up[2], up[3]), sees[c], float16v{});
                                const float16v g = mfma(operand(down[0], down[1], down[2], down[3]), sees[c], float16v{});
                                for (int r = 0; r < 16; ++r) acc[c][b][r] += ill_sum(f[r], g[r]);
                            }
                        }
                    }
                }
            };
            const auto walk = [&](auto from, int32_t begin, int32_t end) {
                constexpr int FIRST = decltype(from)::value;
                for (int32_t blk = begin; blk < end; ++blk) {
                    if (blk + 1 < blk_end) fetch(blk + 1);
                    const BlockLds<NB>& in = lds.block[blk & 1];
#pragma unroll 1
                    for (int tt = 0; tt < kBlock / 32; ++tt) {
                        const int32_t t0 = blk * kBlock + 32 * tt;
                        bool on = false;
                        for (int c = FIRST; c < CT; ++c) on |= t0 < t_hi[c] && t0 + 32 > t_lo[c];
                        if (on) sub(from, in, t0, tt);
                    }
                    if (blk + 1 < blk_end) put(blk + 1);
                    __syncthreads();
                }
            };

            if (blk_begin < blk_end) put(blk_begin);
            __syncthreads();
            if constexpr (CT == 2) {
                // once all of the workgroup's front sets have seen their positions, the back sets go on alone
                int32_t both = blk_end;
                if (mirrored) {
                    int32_t front_lo, front_hi, x, y;
                    range(std::min(set * kWaves + kWaves, halves_of) - 1, x, y, front_lo, front_hi);
                    both = std::min(blk_end, std::max(blk_begin, (front_hi + kBlock - 1) / kBlock));
                }
                walk(std::integral_constant<int, 0>{}, blk_begin, both);
                walk(std::integral_constant<int, 1>{}, both, blk_end);
            } else {
                walk(std::integral_constant<int, 0>{}, blk_begin, blk_end);
            }

            // out by way of the wave's part of LDS, so that rows are written whole
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const float sum = l[c] + __shfl_xor(l[c], 32);
                const float f = a.splits != 1 ? 1.0f : sum == 0 ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float4v y;
                        for (int r = 0; r < 4; ++r) y[r] = sum == 0 ? 0.0f : acc[c][b][4 * x + r] * f;
                        *reinterpret_cast<float4v*>(&lds.out[wave][col][32 * b + 8 * x + 4 * half]) = y;
                    }
                }
                const uint32_t cc = tile[c] * kWide + col;
                if (a.splits != 1 && half == 0 && cc < cols) {
                    const uint32_t row = over(cc, a.group);
                    float* ml = a.part + static_cast<size_t>(a.b.rows) * a.heads * a.splits * HD +
                                ((static_cast<size_t>(sr.begin + row) * a.heads + h * a.group.d + (cc - row * a.group.d)) * a.splits + split) * 2;
                    ml[0] = m[c];
                    ml[1] = sum;
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                for (int n = lane; n < kWide * (HD / 8); n += 64) {
                    const int r = n / (HD / 8), d = n % (HD / 8) * 8;
                    const uint32_t oc = tile[c] * kWide + r;
                    if (oc >= cols) continue;
                    const uint32_t row = over(oc, a.group), head = h * a.group.d + (oc - row * a.group.d);
                    const float4v *from = reinterpret_cast<const float4v*>(&lds.out[wave][r][d]), lo = from[0], hi = from[1];
                    const float y[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    if (a.splits != 1) {
                        store8(a.part + ((static_cast<size_t>(sr.begin + row) * a.heads + head) * a.splits + split) * HD, kTypeF32, true, d, y);
                    } else {
                        char* op = row_ptr(a.out, sr.begin + row, head);
                        store8(op, a.out.type, (reinterpret_cast<uintptr_t>(op) & 15) == 0, d, y);
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
}

template <int NB, int CT>
hipError_t launch_typed(const PagedAttnArgs& a, dim3 grid, hipStream_t st) {
    if (a.kv.q4) k_paged_prompt<NB, CT, true><<<grid, dim3(64 * kWaves), 0, st>>>(a);
    else k_paged_prompt<NB, CT, false><<<grid, dim3(64 * kWaves), 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

uint32_t prompt_columns(uint32_t head_dim) { return head_dim <= 128 ? 2 * kWide * kWaves : kWide * kWaves; }

hipError_t launch_paged_prompt(const PagedAttnArgs& a, uint32_t max_rows, hipStream_t st) {
    const uint32_t wide = prompt_columns(a.kv.head_dim);
    const uint64_t cols = static_cast<uint64_t>(max_rows) * a.group.d, sets = std::min<uint64_t>((cols + wide - 1) / wide, 65535 / a.splits);
    const dim3 grid(a.kv.kv_heads, static_cast<uint32_t>(sets * a.splits), std::min<uint32_t>(a.b.seqs, 65535));
    switch (a.kv.head_dim / 32) {
        case 2: return launch_typed<2, 2>(a, grid, st);
        case 3: return launch_typed<3, 2>(a, grid, st);
        case 4: return launch_typed<4, 2>(a, grid, st);
        case 8: return launch_typed<8, 1>(a, grid, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace bh
