// Attention of prompts over their pages: many rows of a sequence at once.
//
// As in paged_attention.hip the product's sides are swapped, S^T = K Q^T and O^T = V^T P^T, here with
// v_mfma_f32_32x32x16_f16 (twice the rate of the 16-wide one: 2.08 against 1.14 PFLOP/s measured), and
// a lane's probabilities are its second product's operand as they stand.  Keys and values pass through
// LDS, 64 or 128 positions at a time, as halves in operand order: a tile is unpacked once for the workgroup's
// columns, and an operand is one conflict-free 16-byte read of a lane.  (128 in the place of 64: 263 us for 306, half the barriers.)
#include <algorithm>

#include "paged.h"
#include "paged_device.h"

namespace bh {
namespace {

constexpr int kBlock = 64;  // positions of a wave's step
constexpr int kVector = 0x2, kMfma = 0x8;  // instructions' classes, for their order
constexpr int kWide = 32;   // columns of a wave: (row, head) pairs of a key/value head

// Waves of a workgroup, a CU's only one: two a SIMD where 256 registers hold a wave's queries and sums, otherwise one.
constexpr int waves_of(int nb, bool exact) { return nb * (exact ? 2 : 1) <= 4 ? 8 : 4; }

// What a thread holds of its wave's half of a tile, blocks b0 .. b0 + HB - 1 of every position, until it goes to LDS.
template <int NB, bool Q4>
struct RawTile {
    static constexpr int GS = NB < 4 ? NB : 4, HB = (NB + 1) / 2, ALIGN = NB % 4 == 0 ? HB * 4 : 4;
    uint32_t k[HB][Q4 ? 1 : 4], ks[Q4 ? HB : 1], v[Q4 ? 1 : 4][HB], vs[Q4 ? 2 * HB : 1];

    // (of three blocks both halves take the middle one)
    static __device__ inline int first(int part) { return part ? NB - HB : 0; }

    __device__ inline void load(const uint8_t* tile, int b0, int lane) {
        const uint32_t at = ((b0 / GS * 64 + lane) * GS + b0 % GS) * 4;
        if constexpr (Q4) {
            uint32_t x[HB];
            load_words<HB, ALIGN>(tile + at, x);
#pragma unroll
            for (int j = 0; j < HB; ++j) {
                k[j][0] = x[j];
                ks[j] = *reinterpret_cast<const uint16_t*>(tile + scale_offset(NB, false, lane % 16, b0 + j)) * 0x10001u;  // the lane's position's, twice
            }
            load_words<HB, ALIGN>(tile + tile_values_at(true, NB) + at, v[0]);
            load_words<2 * HB, 8>(tile + tile_value_scales_at(NB) + (lane / 16 * NB + b0) * 8, vs);
        } else {
#pragma unroll
            for (int j = 0; j < HB; ++j) load_words<4>(tile + ((b0 + j) * 64 + lane) * 16, k[j]);
#pragma unroll
            for (int r = 0; r < 4; ++r) load_words<HB, ALIGN>(tile + tile_values_at(false, NB) + r * NB * 256 + at, v[r]);
        }
    }
    // The values of positions 4 g + r whose bit r of `keep` is not set become zeros.
    __device__ inline void keep_values(uint32_t keep) {
        if constexpr (Q4) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t b = keep >> (2 * j), mask = (b & 1 ? 0xFFFF : 0) | (b & 2 ? 0xFFFF0000 : 0);
                for (int e = 0; e < HB; ++e) vs[2 * e + j] &= mask;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t mask = keep >> r & 1 ? 0xFFFFFFFF : 0;
                for (int e = 0; e < HB; ++e) v[r][e] &= mask;
            }
        }
    }
    // Whether an infinity or NaN is among the values; and zeros in their place.
    __device__ inline bool any_ill() const {
        uint32_t found = 0;
        if constexpr (Q4) {
            for (int e = 0; e < 2 * HB; ++e) found |= ill<true>(vs[e]);
        } else {
            for (int r = 0; r < 4; ++r)
                for (int e = 0; e < HB; ++e) found |= ill<false>(v[r][e]);
        }
        return __any((found & kIll) != 0);
    }
    __device__ inline void drop_ill() {
        if constexpr (Q4) {
            for (int e = 0; e < 2 * HB; ++e) vs[e] = scale_marks(vs[e]).rest;
        } else {
            for (int r = 0; r < 4; ++r)
                for (int e = 0; e < HB; ++e) v[r][e] = marks(v[r][e]).rest;
        }
    }
};

// STEPS x 64 positions as operands [32 positions][16 dimensions] and [32 dimensions][16 positions], 64 lanes x 16 bytes
// each, in one plane or, for 4-bit values with 32-bit results, in two that add up to them.
template <int NB, int PLANES, int STEPS>
struct BlockLds {
    word4v k[PLANES][STEPS * 2][2 * NB][64];
    word4v v[PLANES][NB][STEPS * 4][64];
    uint8_t there[8], poison[8];  // whether a wave's half tile is there, and holds values that are not finite (here they are zeros)
};

// A code times its scale, in one half (rounded: 2^-11 of the value at most, as the probabilities are), or in two (exact).
template <int PLANES>
__device__ inline void scaled(half2v code, uint32_t scale, uint32_t (&out)[PLANES]) {
    const half2v d = halves(scale), x = code * d;
    out[0] = bits(x);
    if constexpr (PLANES == 2) out[1] = bits(__builtin_elementwise_fma(code, d, -x));
}

template <int NB, bool Q4, int PLANES, int STEPS>
__device__ inline void unpack(const RawTile<NB, Q4>& raw, BlockLds<NB, PLANES, STEPS>& out, int x, int b0, int lane) {
    const int i = lane % 16, g = lane / 16;
#pragma unroll
    for (int j = 0; j < RawTile<NB, Q4>::HB; ++j) {
        uint32_t key[4][PLANES];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (Q4) scaled<PLANES>(codes(raw.k[j][0] >> (e / 2 * 8), e % 2), raw.ks[j], key[e]);
            else key[e][0] = raw.k[j][e];
        }
#pragma unroll
        for (int p = 0; p < PLANES; ++p) out.k[p][x / 2][2 * (b0 + j) + g / 2][g % 2 * 32 + x % 2 * 16 + i] = word4v{key[0][p], key[1][p], key[2][p], key[3][p]};
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
            uint32_t val[2][PLANES];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if constexpr (Q4) scaled<PLANES>(codes(raw.v[0][j] >> (e * 8), c2), raw.vs[2 * j + e], val[e]);
                else val[e][0] = __builtin_amdgcn_perm(raw.v[2 * e + 1][j], raw.v[2 * e][j], c2 ? 0x07060302 : 0x05040100);
            }
#pragma unroll
            for (int p = 0; p < PLANES; ++p) reinterpret_cast<word2v*>(&out.v[p][b0 + j][x][g % 2 * 32 + 2 * i + c2])[g / 2] = word2v{val[0][p], val[1][p]};
        }
    }
}

// A workgroup takes 256 columns, or 128, and one part of the positions, a wave 32 columns.  Without a window half of eight
// waves' columns are from the front of the prompt and half are their mirror image from the back: what
// two such waves, which share a SIMD, see adds up to the same for all.  Four waves have a SIMD each and columns next to each
// other, the last of the prompt, which see most, first.
//
// Bound by the issue of vector and matrix instructions together.  4000 rows of 8100 positions, 16 heads of 128 in 4 bits: 263 us,
// 760 TFLOP/s, where the products and their operands' reads take 160, the softmax 30, the unpacking 45 and the fetches and
// searches for what is not finite the rest, as far as they do not overlap; of fp16 pages 304.  With four waves, one a SIMD, the latter
// take 443: a lone wave issues a vector instruction every eight cycles, two every four each.  Heads of 256 do not
// fit eight: 494 us spilled, 137 by four (2000 rows of 4000, 8 heads in 4 bits; 360 TFLOP/s).  Four for 32-bit results: 406 spilled, 236 (2000 of
// 4000, 16 heads of 128 in 4 bits, three products in the place of one).
template <int NB, bool Q4, bool EXACT>
__global__ __launch_bounds__(64 * waves_of(NB, EXACT)) __attribute__((amdgpu_waves_per_eu(waves_of(NB, EXACT) / 4, waves_of(NB, EXACT) / 4))) void k_paged_prompt(PagedAttnArgs a) {
    constexpr int HD = 32 * NB, PLANES = Q4 && EXACT ? 2 : 1, PARTS = EXACT ? 2 : 1, PRODUCTS = EXACT + PLANES, kWaves = waves_of(NB, EXACT);
    // Two blocks in LDS, one multiplied while the other is filled: of 128 positions for eight waves, where they fit
    // (two 64-KB blocks), and of 64 for four: a tile for each wave.
    constexpr int STEPS = kWaves / 4, BLOCK = STEPS * kBlock, HALVES = 2 / STEPS;
    constexpr int CHUNK = NB < 4 ? 2 * NB : 8, CHUNKS = 4 * NB / CHUNK;  // operands that are read at a time
    typedef BlockLds<NB, PLANES, STEPS> Block;
    __shared__ union {
        Block block[2];
        struct {
            _Float16 part[PARTS][kWaves][16][HD + 8];  // (half of a wave's columns at a time)
            float scale[kWaves][16];
        } q;
        float out[kWaves][16][HD + 4];
    } lds;
    const int lane = static_cast<int>(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int col = lane % 32, half = lane / 32;
    const uint32_t h = blockIdx.x, split = blockIdx.y % a.splits, first_set = blockIdx.y / a.splits, set_step = gridDim.y / a.splits;
    const int32_t window = a.window > static_cast<uint32_t>(kMaxLength) ? 0 : static_cast<int32_t>(a.window);
    const int32_t capacity = static_cast<int32_t>(std::min<int64_t>(kMaxLength, static_cast<int64_t>(a.b.page_stride) << a.kv.page_shift));

    for (uint32_t s = blockIdx.z; s < a.b.seqs; s += gridDim.z) {
        const SeqRows sr = seq_rows(a.b, s);
        const uint32_t cols = (sr.end - sr.begin) * a.group.d, tiles = (cols + kWide - 1) / kWide;
        const bool mirrored = kWaves == 8 && window == 0;
        const uint32_t fronts = mirrored ? (tiles + 1) / 2 : tiles, per_set = mirrored ? kWaves / 2 : kWaves, sets = (fronts + per_set - 1) / per_set;
        // the positions of a column tile's rows, and those that they see
        const auto range = [&](uint32_t t, int32_t& plo, int32_t& phi, int32_t& tlo, int32_t& thi) {
            const uint32_t last = std::min<uint32_t>((t + 1) * kWide, cols) - 1;
            plo = sr.first + static_cast<int32_t>(over(t * kWide, a.group));
            phi = sr.first + static_cast<int32_t>(over(last, a.group));
            tlo = window != 0 && plo - window + 1 > 0 ? plo - window + 1 : 0;
            thi = std::min(phi + 1, capacity);
        };
        for (uint32_t set = first_set; set < sets; set += set_step) {
            const uint32_t front = (mirrored ? set : sets - 1 - set) * per_set, back_last = std::min(front + per_set, fronts) - 1;
            uint32_t tile = front + (wave & (per_set - 1));
            if (mirrored && wave >= kWaves / 2) tile = tile < fronts && tiles - 1 - tile >= fronts ? tiles - 1 - tile : tiles;
            else if (tile >= fronts) tile = tiles;
            int32_t pos_lo = 0, pos_hi = 0, t_lo = 0, t_hi = 0;
            if (tile < tiles) range(tile, pos_lo, pos_hi, t_lo, t_hi);
            const int32_t pos = tile * kWide + col < cols ? sr.first + static_cast<int32_t>(over(tile * kWide + col, a.group)) : pos_lo;
            int32_t wg_lo, wg_plo, wg_phi, wg_hi, y0, y1, y2;  // the workgroup's, from its first tile's to its last one's
            range(front, wg_plo, y0, wg_lo, y1);
            range(mirrored ? tiles - 1 - front : back_last, y0, wg_phi, y2, wg_hi);
            const int32_t blk_lo = wg_lo / BLOCK, blocks = wg_hi > wg_lo ? (wg_hi + BLOCK - 1) / BLOCK - blk_lo : 0;
            const int32_t per = (blocks + static_cast<int32_t>(a.splits) - 1) / static_cast<int32_t>(a.splits);
            const int32_t blk_begin = blk_lo + static_cast<int32_t>(std::min<int64_t>(blocks, static_cast<int64_t>(per) * split));
            const int32_t blk_end = blk_lo + static_cast<int32_t>(std::min<int64_t>(blocks, static_cast<int64_t>(per) * (split + 1)));

            RawTile<NB, Q4> raw[2];  // the wave's tile of a block, in halves: one for each step, or both for the only one
            bool there = false, poison = false;
            const auto part = [&](int n) { return RawTile<NB, Q4>::first(n); };
            const WavePages pages(a.kv, a.b, s, h);
            const auto page_at = [&](int32_t blk) { return pages.page(blk * BLOCK + 16 * wave); };
            uint32_t page = 0, page_next = 0;
            const auto fetch = [&](int32_t blk, int step) {
#pragma unroll
                for (int n = step * HALVES; n < (step + 1) * HALVES; ++n) raw[n].load(pages.tile(page, blk * BLOCK + 16 * wave, tile_bytes(Q4, NB)), part(n), lane);
            };
            // some column does not see all of a block: what none sees is left out; and what is not finite
            const auto check = [&](int32_t blk) {
                if (!there || (blk + 1) * BLOCK - 1 > wg_plo || (window != 0 && blk * BLOCK <= wg_phi - window)) {
                    const int32_t t = blk * BLOCK + 16 * wave + 4 * (lane / 16);
                    uint32_t keep = 0;
                    for (int r = 0; r < 4; ++r) keep |= there && t + r >= wg_lo && t + r <= wg_phi ? 1u << r : 0;
#pragma unroll
                    for (int n = 0; n < 2; ++n) raw[n].keep_values(keep);
                }
                poison = raw[0].any_ill();
                poison |= raw[1].any_ill();
                if (__builtin_expect(poison, 0)) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) raw[n].drop_ill();
                }
            };
            const auto put = [&](int32_t blk, int n0, int count) {
                Block& out = lds.block[blk & 1];
#pragma unroll
                for (int n = n0; n < n0 + count; ++n) unpack<NB, Q4, PLANES, STEPS>(raw[n], out, wave, part(n), lane);
                out.there[wave] = there;  // (every lane the same: a branch would end the block of instructions that is scheduled)
                out.poison[wave] = poison;
            };
            // A part of the next block goes to LDS; then the same part of the block after it is fetched, of a page whose number
            // was read a block before.
            const auto next = [&](int32_t blk, int step) {
                if (step == 0) {
                    page = page_next;
                    page_next = page_at(blk + 3);
                }
                fetch(blk + 2, step);
            };
            if (blk_begin < blk_end) {
                page = page_at(blk_begin);
                page_next = page_at(blk_begin + 1);
#pragma unroll
                for (int step = 0; step < STEPS; ++step) fetch(blk_begin, step);
            }

            // the columns' queries, through the wave's part of LDS: 16 lanes a column, scaled by a power of two where the
            // type has more range than a half, and by the sign of the score's scale
            __syncthreads();  // the blocks of the columns before
            half8v q[PARTS][2 * NB];
            float qscale = 0;
#pragma unroll 1
            for (int c0 = 0; c0 < kWide; c0 += 16) {
                const int sub = lane % 16;
#pragma unroll 1
                for (int r = lane / 16; r < 16; r += 4) {
                    constexpr int K = (HD + 127) / 128;
                    const uint32_t cc = tile * kWide + c0 + r;
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
                        half8v hi, lo;
                        for (int j = 0; j < 8; ++j) {
                            const float y = __builtin_ldexpf(a.scale < 0 ? -x[k][j] : x[k][j], 9 - e);
                            hi[j] = static_cast<_Float16>(y);
                            lo[j] = static_cast<_Float16>(y - static_cast<float>(hi[j]));
                        }
                        if (d < HD) {
                            *reinterpret_cast<half8v*>(&lds.q.part[0][wave][r][d]) = hi;
                            if constexpr (EXACT) *reinterpret_cast<half8v*>(&lds.q.part[1][wave][r][d]) = lo;
                        }
                    }
                    // (never 0: scores of 0 and of minus infinity, what is not seen, stay what they are)
                    if (sub == 0) lds.q.scale[wave][r] = __builtin_fmaxf(__builtin_ldexpf(__builtin_fabsf(a.scale) * 1.44269504088896f, e - 9), 1.17549435e-38f);
                }
                __builtin_amdgcn_wave_barrier();
                if (col / 16 == c0 / 16) {
#pragma unroll
                    for (int k = 0; k < 2 * NB; ++k)
                        for (int e = 0; e < PARTS; ++e) q[e][k] = *reinterpret_cast<const half8v*>(&lds.q.part[e][wave][col % 16][16 * k + 8 * half]);
                    qscale = lds.q.scale[wave][col % 16];
                }
                __builtin_amdgcn_wave_barrier();
            }
            __syncthreads();  // (the queries' place is taken by the blocks)

            Maximum mx;
            float l = 0;
            float16v acc[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b] = float16v{};

            // A block of 64 positions from t0 on: two products of 32 side by side, since one's steps wait for each other;
            // the next block is unpacked under them.
            const auto sub = [&](const Block& in, int32_t blk, int step) {
                const int32_t t0 = blk * BLOCK + step * kBlock;
                const uint32_t heres = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t*>(in.there)[step]);
                const uint32_t ills = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t*>(in.poison)[step]);
                float16v sc[2] = {};
                // A chunk's operands are read ahead of the products of the chunk before; the barriers keep the compiler
                // from undoing that.
                half8v ops[2][PLANES][CHUNK];
                const auto read_keys = [&](int c) {
#pragma unroll
                    for (int k = 0; k < CHUNK; ++k)
                        for (int e = 0; e < PLANES; ++e) ops[c % 2][e][k] = __builtin_bit_cast(half8v, in.k[e][2 * step + k % 2][c * CHUNK / 2 + k / 2][lane]);
                };
                const auto keys_times = [&](int c) {
#pragma unroll
                    for (int k = 0; k < CHUNK; ++k) {
                        const int at = c * CHUNK / 2 + k / 2;
                        if constexpr (EXACT) {
                            sc[k % 2] = mfma(ops[c % 2][0][k], q[1][at], sc[k % 2]);
                            if constexpr (Q4) sc[k % 2] = mfma(ops[c % 2][1][k], q[0][at], sc[k % 2]);
                        }
                        sc[k % 2] = mfma(ops[c % 2][0][k], q[0][at], sc[k % 2]);
                    }
                };
                read_keys(0);
#pragma unroll
                for (int c = 0; c < CHUNKS; c += 2) {
                    __builtin_amdgcn_sched_barrier(0);
                    read_keys(c + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (CHUNKS == 2) put(blk + 1, step * HALVES, HALVES);
                    else put(blk + 1, c / 2, 1);
                    keys_times(c);
                    if constexpr (CHUNKS != 2) {
#pragma unroll
                        for (int k = 0; k < CHUNK; ++k) {
                            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(kVector, 16, 0);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                        if (c + 2 < CHUNKS) read_keys(c + 2);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    keys_times(c + 1);
                    if constexpr (CHUNKS == 2) {
#pragma unroll
                        for (int k = 0; k < 4 * NB * PRODUCTS; ++k) {
                            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(kVector, EXACT ? 6 : 4, 0);
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                next(blk, step);
                // the values' operands likewise
                const auto read_values = [&](int c) {
#pragma unroll
                    for (int k = 0; k < CHUNK; ++k)
                        for (int e = 0; e < PLANES; ++e) ops[c % 2][e][k] = __builtin_bit_cast(half8v, in.v[e][k % NB][4 * step + c * (CHUNK / NB) + k / NB][lane]);
                };
                read_values(0);
                __builtin_amdgcn_sched_barrier(0);
                // the column sees positions t0 + u with lo < u <= hi, in tiles that are there
                const int32_t hi = pos - t0, lo = window != 0 ? hi - window : -1;
                if (heres != 0x01010101 || t0 + kBlock - 1 > pos_lo || (window != 0 && t0 <= pos_hi - window)) {
                    asm volatile("");  // a branch, not 32 selects for every block
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int32_t u = 32 * tt + 8 * (r / 4) + 4 * half + r % 4;
                            if (u > hi || u <= lo || (heres >> (16 * tt + r / 8 * 8) & 1) == 0) sc[tt][r] = -__builtin_inff();
                        }
                    }
                }
                float tops[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    tops[x] = sc[x / 2][x % 2 * 8];
                    for (int r = 1; r < 8; ++r) tops[x] = __builtin_fmaxf(tops[x], sc[x / 2][x % 2 * 8 + r]);
                }
                float top = __builtin_fmaxf(__builtin_fmaxf(tops[0], tops[1]), __builtin_fmaxf(tops[2], tops[3]));
                if (__any(top * qscale > mx.m + kLazy)) {
                    top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                    const float f = mx.renew(top, qscale);
                    l *= f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) acc[b] *= f;
                }
                if (mx.far) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        sc[0][r] -= mx.shift;
                        sc[1][r] -= mx.shift;
                    }
                }
                half8v p[PARTS][4];
                float sums[2] = {};
                const auto exponentials = [&](int tt) {
#pragma unroll
                    for (int r = 0; r < 16; r += 2) {
                        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[tt][r], qscale, -mx.base));
                        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[tt][r + 1], qscale, -mx.base));
                        const half2v e{static_cast<_Float16>(e0), static_cast<_Float16>(e1)};
                        p[0][2 * tt + r / 8][r % 8] = e[0];
                        p[0][2 * tt + r / 8][r % 8 + 1] = e[1];
                        if constexpr (EXACT) {
                            p[1][2 * tt + r / 8][r % 8] = static_cast<_Float16>(e0 - static_cast<float>(e[0]));
                            p[1][2 * tt + r / 8][r % 8 + 1] = static_cast<_Float16>(e1 - static_cast<float>(e[1]));
                            sums[0] += e0;
                            sums[1] += e1;
                        } else {
                            sums[r / 2 % 2] = __builtin_amdgcn_fdot2(e, half2v{1, 1}, sums[r / 2 % 2], false);  // (the sum of what is multiplied)
                        }
                    }
                };
                const auto values_times = [&](int c) {
#pragma unroll
                    for (int k = 0; k < CHUNK; ++k) {
                        const int u = c * (CHUNK / NB) + k / NB, b = k % NB;
                        if constexpr (EXACT) {
                            acc[b] = mfma(ops[c % 2][0][k], p[1][u], acc[b]);
                            if constexpr (Q4) acc[b] = mfma(ops[c % 2][1][k], p[0][u], acc[b]);
                        }
                        acc[b] = mfma(ops[c % 2][0][k], p[0][u], acc[b]);
                    }
                };
                exponentials(0);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (c + 1 < CHUNKS) read_values(c + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    values_times(c);
                    if (c == 0) {  // the second exponentials under the first products
                        exponentials(1);
#pragma unroll
                        for (int k = 0; k < CHUNK * PRODUCTS; ++k) {
                            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(kVector, 48 / CHUNK, 0);
                        }
                    }
                }
                l += sums[0] + sums[1];
                if (__builtin_expect(ills != 0, 0)) {
                    // the values that are not finite, from the tiles themselves
#pragma unroll 1
                    for (int u = 0; u < 4; ++u) {
                        const int32_t t = t0 + 16 * u;
                        const uint32_t at = pages.page(t);
                        const uint8_t* from = pages.tile(at, t, tile_bytes(Q4, NB));
                        half8v sees;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int32_t token = 16 * u + e / 4 * 8 + 4 * half + e % 4;
                            sees[e] = static_cast<_Float16>(token <= hi && token > lo && pages.there(at) ? 1.0f : 0.0f);
                        }
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            uint32_t up[4] = {}, down[4] = {};
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const uint32_t token = e / 4 * 8 + 4 * half + e % 4, d = 32 * b + col;
                                const uint32_t x = *reinterpret_cast<const uint16_t*>(
                                    from + (Q4 ? scale_offset(NB, true, token, b) : value_offset(false, NB, token, d & ~1) + (d & 1) * 2));
                                const Marks mk = Q4 ? scale_marks(x) : marks(x);
                                up[e / 2] |= mk.up << (16 * (e % 2));
                                down[e / 2] |= mk.down << (16 * (e % 2));
                            }
                            const float16v f = mfma(operand(up[0], up[1], up[2], up[3]), sees, float16v{});
                            const float16v g = mfma(operand(down[0], down[1], down[2], down[3]), sees, float16v{});
                            for (int r = 0; r < 16; ++r) acc[b][r] += ill_sum(f[r], g[r]);
                        }
                    }
                }
            };

            if (blk_begin < blk_end) {
                there = pages.there(page);
                check(blk_begin);
#pragma unroll
                for (int step = 0; step < STEPS; ++step) {
                    put(blk_begin, step * HALVES, HALVES);
                    next(blk_begin - 1, step);
                }
            }
            __syncthreads();
            for (int32_t blk = blk_begin; blk < blk_end; ++blk) {
                there = pages.there(page);
                check(blk + 1);
#pragma unroll
                for (int step = 0; step < STEPS; ++step) {
                    const int32_t t0 = blk * BLOCK + step * kBlock;
                    if (t0 < t_hi && t0 + kBlock > t_lo) {
                        sub(lds.block[blk & 1], blk, step);
                    } else {
                        put(blk + 1, step * HALVES, HALVES);
                        next(blk, step);
                    }
                }
                __syncthreads();
            }

            // out by way of the wave's part of LDS, so that rows are written whole
            const float sum = l + __shfl_xor(l, 32);
            const float f = a.splits != 1 ? 1.0f : sum == 0 ? 0.0f : 1.0f / sum;
            if (a.splits != 1 && half == 0 && tile * kWide + col < cols) {
                const uint32_t cc = tile * kWide + col, row = over(cc, a.group);
                float* ml = a.part + static_cast<size_t>(a.b.rows) * a.heads * a.splits * HD +
                            ((static_cast<size_t>(sr.begin + row) * a.heads + h * a.group.d + (cc - row * a.group.d)) * a.splits + split) * 2;
                ml[0] = mx.m;
                ml[1] = sum;
            }
#pragma unroll 1
            for (int c0 = 0; c0 < kWide; c0 += 16) {
                if (col / 16 == c0 / 16) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            float4v y;
                            for (int r = 0; r < 4; ++r) y[r] = sum == 0 ? 0.0f : acc[b][4 * x + r] * f;
                            *reinterpret_cast<float4v*>(&lds.out[wave][col % 16][32 * b + 8 * x + 4 * half]) = y;
                        }
                    }
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                for (int n = lane; n < 16 * (HD / 8); n += 64) {
                    const int r = n / (HD / 8), d = n % (HD / 8) * 8;
                    const uint32_t oc = tile * kWide + c0 + r;
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

template <int NB>
hipError_t launch_typed(const PagedAttnArgs& a, bool exact, dim3 grid, hipStream_t st) {
    const dim3 threads(64 * waves_of(NB, exact));
    if (!exact) {
        if (a.kv.q4) k_paged_prompt<NB, true, false><<<grid, threads, 0, st>>>(a);
        else k_paged_prompt<NB, false, false><<<grid, threads, 0, st>>>(a);
    } else if constexpr (NB <= 4) {
        if (a.kv.q4) k_paged_prompt<NB, true, true><<<grid, threads, 0, st>>>(a);
        else k_paged_prompt<NB, false, true><<<grid, threads, 0, st>>>(a);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

uint32_t prompt_columns(uint32_t head_dim, bool exact) { return kWide * waves_of(static_cast<int>(head_dim / 32), exact); }

// 32-bit results take twice the registers and, of 4-bit caches, twice the LDS: heads of up to 128 values.
bool prompt_fits(uint32_t head_dim, bool exact) { return head_dim <= (exact ? 128 : 256); }

hipError_t launch_paged_prompt(const PagedAttnArgs& a, bool exact, uint32_t max_rows, hipStream_t st) {
    const uint32_t wide = prompt_columns(a.kv.head_dim, exact);
    const uint64_t cols = static_cast<uint64_t>(max_rows) * a.group.d, sets = std::min<uint64_t>((cols + wide - 1) / wide, 65535 / a.splits);
    const dim3 grid(a.kv.kv_heads, static_cast<uint32_t>(sets * a.splits), std::min<uint32_t>(a.b.seqs, 65535));
    switch (a.kv.head_dim / 32) {
        case 2: return launch_typed<2>(a, exact, grid, st);
        case 3: return launch_typed<3>(a, exact, grid, st);
        case 4: return launch_typed<4>(a, exact, grid, st);
        case 8: return launch_typed<8>(a, exact, grid, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace bh
