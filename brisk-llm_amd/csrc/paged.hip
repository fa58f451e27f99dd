// Rows of queries, keys and values on their way to and from the paged cache: head norms and
// rotations, the append with its 4-bit quantisation, and the read back.
#include <hip/hip_fp16.h>

#include <algorithm>

#include "paged.h"
#include "paged_device.h"

namespace bh {
namespace {

constexpr int kThreads = 256;

// Lanes of a head: one for every eight dimensions, rounded up to a power of two for the shuffles.
int head_lanes(uint32_t head_dim) {
    int t = 4;
    while (t * 8 < static_cast<int>(head_dim)) t *= 2;
    return t;
}

// Whether rows can be read and written 16 bytes at a time.
bool wide(const HeadRows& x) {
    const int64_t size = x.type == kTypeF32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.row * size % 16 == 0 && x.head * size % 16 == 0;
}

template <typename F>
__device__ inline F inverse_root(F x);
template <>
__device__ inline float inverse_root(float x) { return 1.0f / sqrtf(x); }
template <>
__device__ inline double inverse_root(double x) { return 1.0 / sqrt(x); }

__device__ inline float mul_sub(float a, float c, float b, float s) { return __builtin_fmaf(a, c, -(b * s)); }
__device__ inline double mul_sub(double a, double c, double b, double s) { return __builtin_fma(a, c, -(b * s)); }
__device__ inline float mul_add(float a, float c, float b, float s) { return __builtin_fmaf(a, c, b * s); }
__device__ inline double mul_add(double a, double c, double b, double s) { return __builtin_fma(a, c, b * s); }

// Eight values of a head from dimension d on: normed by w (null: not) over the head's `lanes` lanes
// and rotated by the table's row cs (null: not).  Lanes past the head take part in the sums only.
template <typename F>
__device__ inline void turned(const void* head, int type, bool vec, int d, int head_dim, int lanes, const float* w, float eps,
                              const float* cs, int dims, bool neox, float (&out)[8]) {
    const bool live = d < head_dim;
    float own[8] = {};
    if (live) load8(head, type, vec, d, own);
    F scale = 1;
    if (w != nullptr) {
        F sum = 0;
        for (int j = 0; j < 8; ++j) sum += static_cast<F>(own[j]) * static_cast<F>(own[j]);
        for (int m = 1; m < lanes; m *= 2) sum += __shfl_xor(sum, m);
        scale = inverse_root<F>(sum / static_cast<F>(head_dim) + static_cast<F>(eps));
    }
    if (!live) return;
    F x[8];
    for (int j = 0; j < 8; ++j) x[j] = w != nullptr ? static_cast<F>(own[j]) * scale * static_cast<F>(w[d + j]) : static_cast<F>(own[j]);
    if (cs == nullptr || d >= dims) {
        for (int j = 0; j < 8; ++j) out[j] = static_cast<float>(x[j]);
        return;
    }
    if (!neox) {
        for (int j = 0; j < 8; j += 2) {
            if (d + j >= dims) {
                out[j] = static_cast<float>(x[j]);
                out[j + 1] = static_cast<float>(x[j + 1]);
                continue;
            }
            const F c = cs[d + j], s = cs[d + j + 1];
            out[j] = static_cast<float>(mul_sub(x[j], c, x[j + 1], s));
            out[j + 1] = static_cast<float>(mul_add(x[j], s, x[j + 1], c));
        }
        return;
    }
    const int half = dims / 2;
    float other[8];
    const bool whole = half % 8 == 0;  // then the eight partners are eight in a row
    if (whole) load8(head, type, vec, d < half ? d + half : d - half, other);
    for (int j = 0; j < 8; ++j) {
        const int i = d + j;
        if (i >= dims) {
            out[j] = static_cast<float>(x[j]);
            continue;
        }
        const bool low = i < half;
        const int p = low ? i + half : i - half, e = low ? i : i - half;
        if (!whole) other[j] = load1(head, type, p);
        const F y = w != nullptr ? static_cast<F>(other[j]) * scale * static_cast<F>(w[p]) : static_cast<F>(other[j]);
        const F c = cs[2 * e], s = cs[2 * e + 1];
        out[j] = static_cast<float>(low ? mul_sub(x[j], c, y, s) : mul_add(y, s, x[j], c));
    }
}

// One group of lanes a head.  A head's lanes read all they need before they write, so y may be x.  Bound by memory: 4011 rows of 40 heads of 64,
// f32 to bf16, 16.7 us, 3.8 TB/s; one row by its launch and one round trip, 6.
__global__ __launch_bounds__(kThreads) void k_norm_rope(NormRopeArgs a, int lanes, int vec) {
    const int lane = static_cast<int>(threadIdx.x) % lanes, d = lane * 8;
    const uint32_t per = kThreads / lanes, total = static_cast<uint32_t>(a.n) * a.all.d;
    // the shuffles of a group want its whole wave in the loop: the bound is the block's first head
    for (uint32_t base = blockIdx.x * per; base < total; base += gridDim.x * per) {
        const uint32_t u = base + threadIdx.x / lanes;
        const bool in = u < total;
        const uint32_t row = in ? over(u, a.all) : 0;
        uint32_t h = in ? u - row * a.all.d : 0;
        const int t = h >= a.heads[0] ? 1 : 0;
        if (t) h -= a.heads[0];
        const float* cs = nullptr;
        bool keep = !in;
        if (a.rope.table != nullptr) {
            const int32_t pos = a.positions[row];
            if (pos < 0 || static_cast<uint32_t>(pos) >= a.rope.positions) keep = true;
            else cs = a.rope.table + static_cast<size_t>(pos) * a.rope.dims;
        }
        const HeadRows &x = a.x[t], &y = a.y[t];
        float out[8];
        turned<float>(row_ptr(x, row, h), x.type, vec & (1 << t), d, static_cast<int>(a.head_dim), lanes, a.w[t], a.eps, cs,
                      static_cast<int>(a.rope.dims), a.rope.neox != 0, out);
        if (!keep && d < static_cast<int>(a.head_dim)) store8(row_ptr(y, row, h), y.type, vec & (4 << t), d, out);
    }
}

// Codes of eight values of a block of 32 held by four neighbouring lanes, and the block's scale.
// The scale is the value of largest magnitude (the first of equals) over -8, rounded to 16 bits;
// the code is floor(x / d + 8.5) within 0..15, decided exactly: (n - 8.5) d has 16 bits and is
// compared with x, so a quotient that the reciprocal rounds over a border is put back.  A block with a
// value that is not finite, or past kMaxScale, has a scale of NaN and codes of 8.
__device__ inline void quantise8(const float (&y)[8], int lane, uint32_t (&code)[8], uint16_t& scale) {
    float top = y[0];
    int at = lane % 4 * 8;
    bool bad = false;
    for (int j = 0; j < 8; ++j) {
        bad |= !(__builtin_fabsf(y[j]) <= 3.402823466e38f);
        if (__builtin_fabsf(y[j]) > __builtin_fabsf(top)) {
            top = y[j];
            at = lane % 4 * 8 + j;
        }
    }
    int ill = bad ? 1 : 0;
    for (int m = 1; m < 4; m *= 2) {
        const float t = __shfl_xor(top, m);
        const int i = __shfl_xor(at, m);
        ill |= __shfl_xor(ill, m);
        const float p = __builtin_fabsf(t), q = __builtin_fabsf(top);
        if (p > q || (p == q && i < at)) {
            top = t;
            at = i;
        }
    }
    const _Float16 dh = static_cast<_Float16>(top * -0.125f);
    const float d = static_cast<float>(dh), a = __builtin_fabsf(d);
    scale = __builtin_bit_cast(uint16_t, dh);
    if (ill || !(a <= kMaxScale)) {
        scale = 0x7e00;
        for (int j = 0; j < 8; ++j) code[j] = 8;
        return;
    }
    const float inv = a > 0 ? __builtin_amdgcn_rcpf(a) : 0.0f;
    for (int j = 0; j < 8; ++j) {
        const float x = d < 0 ? -y[j] : y[j];
        float n = __builtin_floorf(__builtin_fmaf(x, inv, 8.5f));
        n = __builtin_fminf(__builtin_fmaxf(n, 0.0f), 15.0f);
        if (x < (n - 8.5f) * a) n -= 1;
        else if (x >= (n - 7.5f) * a) n += 1;
        code[j] = a > 0 ? static_cast<uint32_t>(__builtin_fminf(__builtin_fmaxf(n, 0.0f), 15.0f)) : 8;
    }
}

// One group of lanes a row's head of keys, then of values.  The rotation is done in 64 bits: both
// products are exact and the sum is rounded once, so the value that is quantised, rounded to 32 bits,
// does not hang on how the sum is written.
__global__ __launch_bounds__(kThreads) void k_kv_append(AppendArgs a, int lanes, int vec) {
    const int lane = static_cast<int>(threadIdx.x) % lanes, d = lane * 8, hd = static_cast<int>(a.kv.head_dim);
    const uint32_t nb = a.kv.head_dim / 32;
    const bool q4 = a.kv.q4 != 0, live = d < hd;
    const uint32_t per = kThreads / lanes, heads = a.kv.kv_heads;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        const uint32_t total = (sr.end - sr.begin) * heads * 2;
        for (uint32_t base = blockIdx.x * per; base < total; base += gridDim.x * per) {
            const uint32_t u = base + threadIdx.x / lanes;
            const bool in = u < total;
            const uint32_t n = in ? over(u, a.pairs) : 0, row = sr.begin + n;
            uint32_t h = in ? u - n * a.pairs.d : 0;
            const bool value = h >= heads;
            if (value) h -= heads;
            const int32_t pos = sr.first + static_cast<int32_t>(n);
            const int32_t page = page_of(a.kv, a.b, s, pos);
            bool keep = !in || page < 0;
            const float* cs = nullptr;
            if (a.rope.table != nullptr) {
                if (pos < 0 || static_cast<uint32_t>(pos) >= a.rope.positions) keep = true;
                else cs = a.rope.table + static_cast<size_t>(pos) * a.rope.dims;
            }
            const HeadRows& x = value ? a.v : a.k;
            float y[8] = {};
            const bool xv = vec & (value ? 2 : 1);
            turned<double>(row_ptr(x, row, h), x.type, xv, d, hd, lanes, value ? nullptr : a.w, a.eps, value ? nullptr : cs,
                           static_cast<int>(a.rope.dims), a.rope.neox != 0, y);
            uint32_t code[8];
            uint16_t scale = 0;
            if (q4) quantise8(y, lane, code, scale);
            if (keep || !live) continue;
            uint8_t* tile = a.kv.data + tile_at(a.kv, page, h, pos);
            const uint32_t token = static_cast<uint32_t>(pos) % kTileTokens;
            if (!q4) {
                uint32_t w[4];
                for (int j = 0; j < 4; ++j) w[j] = pack_half(y[2 * j], y[2 * j + 1]);
                if (!value) {
                    *reinterpret_cast<uint4*>(tile + key_offset(false, nb, token, d)) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(tile + value_offset(false, nb, token, d + 2 * j)) = w[j];
                }
                continue;
            }
            if (!value) {
                uint32_t w = 0;
                for (int m = 0; m < 4; ++m) w |= code[2 * m] << (4 * m) | code[2 * m + 1] << (4 * m + 16);
                *reinterpret_cast<uint32_t*>(tile + key_offset(true, nb, token, d)) = w;
            } else {
                for (int j = 0; j < 4; ++j) tile[value_offset(true, nb, token, d + 2 * j)] = static_cast<uint8_t>(code[2 * j] | code[2 * j + 1] << 4);
            }
            if (lane % 4 == 0) *reinterpret_cast<uint16_t*>(tile + scale_offset(nb, value, token, d / 32)) = scale;
        }
    }
}

// The larger of a value and those of the lanes 16, 32 and 48 away, and the smaller.
template <bool MAX>
__device__ inline uint32_t across16(uint32_t x) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = MAX ? max(a[0], a[1]) : min(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return MAX ? max(b[0], b[1]) : min(b[0], b[1]);
}

// Codes of eight values of a block of 32 held by the lanes 16 apart, and the block's scale: as quantise8's,
// whose comments hold.  Magnitudes are compared as their bits, in which NaN is largest.
__device__ inline void quantise8_tile(const float (&y)[8], int g, uint32_t (&code)[8], uint16_t& scale) {
    uint32_t top = 0;
    for (int j = 0; j < 8; ++j) top = max(top, __builtin_bit_cast(uint32_t, y[j]) & 0x7FFFFFFF);
    top = across16<true>(top);
    uint32_t at = 1024;  // the first of them, and its sign
    for (int j = 7; j >= 0; --j) {
        const uint32_t b = __builtin_bit_cast(uint32_t, y[j]);
        if ((b & 0x7FFFFFFF) == top) at = (8 * g + j) * 2 + (b >> 31);
    }
    at = across16<false>(at);
    const float size = __builtin_bit_cast(float, top);
    const _Float16 ah = static_cast<_Float16>(size * 0.125f);
    const float a = static_cast<float>(ah);
    const bool up = at & 1;  // a negative top: a positive scale
    if (!(a <= kMaxScale)) {
        scale = 0x7e00;
        for (int j = 0; j < 8; ++j) code[j] = 8;
        return;
    }
    scale = static_cast<uint16_t>(__builtin_bit_cast(uint16_t, ah) | (up ? 0 : 0x8000));
    const float inv = a > 0 ? __builtin_amdgcn_rcpf(a) : 0.0f;
    for (int j = 0; j < 8; ++j) {
        const float x = up ? y[j] : -y[j];
        float n = __builtin_floorf(__builtin_fmaf(x, inv, 8.5f));
        n = __builtin_fminf(__builtin_fmaxf(n, 0.0f), 15.0f);
        n += x >= (n - 7.5f) * a ? 1.0f : x < (n - 8.5f) * a ? -1.0f : 0.0f;
        code[j] = a > 0 ? static_cast<uint32_t>(__builtin_fminf(__builtin_fmaxf(n, 0.0f), 15.0f)) : 8;
    }
}

// A 4 x 4 transposition of bytes in each four lanes: lane j's byte q, of position j, goes to lane q; a
// word's positions in the order 0, 2, 1, 3.
__device__ inline uint32_t transposed(uint32_t w, int lane) {
    const uint32_t a = __builtin_amdgcn_update_dpp(0, w, 0xB1, 0xF, 0xF, true);  // lanes 1, 0, 3, 2
    w = __builtin_amdgcn_perm(a, w, lane & 1 ? 0x03070105 : 0x06020400);
    const uint32_t b = __builtin_amdgcn_update_dpp(0, w, 0x4E, 0xF, 0xF, true);  // lanes 2, 3, 0, 1
    return __builtin_amdgcn_perm(b, w, lane & 2 ? 0x03070206 : 0x05010400);
}

// Where a rotation's pairs are: adjacent, whole blocks apart, or anywhere.
constexpr int kAdjacent = 0, kBlocks = 1, kFar = 2;

// One wave a tile's keys or values: lane 16 g + i has dimensions 32 b + 8 g + 0..7 of position i, for each block b, which is
// how the tile holds keys.  A rotation's pairs lie in one lane where they are adjacent or half the rotated dimensions,
// whole blocks, apart; norms and quantisation cross four lanes, 4-bit values' bytes four others.
// Bound by the latency of what a wave reads: 8190 rows of 8 heads of 64, f32 to 4 bits, take 17 us (3.3 TB/s; 11 at a copy's rate), a call of
// 8000 of 8 heads of 128 with norms, bf16 to fp16, 39 (all reads at once; 46 one after the other), and 48 single tokens, one
// lane in 16, 8, of which a launch is 4.
template <int NB, bool Q4, int PAIRS>
__global__ __launch_bounds__(kThreads) void k_kv_append_tiles(AppendArgs a) {
    constexpr int GS = NB < 4 ? NB : 4, NG = NB / GS, HD = 32 * NB;
    constexpr bool IN_LANE = PAIRS != kFar, NEOX = PAIRS == kBlocks, EARLY = NB <= 8 && IN_LANE;  // (the others have no registers for early loads)
    const int lane = static_cast<int>(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 16, g = lane / 16;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        if (sr.end <= sr.begin) continue;
        const int32_t last = sr.first + (sr.end - sr.begin) - 1, t_lo = sr.first < 0 ? 0 : sr.first / 16, t_hi = last < 0 ? 0 : last / 16 + 1;
        const uint32_t total = (t_hi - t_lo) * a.pairs.d;
        for (uint32_t u = blockIdx.x * 4 + wave; u < total; u += gridDim.x * 4) {
            const uint32_t n = over(u, a.pairs), rest = u - n * a.pairs.d;
            const bool value = rest >= a.kv.kv_heads;
            const uint32_t h = value ? rest - a.kv.kv_heads : rest;
            const int32_t t0 = (t_lo + static_cast<int32_t>(n)) * 16, page = page_of(a.kv, a.b, s, t0), pos = t0 + i;
            const int32_t row = sr.begin + (pos - sr.first);
            const bool live = row >= sr.begin && row < sr.end && (a.rope.table == nullptr || static_cast<uint32_t>(pos) < a.rope.positions);
            const bool full = __all(live);
            if (!__any(live)) continue;
            const HeadRows& from = value ? a.v : a.k;
            const char* head = row_ptr(from, live ? row : sr.begin, h);
            // all that is read is on its way at once: rows, norm weights and the rotation's (cos, sin)
            float y[NB][8];
#pragma unroll
            for (int b = 0; b < NB; ++b) load8(head, from.type, true, 32 * b + 8 * g, y[b]);
            const int dims = static_cast<int>(a.rope.dims);
            const float* cs = !value && a.rope.table != nullptr ? a.rope.table + static_cast<size_t>(live ? pos : 0) * a.rope.dims : nullptr;
            float t[EARLY ? NB : 1][8], wt[EARLY ? NB : 1][8];
            if (EARLY && !value && a.w != nullptr) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    for (int j = 0; j < 8; ++j) wt[EARLY ? b : 0][j] = a.w[32 * b + 8 * g + j];
            }
            if (EARLY && cs != nullptr && IN_LANE) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    // (half a head's blocks of pairs take two blocks of the table each)
                    const int d = NEOX ? b / 2 * 64 + 16 * g + b % 2 * 8 : 32 * b + 8 * g;
                    if (d < dims) load8(cs, kTypeF32, true, d, t[EARLY ? b : 0]);
                }
            }
            if (page < 0) continue;
            uint8_t* tile = a.kv.data + tile_at(a.kv, page, h, t0);
            if (!value && (a.w != nullptr || cs != nullptr)) {
                double scale = 1;
                if (a.w != nullptr) {
                    double sums[4] = {};
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        for (int j = 0; j < 8; ++j) sums[j % 4] = __builtin_fma(static_cast<double>(y[b][j]), static_cast<double>(y[b][j]), sums[j % 4]);
                    double sum = sums[0] + sums[1] + (sums[2] + sums[3]);
                    sum += __shfl_xor(sum, 16);
                    sum += __shfl_xor(sum, 32);
                    scale = 1.0 / sqrt(sum / HD + static_cast<double>(a.eps));
                }
                const auto weighed = [&](float z, float w) { return a.w != nullptr ? static_cast<double>(z) * scale * static_cast<double>(w) : static_cast<double>(z); };
                const auto weight_of = [&](int b, int j) { return EARLY ? wt[EARLY ? b : 0][j] : a.w != nullptr ? a.w[32 * b + 8 * g + j] : 0.0f; };
                const auto plain = [&](int b) {
                    for (int j = 0; j < 8; ++j) y[b][j] = static_cast<float>(weighed(y[b][j], weight_of(b, j)));
                };
                bool turned[NB] = {};  // (of blocks: known where a block's number is)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    int d = 32 * b + 8 * g;
                    if constexpr (!IN_LANE) asm volatile("" : "+v"(d));  // (or the places of all of a head's partners are held in registers)
                    if (NEOX ? turned[b] : false) continue;
                    if (cs == nullptr || (IN_LANE ? !NEOX && d >= dims : 32 * b >= dims)) {
                        plain(b);
                    } else if constexpr (!IN_LANE) {
                        // pairs half the rotated dimensions apart, which another lane has: from the row once more; dimensions
                        // that are not rotated (in this block, of other lanes) go the same way, and are chosen at the end
                        const int half = dims / 2;
                        const bool whole = half % 8 == 0;  // then the partners are eight in a row
                        float other[8];
                        if (whole) {
                            load8(head, from.type, true, d >= dims ? d : d < half ? d + half : d - half, other);
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; ++j) other[j] = load1(head, from.type, d + j >= dims ? d + j : d + j < half ? d + j + half : d + j - half);
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int i = d + j, p = i >= dims ? i : i < half ? i + half : i - half, e = i >= dims ? 0 : i < half ? i : i - half;
                            const double x = weighed(y[b][j], weight_of(b, j)), z = weighed(other[j], a.w != nullptr ? a.w[p] : 0.0f), c = cs[2 * e], si = cs[2 * e + 1];
                            const double r = i < half ? mul_sub(x, c, z, si) : mul_add(z, si, x, c);
                            y[b][j] = static_cast<float>(i < dims ? r : x);
                        }
                        __builtin_amdgcn_sched_barrier(0);  // (a block's loads at a time)
                    } else if constexpr (!NEOX) {
                        float u[8];
                        if constexpr (!EARLY) load8(cs, kTypeF32, true, d, u);
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const double x = weighed(y[b][j], weight_of(b, j)), z = weighed(y[b][j + 1], weight_of(b, j + 1));
                            const double c = EARLY ? t[EARLY ? b : 0][j] : u[j], si = EARLY ? t[EARLY ? b : 0][j + 1] : u[j + 1];
                            y[b][j] = static_cast<float>(mul_sub(x, c, z, si));
                            y[b][j + 1] = static_cast<float>(mul_add(x, si, z, c));
                        }
                    } else {
                        // dims / 64 blocks on: one of the lane's own, known when its number is
#pragma unroll
                        for (int o = 2 * b + 1; o < NB; ++o) {
                            if (dims != 64 * (o - b)) continue;
                            turned[b] = turned[o] = true;
                            float u[16];
                            if constexpr (!EARLY) {
                                load8(cs, kTypeF32, true, 2 * d, reinterpret_cast<float(&)[8]>(u[0]));
                                load8(cs, kTypeF32, true, 2 * d + 8, reinterpret_cast<float(&)[8]>(u[8]));
                            }
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const double c = EARLY ? t[EARLY ? 2 * b + j / 4 : 0][2 * j % 8] : u[2 * j], si = EARLY ? t[EARLY ? 2 * b + j / 4 : 0][2 * j % 8 + 1] : u[2 * j + 1];
                                const double x = weighed(y[b][j], weight_of(b, j)), z = weighed(y[o][j], weight_of(o, j));
                                y[b][j] = static_cast<float>(mul_sub(x, c, z, si));
                                y[o][j] = static_cast<float>(mul_add(x, si, z, c));
                            }
                        }
                        if (!turned[b]) plain(b);
                    }
                }
            }
            if constexpr (!Q4) {
#pragma unroll
                for (int n2 = 0; n2 < NG; ++n2) {
                    uint32_t w[GS][4];
#pragma unroll
                    for (int e = 0; e < GS; ++e)
                        for (int j = 0; j < 4; ++j) w[e][j] = pack_half(y[n2 * GS + e][2 * j], y[n2 * GS + e][2 * j + 1]);
                    if (!live) continue;
                    if (!value) {
#pragma unroll
                        for (int e = 0; e < GS; ++e) *reinterpret_cast<word4v*>(tile + ((n2 * GS + e) * 64 + lane) * 16) = word4v{w[e][0], w[e][1], w[e][2], w[e][3]};
                    } else {
                        uint8_t* to = tile + tile_values_at(false, NB) + ((i % 4 * NG + n2) * 64 + i / 4 * 16 + 4 * g) * GS * 4;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t z[GS];
                            for (int e = 0; e < GS; ++e) z[e] = w[e][j];
                            store_words<GS>(to + j * GS * 4, z);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int n2 = 0; n2 < NG; ++n2) {
                    uint32_t w[GS];
#pragma unroll
                    for (int e = 0; e < GS; ++e) {
                        const int b = n2 * GS + e;
                        uint32_t code[8];
                        uint16_t scale;
                        quantise8_tile(y[b], g, code, scale);
                        w[e] = 0;
                        for (int j = 0; j < 4; ++j)
                            w[e] |= value ? (code[2 * j] | code[2 * j + 1] << 4) << (8 * j) : code[2 * j] << (4 * j) | code[2 * j + 1] << (4 * j + 16);
                        if (live && g == b % 4) *reinterpret_cast<uint16_t*>(tile + scale_offset(NB, value, i, b)) = scale;
                    }
                    if (!value) {
                        if (live) store_words<GS>(tile + (n2 * 64 + lane) * GS * 4, w);
                    } else if (full) {
#pragma unroll
                        for (int e = 0; e < GS; ++e) w[e] = transposed(w[e], lane);
                        store_words<GS>(tile + tile_values_at(true, NB) + (n2 * 64 + i / 4 * 16 + 4 * g + i % 4) * GS * 4, w);
                    } else if (live) {
#pragma unroll
                        for (int e = 0; e < GS; ++e)
                            for (int j = 0; j < 4; ++j)
                                tile[value_offset(true, NB, i, 32 * (n2 * GS + e) + 8 * g + 2 * j)] = static_cast<uint8_t>(w[e] >> (8 * j));
                    }
                }
            }
        }
    }
}

template <int NB, int PAIRS>
hipError_t launch_append_pairs(const AppendArgs& a, dim3 grid, hipStream_t st) {
    if (a.kv.q4) k_kv_append_tiles<NB, true, PAIRS><<<grid, dim3(kThreads), 0, st>>>(a);
    else k_kv_append_tiles<NB, false, PAIRS><<<grid, dim3(kThreads), 0, st>>>(a);
    return hipGetLastError();
}
template <int NB>
hipError_t launch_append(const AppendArgs& a, dim3 grid, hipStream_t st) {
    if (a.rope.table == nullptr || !a.rope.neox) return launch_append_pairs<NB, kAdjacent>(a, grid, st);
    if (a.rope.dims % 64 == 0) return launch_append_pairs<NB, kBlocks>(a, grid, st);
    if constexpr (NB <= 4) return launch_append_pairs<NB, kFar>(a, grid, st);
    return hipErrorInvalidValue;
}

// The inverse of transposed(): a word's positions in the order 0, 2, 1, 3 go to the four lanes, in the order of the dimensions.
__device__ inline uint32_t untransposed(uint32_t w, int lane) {
    w = transposed(__builtin_amdgcn_perm(0, w, 0x03010200), lane);
    return __builtin_amdgcn_perm(0, w, 0x03010200);
}

// A 4 x 4 transposition of words in each four lanes: lane j's word q goes to lane q's word j.
__device__ inline void transpose_words(uint32_t (&x)[4], int lane) {
    for (int r = 0; r < 4; r += 2) {
        const uint32_t t = __builtin_amdgcn_update_dpp(0, lane & 1 ? x[r] : x[r + 1], 0xB1, 0xF, 0xF, true);
        (lane & 1 ? x[r] : x[r + 1]) = t;
    }
    for (int r = 0; r < 2; ++r) {
        const uint32_t t = __builtin_amdgcn_update_dpp(0, lane & 2 ? x[r] : x[r + 2], 0x4E, 0xF, 0xF, true);
        (lane & 2 ? x[r] : x[r + 2]) = t;
    }
}

// One wave a tile's keys or values: loads of the whole of them, as the attention's.  A lane then has eight values of a
// position, of values after a transposition among four lanes, and four lanes write 64 bytes or more of a row,
// past the caches: 4 sequences of 16000 positions, 8 heads of 128 in 4 bits to fp16, take 50 us, less than a
// copy of as many bytes (5.8 TB/s), and through the caches 86.  (Keys and values by one wave: 8 us for 48 single rows in the place of 5.)
template <int NB, bool Q4>
__global__ __launch_bounds__(kThreads) void k_kv_read(ReadArgs a, int vec) {
    constexpr int GS = NB < 4 ? NB : 4, NG = NB / GS;
    const int lane = static_cast<int>(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 16, g = lane / 16;
    const uint32_t sides = a.k.data != nullptr && a.v.data != nullptr ? 2 : 1;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        if (sr.end <= sr.begin) continue;
        const int32_t last = sr.first + (sr.end - sr.begin) - 1, t_lo = sr.first < 0 ? 0 : sr.first / 16, t_hi = last < 0 ? 0 : last / 16 + 1;
        const uint32_t total = (t_hi - t_lo) * a.heads.d * sides;
        for (uint32_t w = blockIdx.x * 4 + wave; w < total; w += gridDim.x * 4) {
            const uint32_t u = w / sides, n = over(u, a.heads), h = u - n * a.heads.d;
            const bool value = sides == 2 ? w % 2 != 0 : a.k.data == nullptr;
            const int32_t t0 = (t_lo + static_cast<int32_t>(n)) * 16, page = page_of(a.kv, a.b, s, t0);
            if (page < 0) continue;
            const uint8_t *tile = a.kv.data + tile_at(a.kv, page, h, t0), *from = tile + tile_values_at(Q4, NB);
            uint32_t k[NG][Q4 ? 1 : GS][Q4 ? GS : 4], v[NG][Q4 ? 1 : 4][GS], vs[NG][Q4 ? 2 * GS : 1];
            uint16_t ks[Q4 ? NB : 1];
            if (!value) {
#pragma unroll
                for (int m = 0; m < NG; ++m) {
                    if constexpr (Q4) {
                        load_words<GS>(tile + (m * 64 + lane) * GS * 4, k[m][0]);
                        for (int e = 0; e < GS; ++e) ks[m * GS + e] = *reinterpret_cast<const uint16_t*>(tile + scale_offset(NB, false, i, m * GS + e));
                    } else {
                        for (int e = 0; e < GS; ++e) load_words<4>(tile + ((m * GS + e) * 64 + lane) * 16, k[m][e]);
                    }
                }
            }
            if (value) {
#pragma unroll
                for (int m = 0; m < NG; ++m) {
                    if constexpr (Q4) {
                        load_words<GS>(from + (m * 64 + lane) * GS * 4, v[m][0]);
                        load_words<2 * GS>(tile + tile_value_scales_at(NB) + (g * NB + m * GS) * 8, vs[m]);
                    } else {
                        for (int r = 0; r < 4; ++r) load_words<GS>(from + ((r * NG + m) * 64 + lane) * GS * 4, v[m][r]);
                    }
                }
            }
            const int32_t row0 = sr.begin + (t0 - sr.first);  // of the tile's first position; rows before sr.begin are not there
            const auto to = [&](int32_t row, const HeadRows& y) -> char* { return row >= sr.begin && row < sr.end ? row_ptr(y, row, h) : nullptr; };
            if (!value) {
                char* out = to(row0 + i, a.k);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float x[8];
                    if constexpr (Q4) key_codes(k[b / GS][0][b % GS], from_half(ks[b]), x);
                    else halves8(k[b / GS][b % GS], x);
                    if (out != nullptr) store8<true>(out, a.k.type, vec & 1, 32 * b + 8 * g, x);
                }
            }
            if (value) {
                char* out = to(row0 + 4 * g + i % 4, a.v);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int m = b / GS, e = b % GS;
                    float x[8];
                    if constexpr (Q4) {
                        const uint32_t c = untransposed(v[m][0][e], lane);
                        const float d = from_half(vs[m][2 * e + i % 4 / 2] >> (i % 2 * 16) & 0xFFFF);
                        for (int j = 0; j < 8; ++j) x[j] = (static_cast<float>(c >> (4 * j) & 15) - 8) * d;
                    } else {
                        uint32_t t[4] = {v[m][0][e], v[m][1][e], v[m][2][e], v[m][3][e]};
                        transpose_words(t, lane);
                        halves8(t, x);
                    }
                    if (out != nullptr) store8<true>(out, a.v.type, vec & 2, 32 * b + i / 4 * 8, x);
                }
            }
        }
    }
}

template <int NB>
hipError_t launch_read(const ReadArgs& a, dim3 grid, int vec, hipStream_t st) {
    if (a.kv.q4) k_kv_read<NB, true><<<grid, dim3(kThreads), 0, st>>>(a, vec);
    else k_kv_read<NB, false><<<grid, dim3(kThreads), 0, st>>>(a, vec);
    return hipGetLastError();
}

// Blocks for the tiles that a sequence's rows may touch, a wave each for `units` of a tile.
dim3 tile_grid(const PagedBatch& b, uint64_t units) {
    const uint64_t most = b.max_rows == 0 || b.max_rows > b.rows ? b.rows : b.max_rows, tiles = (most + 14) / 16 + 1;
    const uint64_t y = std::min<uint64_t>(b.seqs, 65535), x = std::min<uint64_t>((tiles * units + 3) / 4, std::max<uint64_t>(1, (1 << 18) / y));
    return dim3(static_cast<uint32_t>(x), static_cast<uint32_t>(y));
}

// Blocks along a sequence's rows: enough for the largest, not many more than fill the card.
dim3 row_grid(const PagedBatch& b, uint64_t heads, int lanes) {
    const uint64_t per = kThreads / lanes, most = b.max_rows == 0 || b.max_rows > b.rows ? b.rows : b.max_rows;
    const uint64_t y = std::min<uint64_t>(b.seqs, 65535);
    uint64_t x = (most * heads * 2 + per - 1) / per;
    x = std::min<uint64_t>(x, std::max<uint64_t>(1, 65536 / y));
    return dim3(static_cast<uint32_t>(std::max<uint64_t>(1, x)), static_cast<uint32_t>(y));
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t st) {
    const int lanes = head_lanes(a.head_dim);
    int vec = 0;
    for (int t = 0; t < 2; ++t) {
        if (a.x[t].data == nullptr) continue;
        vec |= (wide(a.x[t]) ? 1 << t : 0) | (wide(a.y[t]) ? 4 << t : 0);
    }
    const size_t per = kThreads / lanes, total = a.n * a.all.d;
    const size_t blocks = std::min<size_t>((total + per - 1) / per, 1 << 20);
    k_norm_rope<<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, st>>>(a, lanes, vec);
    return hipGetLastError();
}

hipError_t launch_kv_append(const AppendArgs& a, hipStream_t st) {
    // By tiles where rows and the table are read 16 bytes at a time, and registers hold a rotation across lanes; otherwise row by row
    // (2653 rows of three sequences, 16 heads of 96 in 4 bits, 24 dimensions rotated: 160 us so, and 75 by tiles).
    const bool far = a.rope.table != nullptr && a.rope.neox && a.rope.dims % 64 != 0;
    const bool wide_table = a.rope.table == nullptr || (reinterpret_cast<uintptr_t>(a.rope.table) % 16 == 0 && a.rope.dims % 8 == 0);
    if (wide(a.k) && wide(a.v) && (far ? a.kv.head_dim <= 128 : wide_table)) {
        const dim3 grid = tile_grid(a.b, a.pairs.d);
        switch (a.kv.head_dim / 32) {
            case 2: return launch_append<2>(a, grid, st);
            case 3: return launch_append<3>(a, grid, st);
            case 4: return launch_append<4>(a, grid, st);
            case 8: return launch_append<8>(a, grid, st);
            case 16: return launch_append<16>(a, grid, st);
        }
    }
    const int lanes = head_lanes(a.kv.head_dim);
    const int vec = (wide(a.k) ? 1 : 0) | (wide(a.v) ? 2 : 0);
    k_kv_append<<<row_grid(a.b, a.kv.kv_heads, lanes), dim3(kThreads), 0, st>>>(a, lanes, vec);
    return hipGetLastError();
}

hipError_t launch_kv_read(const ReadArgs& a, hipStream_t st) {
    const int vec = (a.k.data != nullptr && wide(a.k) ? 1 : 0) | (a.v.data != nullptr && wide(a.v) ? 2 : 0);
    const dim3 grid = tile_grid(a.b, static_cast<uint64_t>(a.kv.kv_heads) * (a.k.data != nullptr && a.v.data != nullptr ? 2 : 1));
    switch (a.kv.head_dim / 32) {
        case 2: return launch_read<2>(a, grid, vec, st);
        case 3: return launch_read<3>(a, grid, vec, st);
        case 4: return launch_read<4>(a, grid, vec, st);
        case 8: return launch_read<8>(a, grid, vec, st);
        case 16: return launch_read<16>(a, grid, vec, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace bh
