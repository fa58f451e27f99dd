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

// One group of lanes a head.  A head's lanes read all they need before they write, so y may be x.
__global__ __launch_bounds__(kThreads) void k_norm_rope(NormRopeArgs a, int lanes, int vec) {
    const int lane = static_cast<int>(threadIdx.x) % lanes, d = lane * 8;
    const size_t per = kThreads / lanes, all = a.heads[0] + (a.x[1].data != nullptr ? a.heads[1] : 0), total = a.n * all;
    // the shuffles of a group want its whole wave in the loop: the bound is the block's first head
    for (size_t base = blockIdx.x * per; base < total; base += static_cast<size_t>(gridDim.x) * per) {
        const size_t u = base + threadIdx.x / lanes;
        const bool in = u < total;
        const size_t row = in ? u / all : 0;
        uint32_t h = in ? static_cast<uint32_t>(u % all) : 0;
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
    const int64_t per = kThreads / lanes, heads = a.kv.kv_heads;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        const int64_t total = static_cast<int64_t>(sr.end - sr.begin) * heads * 2;
        for (int64_t base = blockIdx.x * per; base < total; base += static_cast<int64_t>(gridDim.x) * per) {
            const int64_t u = base + threadIdx.x / lanes;
            const bool in = u < total;
            const int64_t row = sr.begin + (in ? u / (2 * heads) : 0);
            const uint32_t h = in ? static_cast<uint32_t>(u % heads) : 0;
            const bool value = in && u % (2 * heads) >= heads;
            const int32_t pos = sr.first + static_cast<int32_t>(row - sr.begin);
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

// One group of lanes a row's head of keys, then of values.
__global__ __launch_bounds__(kThreads) void k_kv_read(ReadArgs a, int lanes, int vec) {
    const int lane = static_cast<int>(threadIdx.x) % lanes, d = lane * 8;
    const uint32_t nb = a.kv.head_dim / 32;
    if (d >= static_cast<int>(a.kv.head_dim)) return;
    const int64_t per = kThreads / lanes, heads = a.kv.kv_heads;
    for (uint32_t s = blockIdx.y; s < a.b.seqs; s += gridDim.y) {
        const SeqRows sr = seq_rows(a.b, s);
        const int64_t total = static_cast<int64_t>(sr.end - sr.begin) * heads * 2;
        for (int64_t u = blockIdx.x * per + threadIdx.x / lanes; u < total; u += static_cast<int64_t>(gridDim.x) * per) {
            const int64_t row = sr.begin + u / (2 * heads);
            const uint32_t h = static_cast<uint32_t>(u % heads);
            const bool value = u % (2 * heads) >= heads;
            const HeadRows& y = value ? a.v : a.k;
            const int32_t pos = sr.first + static_cast<int32_t>(row - sr.begin), page = page_of(a.kv, a.b, s, pos);
            if (y.data == nullptr || page < 0) continue;
            const uint8_t* tile = a.kv.data + tile_at(a.kv, page, h, pos);
            const uint32_t token = static_cast<uint32_t>(pos) % kTileTokens;
            float out[8];
            read8(tile, a.kv.q4 != 0, nb, value, token, d, out);
            store8(row_ptr(y, row, h), y.type, vec & (value ? 2 : 1), d, out);
        }
    }
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
    const size_t per = kThreads / lanes, total = a.n * (a.heads[0] + (a.x[1].data != nullptr ? a.heads[1] : 0));
    const size_t blocks = std::min<size_t>((total + per - 1) / per, 1 << 20);
    k_norm_rope<<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, st>>>(a, lanes, vec);
    return hipGetLastError();
}

hipError_t launch_kv_append(const AppendArgs& a, hipStream_t st) {
    const int lanes = head_lanes(a.kv.head_dim);
    const int vec = (wide(a.k) ? 1 : 0) | (wide(a.v) ? 2 : 0);
    k_kv_append<<<row_grid(a.b, a.kv.kv_heads, lanes), dim3(kThreads), 0, st>>>(a, lanes, vec);
    return hipGetLastError();
}

hipError_t launch_kv_read(const ReadArgs& a, hipStream_t st) {
    const int lanes = head_lanes(a.kv.head_dim);
    const int vec = (a.k.data != nullptr && wide(a.k) ? 1 : 0) | (a.v.data != nullptr && wide(a.v) ? 2 : 0);
    k_kv_read<<<row_grid(a.b, a.kv.kv_heads, lanes), dim3(kThreads), 0, st>>>(a, lanes, vec);
    return hipGetLastError();
}

}  // namespace bh
