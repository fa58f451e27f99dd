// Device helpers of the paged-cache kernels: rows of any type, and values of a tile.
#pragma once

#include "paged.h"

namespace bh {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef uint32_t word2v __attribute__((ext_vector_type(2)));
typedef uint32_t word4v __attribute__((ext_vector_type(4)));

__device__ inline char* row_ptr(const HeadRows& x, int64_t row, int64_t head) {
    return static_cast<char*>(x.data) + (row * x.row + head * x.head) * (x.type == kTypeF32 ? 4 : 2);
}

// A sequence's pages of one key/value head, for positions that are the same for the whole wave, not before 0, in a
// table that is not empty: a scalar load and no branch.  Past the table's end the last entry is given: no row sees
// such positions.
struct WavePages {
    typedef const __attribute__((address_space(4))) int32_t* Table;
    Table table;
    const uint8_t* head;  // the head's tiles of page 0
    uint32_t last, shift, mask, pages, page_bytes;
    __device__ inline WavePages(const PagedKv& kv, const PagedBatch& b, uint32_t s, uint32_t h) {
        const uint32_t bytes = tile_bytes(kv.q4 != 0, kv.head_dim / 32), per = kv.page_tokens / kTileTokens;
        table = (Table)(uintptr_t)(b.page_table + static_cast<size_t>(s) * b.page_stride);
        last = b.page_stride - 1;
        shift = kv.page_shift;
        mask = kv.page_tokens - 1;
        pages = kv.pages;
        page_bytes = kv.kv_heads * per * bytes;  // (at most 2^31: 1024 heads of 64 tiles of 32 KB)
        head = kv.data + static_cast<size_t>(h) * per * bytes;
    }
    // The page, or one past all pages.
    __device__ inline uint32_t page(int32_t pos) const {
        const uint32_t e = static_cast<uint32_t>(pos) >> shift;
        return static_cast<uint32_t>(table[e < last ? e : last]);
    }
    __device__ inline bool there(uint32_t p) const { return p < pages; }
    // The tile of a position of a page; of page 0 where there is none.
    __device__ inline const uint8_t* tile(uint32_t p, int32_t pos, uint32_t bytes) const {
        return head + static_cast<uint64_t>(p < pages ? p : 0) * page_bytes + (static_cast<uint32_t>(pos) & mask) / kTileTokens * bytes;
    }
};

__device__ inline float from_bf16(uint32_t b) { return __builtin_bit_cast(float, b << 16); }
__device__ inline float from_half(uint32_t h) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h))); }
__device__ inline uint32_t to_half(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }
// Round to nearest, ties to even; a NaN stays one.
__device__ inline uint32_t to_bf16(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    if (x != x) return u >> 16 | 0x40;
    return (u + 0x7FFF + (u >> 16 & 1)) >> 16;
}
__device__ inline uint32_t pack_half(float lo, float hi) { return to_half(lo) | to_half(hi) << 16; }

__device__ inline float load1(const void* head, int type, int d) {
    if (type == kTypeF32) return static_cast<const float*>(head)[d];
    const uint32_t u = static_cast<const uint16_t*>(head)[d];
    return type == kTypeF16 ? from_half(u) : from_bf16(u);
}

__device__ inline void load8(const void* head, int type, bool vec, int d, float (&x)[8]) {
    if (!vec) {
        for (int j = 0; j < 8; ++j) x[j] = load1(head, type, d + j);
        return;
    }
    if (type == kTypeF32) {
        const float4v *p = reinterpret_cast<const float4v*>(static_cast<const float*>(head) + d), a = p[0], b = p[1];
        for (int j = 0; j < 4; ++j) {
            x[j] = a[j];
            x[4 + j] = b[j];
        }
        return;
    }
    const word4v w = *reinterpret_cast<const word4v*>(static_cast<const uint16_t*>(head) + d);
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = type == kTypeF16 ? from_half(w[j] & 0xFFFF) : from_bf16(w[j] & 0xFFFF);
        x[2 * j + 1] = type == kTypeF16 ? from_half(w[j] >> 16) : from_bf16(w[j] >> 16);
    }
}

// PAST: past the caches, for rows that are written in pieces and not read again soon.
template <bool PAST, typename T>
__device__ inline void store(T* p, T x) {
    if constexpr (PAST) __builtin_nontemporal_store(x, p);
    else *p = x;
}

template <bool PAST = false>
__device__ inline void store8(void* head, int type, bool vec, int d, const float (&x)[8]) {
    if (type == kTypeF32) {
        float* p = static_cast<float*>(head) + d;
        if (vec) {
            store<PAST>(reinterpret_cast<float4v*>(p), float4v{x[0], x[1], x[2], x[3]});
            store<PAST>(reinterpret_cast<float4v*>(p + 4), float4v{x[4], x[5], x[6], x[7]});
        } else {
            for (int j = 0; j < 8; ++j) p[j] = x[j];
        }
        return;
    }
    uint32_t u[8];
    for (int j = 0; j < 8; ++j) u[j] = type == kTypeF16 ? to_half(x[j]) : to_bf16(x[j]);
    uint16_t* p = static_cast<uint16_t*>(head) + d;
    if (vec) {
        store<PAST>(reinterpret_cast<word4v*>(p), word4v{u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16});
    } else {
        for (int j = 0; j < 8; ++j) p[j] = static_cast<uint16_t>(u[j]);
    }
}

// Probabilities are held as 2^kLift p relative to a maximum that is renewed once it is passed by
// 2^kLazy: at most 2^15 as halves, and those of a half's smallest steps 2^-31 of the largest.
constexpr float kLazy = 8.0f, kLift = 7.0f;

// The factor of sums relative to maximum m once it is `next`.  Never 0, so that an infinity stays one.
__device__ inline float weight(float m, float next) {
    return __builtin_fmaxf(__builtin_amdgcn_exp2f(m - (next == -__builtin_inff() ? 0.0f : next)), 1.17549435e-38f);
}

// A column's running maximum: a raw score's, and times its scale.  A score's exponent is one fused operation, x scale -
// base; for a scaled maximum past 2^20, whose rounding error would be an exponent of its own, the scores are
// first moved by the maximum.
struct Maximum {
    float raw = -__builtin_inff(), m = -__builtin_inff(), base = 0, shift = 0;
    bool far = false;  // whether some column of the wave is
    // The factor of what has been summed, with a new score's maximum.
    __device__ inline float renew(float top, float scale) {
        raw = __builtin_fmaxf(raw, top);
        const float next = raw * scale, f = weight(m, next);
        m = next;
        const bool none = m == -__builtin_inff(), mine = !none && __builtin_fabsf(m) > 1048576.0f;
        shift = mine ? raw : 0.0f;
        base = none ? 0.0f : mine ? -kLift : m - kLift;
        far = __any(mine);
        return f;
    }
};

__device__ inline half8v operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(half8v, word4v{a, b, c, d}); }
__device__ inline float4v mfma(half8v a, half8v b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline float16v mfma(half8v a, half8v b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
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
// Values that are not finite are kept out of a product, where a probability of 0 (a position that a column does not
// see, or one rounded to 0) would make them NaN, and added by two products of marks against 1 for each
// position a column sees: 32768 for an infinity or NaN, and for a minus infinity or NaN.
struct Marks {
    uint32_t up, down, rest;  // two halves each
};
__device__ inline Marks marks(uint32_t w) {
    const uint32_t i = ill<false>(w) & kIll, sign = w & kIll, nan = (((w & 0x03FF03FF) + 0x03FF03FF) & 0x04000400) << 5;
    return {((i & (~sign | nan)) >> 15) * 0x7800, ((i & (sign | nan)) >> 15) * 0x7800, w & ~((i >> 15) * 0xFFFF)};
}
// (each product is rounded, to an infinity or 0: a fused one would not be)
__device__ inline float ill_sum(float up, float down) { return up * 3e38f - down * 3e38f; }
__device__ inline Marks scale_marks(uint32_t w) {  // blocks without a scale are NaN
    const uint32_t i = (ill<true>(w) & kIll) >> 15;
    return {i * 0x7800, i * 0x7800, w & ~(i * 0xFFFF)};
}

template <int N, int ALIGN>
struct alignas(ALIGN) Words {
    uint32_t w[N];
};
template <int N, int ALIGN = N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4>
__device__ inline void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    const Words<N, ALIGN> x = *reinterpret_cast<const Words<N, ALIGN>*>(p);
    for (int k = 0; k < N; ++k) w[k] = x.w[k];
}

template <int N, int ALIGN = N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4>
__device__ inline void store_words(uint8_t* p, const uint32_t (&w)[N]) {
    Words<N, ALIGN> x;
    for (int k = 0; k < N; ++k) x.w[k] = w[k];
    *reinterpret_cast<Words<N, ALIGN>*>(p) = x;
}

// Eight halves.
__device__ inline void halves8(const uint32_t (&w)[4], float (&x)[8]) {
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = from_half(w[j] & 0xFFFF);
        x[2 * j + 1] = from_half(w[j] >> 16);
    }
}

// The eight keys of a word of codes.
__device__ inline void key_codes(uint32_t w, float scale, float (&x)[8]) {
    for (int m = 0; m < 4; ++m) {
        x[2 * m] = (static_cast<float>(w >> (4 * m) & 15) - 8) * scale;
        x[2 * m + 1] = (static_cast<float>(w >> (4 * m + 16) & 15) - 8) * scale;
    }
}

}  // namespace bh
