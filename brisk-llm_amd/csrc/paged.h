// The paged key/value cache: its layout, the batch that addresses it, and the launchers of its kernels.
//
// A page holds page_tokens positions of every key/value head.  Its unit is the tile: 16 positions
// of one head, keys and values, in the order in which a wave's lanes hold the operands of
// v_mfma_f32_16x16x32_f16, so that a lane's operand is one wide load and a wave's load is
// contiguous.  With nb = head_dim / 32 blocks a row, lane l = 16 g + i (i < 16, g < 4), and blocks
// taken gs = min(nb, 4) at a time:
//
//   F16   keys    [block][l][8]             position i, dimensions 32 block + 8 g + 0..7
//         values  [r][block / gs][l][gs][2] position 4 g + r, dimensions 32 block + 2 i + 0..1
//   Q4_0  keys    [block / gs][l][gs] words position i, dimensions 32 block + 8 g + 0..7: dimension
//                                           2 m in the word's nibble m, 2 m + 1 in nibble m + 4
//         values  [block / gs][l][gs] words positions 4 g + 0..3, dimensions 32 block + 2 i (low
//                                           nibbles) and + 1 (high): bytes of positions 0, 2, 1, 3
//         scales of the keys, then of the values: [g][block][4] halves, positions 4 g + 0..3
//
// Tiles of a page follow each other as [kv_head][page_tokens / 16].  The functions that find a
// position's place are compiled for the host too.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define BH_BOTH __host__ __device__ inline
#else
#define BH_BOTH inline
#endif

namespace bh {

constexpr uint32_t kTileTokens = 16;
constexpr uint32_t kMaxPageTokens = 1024;
constexpr uint32_t kMaxPagedHead = 512;

// The largest 4-bit scale that is kept: eight times it is a half's largest value, so a code's product
// with it stays finite in 16 bits.
constexpr float kMaxScale = 8188.0f;

constexpr int kTypeF32 = 0, kTypeF16 = 1, kTypeQ4 = 2, kTypeBF16 = 30;

// A [rows][heads][head_dim] tensor: strides in elements, a head's values contiguous.
struct HeadRows {
    void* data;
    int type;
    int64_t row, head;
};

struct RopeTable {
    const float* table;  // [positions][dims / 2] (cos, sin); null: no rotation
    uint32_t positions, dims;
    int neox;            // pairs (i, i + dims / 2); otherwise (2 i, 2 i + 1)
};

struct PagedKv {
    uint8_t* data;
    int q4;
    uint32_t kv_heads, head_dim, page_tokens, pages;
    uint32_t page_shift;
};

// Sequence s has rows row_start[s] .. row_start[s + 1] - 1: its last positions, lengths[s] in all.
struct PagedBatch {
    const int32_t* row_start;
    const int32_t* lengths;
    const int32_t* page_table;  // [seqs][page_stride]
    uint32_t seqs, rows, page_stride, max_rows, max_length;
};

BH_BOTH uint32_t group_blocks(uint32_t nb) { return nb < 4 ? nb : 4; }
BH_BOTH uint32_t tile_bytes(bool q4, uint32_t nb) { return q4 ? 576 * nb : 2048 * nb; }
BH_BOTH uint32_t tile_values_at(bool q4, uint32_t nb) { return q4 ? 256 * nb : 1024 * nb; }
BH_BOTH uint32_t tile_key_scales_at(uint32_t nb) { return 512 * nb; }
BH_BOTH uint32_t tile_value_scales_at(uint32_t nb) { return 544 * nb; }

// A sequence's rows in the batch's tensors and their positions.  A row table that is out of order or
// past the tensors gives no rows outside them; positions stay below kMaxLength.
constexpr int32_t kMaxLength = 0x7FFFFC00;
struct SeqRows {
    int32_t begin, end;  // rows of the tensors
    int32_t first;       // position of row `begin`; negative positions hold nothing
};
BH_BOTH SeqRows seq_rows(const PagedBatch& b, uint32_t s) {
    const int32_t lo = b.row_start[s], hi = b.row_start[s + 1], n = b.lengths[s];
    const int32_t length = n < 0 ? 0 : n > kMaxLength ? kMaxLength : n, rows = static_cast<int32_t>(b.rows);
    SeqRows q;
    q.begin = lo < 0 ? 0 : lo;
    q.end = hi > rows ? rows : hi;
    if (q.end < q.begin) q.end = q.begin;
    q.first = length - (hi < q.begin ? 0 : hi - q.begin);
    return q;
}

// The page of a position, or -1: a position outside the table's row, or an entry that names no page.
BH_BOTH int32_t page_of(const PagedKv& kv, const PagedBatch& b, uint32_t s, int32_t pos) {
    if (pos < 0) return -1;
    const uint32_t e = static_cast<uint32_t>(pos) >> kv.page_shift;
    if (e >= b.page_stride) return -1;
    const int32_t p = b.page_table[static_cast<size_t>(s) * b.page_stride + e];
    return p < 0 || static_cast<uint32_t>(p) >= kv.pages ? -1 : p;
}

// Byte offset of the tile of position `pos` of head h in page `page`.
BH_BOTH size_t tile_at(const PagedKv& kv, int32_t page, uint32_t h, int32_t pos) {
    const uint32_t t = (static_cast<uint32_t>(pos) & (kv.page_tokens - 1)) / kTileTokens;
    return ((static_cast<size_t>(static_cast<uint32_t>(page)) * kv.kv_heads + h) * (kv.page_tokens / kTileTokens) + t) * tile_bytes(kv.q4 != 0, kv.head_dim / 32);
}

// Offsets in a tile.  `d` is a multiple of 8 for the keys (eight values: 16 bytes, or a word) and of
// 2 for the values (two values: 4 bytes, or a byte).
BH_BOTH uint32_t key_offset(bool q4, uint32_t nb, uint32_t token, uint32_t d) {
    const uint32_t gs = group_blocks(nb), b = d / 32, l = d % 32 / 8 * 16 + token;
    return q4 ? ((b / gs * 64 + l) * gs + b % gs) * 4 : (b * 64 + l) * 16;
}
BH_BOTH uint32_t value_offset(bool q4, uint32_t nb, uint32_t token, uint32_t d) {
    const uint32_t gs = group_blocks(nb), b = d / 32, l = token / 4 * 16 + d % 32 / 2, r = token % 4;
    if (!q4) return tile_values_at(false, nb) + (((r * (nb / gs) + b / gs) * 64 + l) * gs + b % gs) * 4;
    return tile_values_at(true, nb) + ((b / gs * 64 + l) * gs + b % gs) * 4 + ((r & 1) << 1 | r >> 1);
}
BH_BOTH uint32_t scale_offset(uint32_t nb, bool value, uint32_t token, uint32_t b) {
    return (value ? tile_value_scales_at(nb) : tile_key_scales_at(nb)) + ((token / 4 * nb + b) * 4 + token % 4) * 2;
}

// Division of numbers below 2^31 by a divisor known when a kernel is launched: n * m >> s with m =
// ceil(2^s / d) and s = 31 + ceil(log2 d), which is exact there.
struct Divisor {
    uint32_t d, m, s;
};
BH_BOTH Divisor divisor(uint32_t d) {
    uint32_t s = 31;
    while ((uint64_t{1} << (s - 31)) < d) ++s;
    return {d, static_cast<uint32_t>(((uint64_t{1} << s) + d - 1) / d), s};
}
BH_BOTH uint32_t over(uint32_t n, const Divisor& d) { return static_cast<uint32_t>(static_cast<uint64_t>(n) * d.m >> d.s); }

#ifdef __HIPCC__

struct NormRopeArgs {
    HeadRows x[2], y[2];    // queries and keys; x[1].data null: no keys
    const float* w[2];      // norm weights, or null
    uint32_t heads[2], head_dim;
    Divisor all;  // heads a row, of both
    size_t n;
    float eps;
    RopeTable rope;
    const int32_t* positions;
};
hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t st);

struct AppendArgs {
    PagedKv kv;
    PagedBatch b;
    HeadRows k, v;
    Divisor pairs;   // 2 x key/value heads
    const float* w;  // the keys' norm weights, or null
    float eps;
    RopeTable rope;
};
hipError_t launch_kv_append(const AppendArgs& a, hipStream_t st);

struct ReadArgs {
    PagedKv kv;
    PagedBatch b;
    HeadRows k, v;  // data null: not wanted
    Divisor heads;  // key/value heads
};
hipError_t launch_kv_read(const ReadArgs& a, hipStream_t st);

struct PagedAttnArgs {
    PagedKv kv;
    PagedBatch b;
    HeadRows q, out;
    uint32_t heads;
    Divisor group, per_row, kv_heads;  // query heads of a key/value head, query heads, key/value heads
    float scale;
    uint32_t window;  // 0: none
    uint32_t splits;  // parts of the positions (set by the launcher, as `per`, the steps of one)
    int32_t per;
    float* part;      // [rows][heads][splits][head_dim], then [rows][heads][splits][2] (maximum, sum)
};
// The workspace for the parts that positions are split into.
size_t paged_workspace(const PagedKv& kv, const PagedBatch& b, uint32_t heads);  // (for either precision)
hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t st);
// The prompts' kernel: the columns, (row, head) pairs of a key/value head, of its workgroup, and whether it takes a head size.
uint32_t prompt_columns(uint32_t head_dim, bool exact);
bool prompt_fits(uint32_t head_dim, bool exact);
hipError_t launch_paged_prompt(const PagedAttnArgs& a, bool exact, uint32_t max_rows, hipStream_t st);

#endif  // __HIPCC__

}  // namespace bh
