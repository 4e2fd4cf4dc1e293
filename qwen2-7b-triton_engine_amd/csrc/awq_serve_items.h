// How attention over the paged cache is cut into items (csrc/awq_serve_attention.hip):
// the arithmetic that its kernels, their grids and the workspace have in common.
// Plain C++ without the HIP headers (constexpr functions are the device's too), so that
// tests/test_attention_items.py runs it on the host: every item has to have a
// workgroup, and every item that is one of several a place for its sums.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace awq {

constexpr int kCols = 16;              // (row, query head) pairs of a decode workgroup: the columns of an MFMA
constexpr int kWaveKeys = 32;          // tokens of one inner pass of a decode wave
constexpr int kKeys = 4 * kWaveKeys;   // of a decode workgroup's four waves
constexpr int kTileKeys = 64;          // tokens of a tile kernel's step
constexpr int kTileCols = 64;          // columns of a tile workgroup, 16 a wave

// Items that a launch aims at, all kv heads together.  Decode: three workgroups on each
// of 256 CUs, one round of them.  512 / 768 / 1024: 64 requests of up to 4096 tokens 44.1 /
// 36.1 / 39.5 us, 16 of up to 16000 37.4 / 30.7 / 34.8, one of 16000 14.7 / 15.0 / 15.8.
constexpr int kDecodeItems = 768;
// Tiles, only where the blocks of columns are fewer than CUs: 256 / 512 / 1024 items for
// 3 chunks of up to 389 rows behind up to 4000 tokens, heads of 64, 120 / 61 / 54 us.  Prompts with more
// blocks than that are not split: one of 1024 tokens 40 us whole and 57 split, 1777 78 and 110, 4096 277 and
// 309 (partial sums of every row).
constexpr int kTileItems = 1024, kSplitBelow = 256;
// A request of more columns goes to the tile kernel.  8 requests of 4000 tokens each, all by
// the decode kernel / by the tile kernel: 56 columns 33.0 / 35.1 us, 112 46.8 / 46.3, 224 92 / 66, 448
// 123 / 123 (there the tiles' blocks are as many as CUs and not split); of 2200 tokens on average 25.8 /
// 28.7, 38.3 / 32.9, 56 / 49, 92 / 121.
constexpr int kDecodeColumns = 128;

// The rows of a request in a batch of `total`, from its entries of query_start: the first,
// given the largest of the starts before it (0 of none), and the one past the last.  A start below
// an earlier one counts as that one, so no row is two requests' and all of them have
// `total` rows at most: the plan below counts on it.
constexpr int row_in(int start, int total) { return start < 0 ? 0 : start < total ? start : total; }
constexpr int first_row(int before, int lo, int total) { return before > row_in(lo, total) ? before : row_in(lo, total); }
constexpr int end_row(int row0, int hi, int total) { return hi < row0 ? row0 : hi < total ? hi : total; }

// Tokens to walk over: one past the table where the length is (that one is not
// there, and gives NaN).  A table holds 2^30 tokens at most: 32 bits do.
constexpr int walked_tokens(int width, int page_log2, int len) {
    const int past = (width << page_log2) + 1;
    return len < past ? len : past;
}

// Columns of a request that are computed, its blocks of them in this kernel (COLS says
// which), its tokens in steps.  limit: columns up to which a request is the decode kernel's.
constexpr int request_columns(int rows, int max_query, int group) { return (rows < max_query ? rows : max_query) * group; }
template <int COLS>
constexpr int request_blocks(int columns, int limit) {
    const bool mine = (columns <= limit) == (COLS == kCols);
    return mine ? (int)((uint32_t)(columns + COLS - 1) / COLS) : 0;
}
template <int KEYS>
constexpr int request_steps(int walked) { return (int)((uint32_t)(walked + KEYS - 1) / KEYS); }

// Steps of an item: as few as `target` items in all allow, from the sums over all
// requests of blocks times steps and of blocks.  At most target + the blocks come out.
// Without a target, and where even `target` items would have more than any request has,
// an item has all of its request's: the grid has no place for more, and without a target the
// workspace none for sums.
template <int KEYS>
constexpr int item_steps(int target, int64_t work, int all_blocks, int requests) {
    constexpr int kMost = (1 << 30) / KEYS + 1;          // of a request: 2^30 tokens, and one past the table
    if (!target) return kMost;
    // Each block ends in a shorter item, half of one too many on average: with as many
    // fewer to begin with, the items are one round of workgroups.
    const int extra = requests == 1 ? 0 : all_blocks / 2;
    target = extra < target - target / 4 ? target - extra : (target + 3) / 4;
    const int64_t most = (int64_t)target * kMost;
    const uint32_t few = work < 0x7FFFFFFF - target ? (uint32_t)(work + target - 1) / (uint32_t)target : 0;
    return few ? (few < (uint32_t)kMost ? (int)few : kMost)
               : work == 0 ? 1 : work < most ? (int)((work + target - 1) / target) : kMost;
}
constexpr int request_splits(int steps, int item) { return (int)((uint32_t)(steps + item - 1) / (uint32_t)item); }
// Where an item ends that begins at `start`, of a block that sees `limit` tokens.
constexpr int item_end(int start, int chunk, int limit) {
    return limit - start < chunk ? limit : start + chunk;   // start + chunk may pass 32 bits where limit does not
}

struct AttentionPlan {
    bool decode, tile, combine;
    int limit, decode_target, tile_target;
    int64_t decode_items, tile_items;  // at most, of one kv head
    size_t part_floats(int kvh, int hd) const {          // the items' sums
        return (size_t)(decode_items * kCols + (tile_target ? tile_items * kTileCols : 0)) * kvh * (hd + 2);
    }
};
inline AttentionPlan attention_plan(int requests, int total, int max_query, int group, int kvh) {
    AttentionPlan p = {};
    const int64_t rows = (int64_t)requests * max_query < total ? (int64_t)requests * max_query : total;
    p.tile = (int64_t)max_query * group > kDecodeColumns;
    p.decode = !p.tile || requests > 1;
    p.limit = p.decode ? kDecodeColumns : 0;             // of one request the tile kernel has whatever it is
    if (p.decode) {
        p.decode_target = kvh < kDecodeItems ? kDecodeItems / kvh : 1;
        const int64_t most = (int64_t)requests * ((kDecodeColumns + kCols - 1) / kCols);
        const int64_t blocks = requests + rows * group / kCols;
        p.decode_items = p.decode_target + (p.tile && most < blocks ? most : blocks) + 1;
    }
    if (p.tile) {
        const int64_t blocks = requests + rows * group / kTileCols;
        p.tile_target = blocks * kvh < kSplitBelow ? (kvh < kTileItems ? kTileItems / kvh : 1) : 0;
        p.tile_items = blocks + p.tile_target + 1;
    }
    p.combine = p.decode || p.tile_target;
    return p;
}

}  // namespace awq
