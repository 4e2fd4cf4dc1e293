// How attention over the paged caches is cut into items (csrc/awq_serve_attention.hip for 4 bits,
// csrc/awq_kv16_attention.hip for 16): the arithmetic that the kernels, their grids and the workspace have in common.
// Plain C++ without the HIP headers (constexpr functions are the device's too), so that
// tests/test_attention_items.py and tests/test_attention16_cuts.py run it on the host: every item has to have a
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

// The first token that any of a request's rows may see under a sliding window (0: none), of `walked` tokens.
// Where the window lies past the table that is the missing token there.
constexpr int first_token(int window, int rows, int len, int walked) {
    const int64_t lo = (int64_t)len - rows - window + 1;
    return window == 0 || lo <= 0 || walked == 0 ? 0 : lo < walked ? (int)lo : walked - 1;
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
// The 16-bit cache's tiles: at least four steps an item, sixteen of prompts (nothing lies before the rows), whose blocks see half
// of their items on average.  4 / 16: 300 rows behind 1748 tokens 34 / 40 us, three chunks of up to 389 rows 42 / 46; prompts of
// 700 tokens 34 / 28, 1024 44 / 36.
constexpr int least_tile_steps(int steps, bool prompts) { return steps < (prompts ? 16 : 4) ? (prompts ? 16 : 4) : steps; }
// Steps of an item of that request with its items made alike: as many items, none longer.
constexpr int even_steps(int steps, int splits) { return splits > 1 ? (int)((uint32_t)(steps + splits - 1) / (uint32_t)splits) : steps; }
// Where an item ends that begins at `start`, of a block that sees `limit` tokens.
constexpr int item_end(int start, int chunk, int limit) {
    return limit - start < chunk ? limit : start + chunk;   // start + chunk may pass 32 bits where limit does not
}

struct AttentionPlan {
    bool decode, tile, combine;
    int limit, decode_target, tile_target, tile_cols;
    int64_t decode_items, tile_items;  // at most, of one kv head
    size_t part_floats(int kvh, int floats) const {      // the items' sums, so many floats of a column
        return (size_t)(decode_items * kCols + (tile_target ? tile_items * tile_cols : 0)) * kvh * floats;
    }
};
template <int TILE_COLS = kTileCols>
AttentionPlan attention_plan(int requests, int total, int max_query, int group, int kvh) {
    AttentionPlan p = {};
    p.tile_cols = TILE_COLS;
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
        const int64_t blocks = requests + rows * group / TILE_COLS;
        p.tile_target = blocks * kvh < kSplitBelow ? (kvh < kTileItems ? kTileItems / kvh : 1) : 0;
        p.tile_items = blocks + p.tile_target + 1;
    }
    p.combine = p.decode || p.tile_target;
    return p;
}

// The same for the 16-bit cache, whose tiles have 128 columns: workgroups of four waves, two on a CU, or of eight
// that share 128 columns' tokens.  Blocks that are fewer than half the places of four waves are split into one round of
// workgroups and their sums joined by another launch; those that fit into that round as they are get eight waves each (of heads
// of 128, with twice the LDS, one on a CU: a second round begins past 256), and none joins.
// One request, rows behind a context of 32768 tokens, split for four waves / for eight: 300 rows 174 / 195 us, 512 288 / 295,
// 768 394 / 528 (its 42 blocks have 128 places a head or 64).  Prompts of 1200 / 1777 / 2300 rows: split 38 / 52 / 73 us,
// whole with four waves 35 / 50 / 67, with eight 29 / 41 / 62.  256 / 320 / 400 / 500 blocks of 16 kv heads, four waves and eight:
// causal 55 45 / 69 54 / 86 68 / 108 95, nine documents 26 22 / 28 27 / 40 35 / 58 43; nine documents of 28 heads over 4
// 16 15 / 19 23 / 31 29 / 30 32; heads of 64, causal 54 55 / 63 47 / 78 59 / 96 80.
constexpr int kTile16Cols = 128, kRound16 = 512;
struct AttentionPlan16 : AttentionPlan {
    int tile_parts;                    // 2: eight waves share the tokens of 128 columns
};
inline AttentionPlan16 attention_plan16(int requests, int total, int max_query, int group, int kvh) {
    AttentionPlan16 p = {attention_plan<kTile16Cols>(requests, total, max_query, group, kvh), 1};
    if (!p.tile) return p;
    // Blocks of columns at most, and those to count with: each request may have one more than its columns fill.  Beside the
    // decode kernel only requests of more columns than that takes count, and all have a row as good as always: 64 single
    // tokens beside a chunk are not 64 blocks more, which would leave the chunk's few unsplit.  Split / whole: 300 rows behind
    // 32768 tokens beside 64 tokens behind 2000 each 256 / 587 us, 40 behind 4096 beside 128 behind 1000 each 65 / 140; a prompt
    // of 300 rows beside 64 tokens behind 2000 each 63 / 61.
    auto least = [](int64_t x, int64_t y) { return x < y ? x : y; };
    const int64_t rows = least((int64_t)requests * max_query, total), full = rows * group / kTile16Cols;
    const int64_t few = kDecodeColumns / group;          // rows that the decode kernel takes
    int64_t most = full + (p.decode ? least(requests, rows / (few + 1)) : requests);
    int64_t blocks = full + (p.decode ? least(requests, rows > requests ? (rows - requests) / few : 0) : requests);
    if (p.decode && (full + requests) * kvh < kSplitBelow && 2 * (int64_t)total >= (int64_t)requests * max_query) {
        // Requests are of max_query rows by half: as good as always none is the decode kernel's, and the tile kernel, which
        // has all of them then, splits one that is.  Three chunks of up to 389 rows 41.0 us with its launch, 38.0
        // without, sixteen of 64 rows behind 4032 tokens 60.3 and 57.0; a token behind 32768 beside a prompt of 700 rows
        // 50 and 31, beside 300 rows behind 3796 tokens 65 and 51.
        p.decode = false;
        p.limit = p.decode_target = 0;
        p.decode_items = 0;
        most = blocks = full + requests;
    }
    p.tile_target = 0;
    if (blocks * kvh < kSplitBelow) {
        // One round of workgroups.  The blocks of one request are known, and so are their items; of several each
        // block may come out with an item more than its share (item_steps takes half of them off).
        const int64_t all = kvh < kRound16 ? kRound16 / kvh : 1;
        const int64_t mine = ((int64_t)(max_query < total ? max_query : total) * group + kTile16Cols - 1) / kTile16Cols;
        const int64_t target = requests > 1 ? all - blocks / 2 : mine > 0 ? all / mine * mine : 1;
        p.tile_target = (int)(target > (all + 3) / 4 ? target : (all + 3) / 4);
    }
    p.tile_items = most + p.tile_target + 1;
    p.combine = p.decode || p.tile_target;
    if (!p.tile_target && p.tile_items * kvh <= kRound16) p.tile_parts = 2;
    return p;
}

}  // namespace awq
