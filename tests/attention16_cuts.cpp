// Walks over a call's items exactly as the kernels of the 16-bit cache cut them (find_item in csrc/awq_serve_walk.h): a tile
// item has a least length, and a request's tile items are made alike.
#include "awq_serve_items.h"

using namespace awq;

namespace {

struct Kernel {
    long long items, most_splits, longest, wrong;   // longest: steps of an item
};

template <int COLS, int KEYS>
Kernel walk(int requests, const int* starts, const int* lens, int total, int max_query, int group, int width,
            int page_log2, int window, int limit, int target) {
    constexpr bool kTile = COLS != kCols;
    Kernel k = {};
    int64_t work = 0;
    int all_blocks = 0, item = 0;
    bool prompts = true;                                 // of the first 64 requests
    for (int pass = 0; pass < 2; ++pass) {
        if (pass) {
            item = item_steps<KEYS>(target, work, all_blocks, requests);
            if (target && kTile) item = least_tile_steps(item, prompts);
        }
        int row0 = 0;
        for (int b = 0; b < requests; ++b) {
            row0 = first_row(row0, starts[b], total);
            const int rows = end_row(row0, starts[b + 1], total) - row0;
            const int len = lens[b] < 0 ? 0 : lens[b], n = walked_tokens(width, page_log2, len);
            const int first = first_token(window, rows, len, n) / KEYS;
            const int blocks = request_blocks<COLS>(request_columns(rows, max_query, group), limit);
            const int steps = request_steps<KEYS>(n) - first;
            if (b < 64 && rows < len) prompts = false;
            if (!pass) {
                work += (int64_t)blocks * steps;
                all_blocks += blocks;
                continue;
            }
            const int splits = request_splits(steps, item);
            k.items += (long long)blocks * splits;
            if (!blocks || !splits) continue;
            if (splits > k.most_splits) k.most_splits = splits;
            const int chunk = kTile ? even_steps(steps, splits) : item;
            if (chunk > item) ++k.wrong;
            int64_t at = (int64_t)first * KEYS;
            for (int i = 0; i < splits; ++i) {
                const int64_t start = (int64_t)first * KEYS + (int64_t)i * chunk * KEYS;
                if (start > INT32_MAX || (int64_t)chunk * KEYS > INT32_MAX || start != at) {
                    ++k.wrong;
                    break;
                }
                const int end = item_end((int)start, chunk * KEYS, n);
                if (end <= start) ++k.wrong;             // an item without tokens
                const long long length = (end - start + KEYS - 1) / KEYS;
                if (length > k.longest) k.longest = length;
                at = end;
            }
            if (at != n) ++k.wrong;
        }
    }
    return k;
}

}  // namespace

// out: of the decode kernel items, its grid, most splits, longest item, wrong; the same of the tile kernel; whether that has
// places for sums, its groups of waves, whether the joining launch follows, the columns up to which a request is the decode
// kernel's, bytes of all parts' places for sums (floats of a column: 1).
extern "C" void attention16_cuts(int requests, const int* starts, const int* lens, int total, int max_query, int group,
                                 int kvh, int width, int page_log2, int window, long long* out) {
    const AttentionPlan16 p = attention_plan16(requests, total, max_query, group, kvh);
    const Kernel d = walk<kCols, kKeys>(requests, starts, lens, total, max_query, group, width, page_log2, window, p.limit,
                                        p.decode_target);
    const Kernel t = walk<kTile16Cols, kTileKeys>(requests, starts, lens, total, max_query, group, width, page_log2, window,
                                                  p.limit, p.tile_target);
    const long long values[] = {d.items, p.decode ? p.decode_items : 0, d.most_splits, d.longest, d.wrong,
                                t.items, p.tile ? p.tile_items : 0,     t.most_splits, t.longest, t.wrong,
                                p.tile_target != 0, p.tile_parts, p.combine, p.limit, (long long)p.part_floats(1, 1)};
    for (long long v : values) *out++ = v;
}
