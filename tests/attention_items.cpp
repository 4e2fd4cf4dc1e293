// Walks over a call's items as the attention kernels number them, with their own
// arithmetic (csrc/awq_serve_items.h), one request after another on the host.
#include "awq_serve_items.h"

using namespace awq;

namespace {

struct Kernel {
    long long items, most_splits, most_steps, wrong;
};

template <int COLS, int KEYS>
Kernel walk(int requests, const int* starts, const int* lens, int total, int max_query, int group, int width,
            int page_log2, int limit, int target) {
    Kernel k = {};
    int64_t work = 0;
    int all_blocks = 0, item = 0;
    for (int pass = 0; pass < 2; ++pass) {
        if (pass) item = item_steps<KEYS>(target, work, all_blocks, requests);
        int row0 = 0;
        for (int b = 0; b < requests; ++b) {
            row0 = first_row(row0, starts[b], total);
            const int rows = end_row(row0, starts[b + 1], total) - row0;
            const int len = lens[b] < 0 ? 0 : lens[b], n = walked_tokens(width, page_log2, len);
            const int blocks = request_blocks<COLS>(request_columns(rows, max_query, group), limit);
            const int steps = request_steps<KEYS>(n);
            if (!pass) {
                work += (int64_t)blocks * steps;
                all_blocks += blocks;
                continue;
            }
            const int splits = request_splits(steps, item);
            k.items += (long long)blocks * splits;
            if (!blocks) continue;
            if (splits > k.most_splits) k.most_splits = splits;
            if ((steps < item ? steps : item) > k.most_steps) k.most_steps = steps < item ? steps : item;
            // The items of a block are its tokens, each once.
            int64_t at = 0;
            for (int i = 0; i < splits; ++i) {
                const int64_t start = (int64_t)i * item * KEYS;
                const int end = item_end((int)start, item * KEYS, n);
                if (start != at || end <= start || (int64_t)item * KEYS > INT32_MAX) ++k.wrong;
                at = end;
            }
            if (at != n) ++k.wrong;
        }
    }
    return k;
}

}  // namespace

// out: decode items, its grid, most splits, most steps of an item, wrong items; the same of
// the tile kernel; whether that has places for sums; rows covered by requests.
extern "C" void attention_items(int requests, const int* starts, const int* lens, int total, int max_query, int group,
                                int kvh, int width, int page_log2, long long* out) {
    const AttentionPlan p = attention_plan(requests, total, max_query, group, kvh);
    const Kernel d = walk<kCols, kKeys>(requests, starts, lens, total, max_query, group, width, page_log2, p.limit,
                                        p.decode_target);
    const Kernel t = walk<kTileCols, kTileKeys>(requests, starts, lens, total, max_query, group, width, page_log2,
                                                p.limit, p.tile_target);
    const long long values[] = {d.items, p.decode ? p.decode_items : 0, d.most_splits, d.most_steps, d.wrong,
                                t.items, p.tile ? p.tile_items : 0,     t.most_splits, t.most_steps, t.wrong,
                                p.tile_target != 0};
    for (long long v : values) *out++ = v;
}
