// Walks over a call's items as the attention kernels of the 16-bit cache number them: blocks of 128 columns in
// the tile kernel, and under a sliding window a request's items begin where its first row's window does.
#include "awq_serve_items.h"

using namespace awq;

namespace {

struct Kernel {
    long long items, most_splits, wrong;
};

template <int COLS, int KEYS>
Kernel walk(int requests, const int* starts, const int* lens, int total, int max_query, int group, int width,
            int page_log2, int window, int limit, int target) {
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
            const int first = first_token(window, rows, len, n) / KEYS;
            const int blocks = request_blocks<COLS>(request_columns(rows, max_query, group), limit);
            const int steps = request_steps<KEYS>(n) - first;
            if (steps < 0 || (n > 0 && steps == 0)) ++k.wrong;
            if (!pass) {
                work += (int64_t)blocks * steps;
                all_blocks += blocks;
                continue;
            }
            const int splits = request_splits(steps, item);
            k.items += (long long)blocks * splits;
            if (!blocks) continue;
            if (splits > k.most_splits) k.most_splits = splits;
            // The items of a block are the tokens from the window on, each once, and no token before it is a row's.
            int64_t at = (int64_t)first * KEYS;
            if (window && at > 0 && at > (int64_t)len - rows - window + 1) ++k.wrong;
            for (int i = 0; i < splits; ++i) {
                const int64_t start = (int64_t)first * KEYS + (int64_t)i * item * KEYS;
                const int end = item_end((int)start, item * KEYS, n);
                if (start != at || end <= start || start > INT32_MAX) ++k.wrong;
                at = end;
            }
            if (n > 0 && at != n) ++k.wrong;
        }
    }
    return k;
}

}  // namespace

// out: decode items, its grid, most splits, wrong; the same of the tile kernel; whether that has places for sums.
extern "C" void attention16_items(int requests, const int* starts, const int* lens, int total, int max_query, int group,
                                  int kvh, int width, int page_log2, int window, long long* out) {
    const AttentionPlan16 p = attention_plan16(requests, total, max_query, group, kvh);
    const Kernel d = walk<kCols, kKeys>(requests, starts, lens, total, max_query, group, width, page_log2, window, p.limit,
                                        p.decode_target);
    const Kernel t = walk<kTile16Cols, kTileKeys>(requests, starts, lens, total, max_query, group, width, page_log2, window,
                                                  p.limit, p.tile_target);
    const long long values[] = {d.items, p.decode ? p.decode_items : 0, d.most_splits, d.wrong,
                                t.items, p.tile ? p.tile_items : 0,     t.most_splits, t.wrong, p.tile_target != 0};
    for (long long v : values) *out++ = v;
}
