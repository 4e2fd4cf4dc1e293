// What attention over a paged cache does around its products, for the 4-bit and the
// 16-bit cache: which item a workgroup has (awq_serve_items.h), pages, rows that no item
// has, and the joining of what was split along the tokens.
//
// Args, the kernels' argument block, has next to its fields
//   kTileCols                       columns of a tile workgroup
//   group()                         heads of a kv head
//   first_key(rows, len)            the first token that a row of a request may see
//   sees_none(b, row0, rows, len, i)   whether the i-th row of request b sees no token
//   least_steps(steps, prompts)     steps of a tile item, from those that the target gives; prompts: nothing lies before the rows
//   kEven                           whether a request's tile items are made alike
//   combine                         whether the joining launch follows, and needs records
//   kExtra                          floats of a column in `part` past its sums: its maximum, the sum of its exponentials, ..
//   factor(column)                  what one of that maximum's counts in powers of two
#pragma once

#include "awq_serve_items.h"
#include "awq_serving.h"

namespace awq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// ---- which item a workgroup has --------------------------------------------------

// Requests of few columns (rows times the heads that share a kv head) go to the
// decode kernel in blocks of 16 columns, the others to the tile kernel in blocks
// of more.  An item is a block and a stretch of tokens.
struct Request {
    int row0, rows, len;               // first row, rows, tokens
};
// 64 requests, one a lane, from b0 on.  before: the largest start of those below b0, and
// afterwards of those below b0 + 64.  Starts go up, as good as always: only where they do not is the
// running maximum formed, and up says whether they did (a walk of all requests that found it true need not
// look again).  With the maximum in every walk 1024 requests took 162 us instead of 142.
template <class Args>
__device__ __forceinline__ Request requests64(const Args& a, int b0, int& before, bool look, bool& up) {
    const int b = b0 + (int)(threadIdx.x & 63);
    int lo = a.total, hi = a.total, len = 0;
    if (b < a.requests) {
        lo = a.query_start[b];
        hi = a.query_start[b + 1];
        len = a.seq_lens[b];
    }
    Request r;
    r.row0 = row_in(lo, a.total);
    if (look && __any(hi < lo || r.row0 < before)) {
        r.row0 = wave_scan_max(first_row(before, lo, a.total));
        up = false;
    }
    r.rows = end_row(r.row0, hi, a.total) - r.row0;
    r.len = len < 0 ? 0 : len;
    before = __builtin_amdgcn_readlane(r.row0, 63);
    return r;
}
template <class Args>
__device__ __forceinline__ int walked(const Args& a, int len) { return walked_tokens(a.width, a.s.page_log2, len); }
template <class Args>
__device__ __forceinline__ int columns(const Args& a, int rows) {
    return request_columns(rows, a.max_query, a.group());
}
// Blocks of COLS columns that a request has in this kernel, and its tokens in steps of KEYS.
template <int COLS, int KEYS, class Args>
__device__ __forceinline__ void sizes(const Args& a, const Request& r, int& blocks, int& steps) {
    blocks = request_blocks<COLS>(columns(a, r.rows), a.limit);
    steps = request_steps<KEYS>(walked(a, r.len)) - a.first_key(r.rows, r.len) / KEYS;
}

struct Item {
    Request r;
    int b;                             // the request's number
    int first;                         // the token that the request's first item begins with
    int chunk, splits, blocks;         // tokens of an item, items along the tokens, blocks of columns
    int base, rel;                     // number of the request's first item; this item's after it
};

// Finds an item by its number.  Every wave walks over the requests' lengths by
// itself, 64 at a time and without a barrier: no launch has to prepare a list,
// and the host need not know the lengths.  The tokens of an item are a multiple of
// KEYS (item_steps).
template <int COLS, int KEYS, class Args>
__device__ __forceinline__ bool find_item(const Args& a, int want, int target, Item& it) {
    int start = 0;
    bool up = true;
    Request r = requests64(a, 0, start, true, up);
    int blocks, steps, m = item_steps<KEYS>(0, 0, 0, a.requests);
    sizes<COLS, KEYS>(a, r, blocks, steps);
    if (target) {
        int64_t work = (int64_t)blocks * steps;
        int all_blocks = blocks;
        for (int b0 = 64; b0 < a.requests; b0 += 64) {
            sizes<COLS, KEYS>(a, requests64(a, b0, start, true, up), blocks, steps);
            work += (int64_t)blocks * steps;
            all_blocks += blocks;
        }
        // Sums below 2^24 a lane, as good as always, are added in 32 bits.
        int64_t all;
        if (a.requests == 1) {
            all = (int64_t)__builtin_amdgcn_readfirstlane((int)(work >> 32)) << 32 |
                  (uint32_t)__builtin_amdgcn_readfirstlane((int)work);
        } else if (__all(work < (1 << 24))) {
            all = __builtin_amdgcn_readlane(wave_scan32((int)work), 63);
        } else {
            all = __shfl(wave_scan(work), 63);
        }
        const int blocks_sum = a.requests == 1 ? 0 : __builtin_amdgcn_readlane(wave_scan32(all_blocks), 63);
        m = item_steps<KEYS>(target, all, blocks_sum, a.requests);
        if (COLS != kCols) m = a.least_steps(m, __all(r.rows >= r.len));
        m = __builtin_amdgcn_readfirstlane(m);
    }
    int before = 0;
    start = 0;
    const bool look = !up || !target;                    // (without a target this is the first walk)
    for (int b0 = 0; b0 < a.requests; b0 += 64) {
        if (a.requests > 64) r = requests64(a, b0, start, look, up);
        sizes<COLS, KEYS>(a, r, blocks, steps);
        const int splits = request_splits(steps, m), mine = blocks * splits;
        const int upto = before + wave_scan32(mine);
        const uint64_t hit = __ballot(want >= upto - mine && want < upto);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
            it.r = Request{pick(r.row0), pick(r.rows), pick(r.len)};
            it.b = b0 + at;
            it.first = a.first_key(it.r.rows, it.r.len) / KEYS * KEYS;
            it.splits = pick(splits);
            it.chunk = (COLS != kCols && Args::kEven ? even_steps(pick(steps), it.splits) : m) * KEYS;
            it.blocks = pick(blocks);
            it.base = pick(upto - mine);
            it.rel = want - it.base;
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// What the combining launch has to know of a row.
struct RowRecord {
    int row, base;                     // the row's place in its request; its first item, ~ of it for the tile kernel's
    int blocks, splits;                // 0 items: zeros are to be written; 1: the row is done
};
// Written by the first item of a request.
template <class Args>
__device__ __forceinline__ void write_records(const Args& a, const Item& it, bool tile) {
    if (!a.combine || it.rel != 0 || blockIdx.y != 0) return;
    for (int i = threadIdx.x; i < it.r.rows; i += (int)blockDim.x) {
        const bool blind = a.sees_none(it.b, it.r.row0, it.r.rows, it.r.len, i);
        a.records[it.r.row0 + i] = i32x4{i, tile ? ~it.base : it.base, it.blocks,
                                         i >= a.max_query || it.splits == 1 ? 1 : blind ? 0 : it.splits};
    }
}
// Rows that no item has: those of no request, or of one without tokens, are zeros, those past
// a max_query that was too small NaN (not what the memory held).
// Done by the first workgroup past the items; a grid has at least one.
template <class Args>
__device__ __forceinline__ void fill_rows(const Args& a) {
    const int pieces = a.nh * a.s.hd / 8;                // of 16 bytes
    auto fill = [&](int lo, int hi, uint32_t w) {        // a word of two elements everywhere
        u32x4* out = reinterpret_cast<u32x4*>(a.out);
        for (int64_t i = (int64_t)lo * pieces + threadIdx.x; i < (int64_t)hi * pieces; i += blockDim.x) out[i] = u32x4{w, w, w, w};
        if (!a.combine) return;
        for (int i = lo + (int)threadIdx.x; i < hi; i += (int)blockDim.x) a.records[i] = i32x4{0, 0, 0, 1};
    };
    int start = 0, first = 0, end = 0;                   // of all requests' rows
    bool up = true;
    for (int b0 = 0; b0 < a.requests; b0 += 64) {
        const Request r = requests64(a, b0, start, true, up);
        if (b0 == 0) first = __builtin_amdgcn_readlane(r.row0, 0);
        if (b0 + 64 >= a.requests) end = __builtin_amdgcn_readlane(r.row0 + r.rows, (a.requests - 1) & 63);
        const int done = r.len == 0 ? 0 : a.max_query;   // rows that are an item's
        for (uint64_t some = __ballot(r.rows > done); some; some &= some - 1) {
            const int at = __builtin_ctzll(some), row0 = __builtin_amdgcn_readlane(r.row0, at);
            const int skip = __builtin_amdgcn_readlane(done, at);
            fill(row0 + skip, row0 + __builtin_amdgcn_readlane(r.rows, at), skip ? 0x7FFF7FFFu : 0u);
        }
    }
    fill(0, first, 0);
    fill(end, a.total, 0);
}

// ---- pieces of the kernels ----------------------------------------------------------

// A request's pages from the one that holds `key` on: lane i has the i-th of 64, -1 past
// the length or the table.  One load for 64 pages: a page's number then costs a lane
// read and no wait for memory (a load of it would be waited for behind the codes'
// loads that were issued before it).
struct Pages64 {
    const int32_t* table;
    int first, entry;
    template <class Args>
    __device__ __forceinline__ void fetch(const Args& a, int key, int n) {
        first = key >> a.s.page_log2;
        const int index = first + (int)(threadIdx.x & 63);
        entry = index < a.width && ((int64_t)index << a.s.page_log2) < n ? table[index] : -1;
    }
    // Of a key that is the same for the whole wave.
    template <class Args>
    __device__ __forceinline__ int page(const Args& a, int key, int n) {
        const int index = key >> a.s.page_log2;
        if ((uint32_t)(index - first) >= 64u) fetch(a, key, n);
        return __builtin_amdgcn_readlane(entry, index - first);
    }
};

// ---- joining the items of a row -----------------------------------------------------

// out[row, head] = sum of its items' parts, each weighted by exp2(its maximum -
// the overall maximum).  WAVES waves have a row and head: each every WAVES-th item,
// a lane an item's weight and two columns' sums, eight loads in flight; the
// waves meet in LDS.  All four where rows and heads are few (and items many), else
// one: 2 requests of up to 32768 tokens, 64 rows and heads, 27.8 us with one and 24.7
// with four; 64 of up to 4096, 1792 rows and heads, 35.8 and 38.1.
template <int HD, int WAVES, bool BF16, class Args>
__device__ __forceinline__ void combine_items(const Args& a) {
    constexpr int W = HD / 64;                           // columns a lane
    __shared__ float m_lds[kWaves], l_lds[kWaves], o_lds[kWaves][HD];
    const int group = a.group();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = WAVES == 1 ? 0 : wave;
    const int64_t all = (int64_t)a.total * a.nh;
    constexpr int kUnits = kWaves / WAVES;               // of a workgroup
    const int64_t stride = (int64_t)gridDim.x * kUnits;
    for (int64_t u0 = (int64_t)blockIdx.x * kUnits + (WAVES == 1 ? wave : 0); u0 < all; u0 += 64 * stride) {
        // The records of 64 units in one load: a batch of long prompts has nothing to join (16-bit cache, 52.7 us for
        // 56.5 with a load each).
        const int64_t own = u0 + lane * stride;
        i32x4 records = {0, 0, 0, 1};
        if (own < all) records = a.records[(uint32_t)own / (uint32_t)a.nh];
        for (uint64_t some = __ballot(records[3] != 1); some; some &= some - 1) {
            const int at = __builtin_ctzll(some);
            i32x4 rec;
#pragma unroll
            for (int i = 0; i < 4; ++i) rec[i] = __builtin_amdgcn_readlane(records[i], at);
            const int64_t unit = u0 + at * stride;
            const int head = (int)((uint32_t)unit % (uint32_t)a.nh), g = head / group;
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + unit * HD;
            if (rec[3] == 0) {
                if (first == 0)
#pragma unroll
                    for (int i = 0; i < W; ++i) out[W * lane + i] = 0;
                continue;
            }
            const bool tile = rec[1] < 0;
            const int c = rec[0] * group + head % group, cols = tile ? Args::kTileCols : kCols, block = c / cols, splits = rec[3];
            const int item = tile ? ~rec[1] + rec[2] - 1 - block : rec[1] + block;
            const int64_t step = (int64_t)rec[2] * a.s.kvh * cols * (HD + Args::kExtra);
            const float* base = (tile ? a.tile_part : a.part) + (((int64_t)item * a.s.kvh + g) * cols + c % cols) * (HD + Args::kExtra);
            const float factor = a.factor(base + HD);

            float mx = -INFINITY, l = 0.0f, sum[W] = {};
            for (int s0 = 0; s0 < splits; s0 += 64 * WAVES) {
                const int mine = s0 + first + WAVES * lane;
                const bool have = mine < splits;
                const float* p = base + (have ? mine : 0) * step;
                const int left = splits - s0 - first;
                const int count = left <= 0 ? 0 : left < 64 * WAVES ? (left + WAVES - 1) / WAVES : 64;
                float v[8][W];
                auto fetch = [&](int j0) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int at = j0 + j < count ? s0 + first + WAVES * (j0 + j) : 0;
#pragma unroll
                        for (int i = 0; i < W; ++i) v[j][i] = base[at * step + W * lane + i];
                    }
                };
                const float pm = p[HD], pl = p[HD + 1];
                fetch(0);
                const float own = have ? pm : -INFINITY;
                const float top = fmaxf(mx, wave_max(own)), ref = top == -INFINITY ? 0.0f : top;
                const float w = __builtin_amdgcn_exp2f((own - ref) * factor), old = __builtin_amdgcn_exp2f((mx - ref) * factor);
                l = l * old + wave_sum(have ? pl * w : 0.0f);
#pragma unroll
                for (int i = 0; i < W; ++i) sum[i] *= old;
                mx = top;
                for (int j0 = 0; j0 < count; j0 += 8) {
                    if (j0) fetch(j0);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float wj = __builtin_bit_cast(
                            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), (j0 + j) & 63));
#pragma unroll
                        for (int i = 0; i < W; ++i) sum[i] = j0 + j < count ? fmaf(wj, v[j][i], sum[i]) : sum[i];
                    }
                }
            }
            if constexpr (WAVES == 1) {
                uint32_t y = 0;
#pragma unroll
                for (int i = 0; i < W; ++i) y |= (uint32_t)to16<BF16>(sum[i] / l) << (16 * i);
                if constexpr (W == 2) reinterpret_cast<uint32_t*>(out)[lane] = y;
                else out[lane] = (uint16_t)y;
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i) o_lds[wave][W * lane + i] = sum[i];
                if (lane == 0) {
                    m_lds[wave] = mx;
                    l_lds[wave] = l;
                }
                __syncthreads();
                if (threadIdx.x < HD) {
                    float top = m_lds[0];
#pragma unroll
                    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_lds[w]);
                    const float ref = top == -INFINITY ? 0.0f : top;
                    float y = 0.0f, ls = 0.0f;
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) {
                        const float al = __builtin_amdgcn_exp2f((m_lds[w] - ref) * factor);
                        y = fmaf(al, o_lds[w][threadIdx.x], y);
                        ls = fmaf(al, l_lds[w], ls);
                    }
                    out[threadIdx.x] = to16<BF16>(y / ls);
                }
                __syncthreads();                             // the buffers are read
            }
        }
    }
}

// Workgroups of the combining launch at most, one round of them: 5 chunks of up to 700 rows, 32 heads, nothing to join
// (16-bit cache) 50.1 us with 2048 and 52.7 with 8192; 3 of up to 389, all to join, 42.0 and 42.5.
constexpr int kCombineGroups = 2048;
constexpr int kFewUnits = 512;         // rows times heads that get four waves each there

inline size_t part_bytes(const AttentionPlan& p, int total, int kvh, int floats) {   // row records, then the items' sums
    return (size_t)total * sizeof(i32x4) + p.part_floats(kvh, floats) * sizeof(float);
}

}  // namespace
}  // namespace awq
