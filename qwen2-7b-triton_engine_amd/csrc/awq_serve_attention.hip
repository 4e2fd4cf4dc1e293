// Attention over the 4-bit paged cache (include/awq_serving.h:
// awq_serve_kv4_attention): o = softmax(scale q K^T) V for the rows of many requests,
// each over its own pages, GQA heads.
//
// The cache's values are code * scale + zero per group of columns, and code * scale
// is exact in fp16 (4 + 7 significant bits).  So neither K nor V is rounded on
// the way to the matrix cores:
//   q.k = q.(code scale) + sum over groups of zero * (sum of q in the group)
//   o   = P (code scale)  + sum over groups of P zero
// The first terms are products of tiles; the second are one more k-step (the
// zeros against q's sums, held in three fp16 parts) and one more row block (the zeros
// as further columns of V, with a column of ones that gives the softmax's sum).
// q is scaled by its row's power of two and held in fp16, which is exact for fp16
// input; the probabilities are fp32 and enter as two fp16 parts, hi and lo.
#include "awq_serving.h"

namespace awq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kCols = 16;              // (row, query head) pairs of one workgroup: the columns of an MFMA
constexpr int kWaveKeys = 32;          // tokens of one inner pass of a wave
constexpr int kKeys = kWaveKeys * kWaves;
constexpr int kPExp = 14;              // the probabilities' scale before they are split: 2^14
constexpr int kQExp = 8;               // q's largest value lies in 2^7 .. 2^8: a group's sum stays below 2^15

// What a workgroup works on.
struct Item {
    int b, row0, rows, len, base;      // request, its first row, rows, tokens; its first item
    int chunk, splits, blocks, rel;    // tokens an item, items along them, blocks of columns; this item's number
};

struct Request {
    int row0, rows, len;
};
__device__ __forceinline__ Request request(const Kv4AttnArgs& a, int b) {
    Request r = {0, 0, 0};
    if (b < a.requests) {
        const int lo = a.query_start[b], hi = a.query_start[b + 1];
        r.row0 = lo < 0 ? 0 : lo < a.total ? lo : a.total;
        const int end = hi < r.row0 ? r.row0 : hi < a.total ? hi : a.total;
        r.rows = end - r.row0;
        r.len = a.seq_lens[b] < 0 ? 0 : a.seq_lens[b];
    }
    return r;
}
// Tokens to walk over: one past the table where the length is (that one is not
// there, and gives NaN).
__device__ __forceinline__ int walked(const Kv4AttnArgs& a, int len) {
    const int64_t room = (int64_t)a.width << a.s.page_log2;
    return len <= room ? len : (int)room + 1;
}
__device__ __forceinline__ int column_blocks(const Kv4AttnArgs& a, int rows) {
    const int most = rows < a.max_query ? rows : a.max_query;
    return (int)(((int64_t)most * (a.nh / a.s.kvh) + kCols - 1) / kCols);
}

constexpr int kTarget = 1024;          // items that a launch aims at, all kv heads together
__host__ __device__ inline int items_per_head(int kvh) { return kvh < kTarget ? kTarget / kvh : 1; }

// Finds an item (by number) or a row's items (by row): every workgroup walks over
// the requests' lengths by itself, so that no launch has to prepare a list.
// The tokens of an item are a multiple of kKeys, as few as the target allows.
template <bool BY_ROW>
__device__ bool find_item(const Kv4AttnArgs& a, int want, Item* found, int64_t* sums) {
    const int tid = threadIdx.x;
    if (tid == 0) found->b = -1;
    int64_t work = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kThreads) {
        const Request r = request(a, b0 + tid);
        int64_t all;
        block_scan<kWaves>((int64_t)walked(a, r.len) * column_blocks(a, r.rows), sums, all);
        work += all;
    }
    const int64_t per = (int64_t)kKeys * items_per_head(a.s.kvh);
    const int64_t chunk64 = kKeys * ((work + per - 1) / per);
    const int chunk = (int)(chunk64 < kKeys ? kKeys : chunk64 < (1 << 30) ? chunk64 : (1 << 30));
    int64_t before = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kThreads) {
        const Request r = request(a, b0 + tid);
        const int n = walked(a, r.len), blocks = column_blocks(a, r.rows), splits = (int)(((int64_t)n + chunk - 1) / chunk);
        int64_t all;
        const int64_t mine = (int64_t)blocks * splits, upto = before + block_scan<kWaves>(mine, sums, all);
        before += all;
        const bool hit = BY_ROW ? want >= r.row0 && want < r.row0 + r.rows : want >= upto - mine && want < upto;
        if (hit) *found = Item{b0 + tid, r.row0, r.rows, r.len, (int)(upto - mine), chunk, splits, blocks,
                               (int)(want - (upto - mine))};
    }
    __syncthreads();
    return found->b >= 0;
}
// The item in scalar registers: the same for every lane.
__device__ __forceinline__ Item uniform(const Item* lds) {
    Item it;
    const int* from = reinterpret_cast<const int*>(lds);
    int* to = reinterpret_cast<int*>(&it);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Item) / sizeof(int)); ++i) to[i] = __builtin_amdgcn_readfirstlane(from[i]);
    return it;
}

// Eight codes of a word times a scale, exact: nibble u and nibble u + 4 make
// pair u.  A nibble in bits 6 .. 9 of 0x4C00 is fp16 16 + code; (16 + code) s - 16 s
// is rounded once, to a value that needs no rounding.
__device__ __forceinline__ void scaled_codes(uint32_t w, half2_t s, half2_t minus16s, half2_t (&o)[4]) {
    constexpr uint32_t kMask = 0x03C003C0u, kBase = 0x4C004C00u;
    o[0] = __builtin_elementwise_fma(as_h2(and_or(w << 6, kMask, kBase)), s, minus16s);
    o[1] = __builtin_elementwise_fma(as_h2(and_or(w << 2, kMask, kBase)), s, minus16s);
    o[2] = __builtin_elementwise_fma(as_h2(and_or(w >> 2, kMask, kBase)), s, minus16s);
    o[3] = __builtin_elementwise_fma(as_h2(and_or(w >> 6, kMask, kBase)), s, minus16s);
}
__device__ __forceinline__ half2_t times_minus16(half2_t s) { return s * half2_t{(half_t)-16.0f, (half_t)-16.0f}; }

// What one lane holds of 16 tokens: lane (i, t) = (lane & 15, lane >> 4).
template <int HD, int GN>
struct Tile {
    uint32_t kw[HD / 32];              // token i, columns 32 s + 8 t .. of K
    half2_t ks[GN];                    // its (scale, zero)
    u32x4 vw;                          // tokens 4 t .. 4 t + 3, eight columns of V around HD / 16 * i
    half4_t vs, vz;                    // their scales in these columns' group; zeros of group min(i, GN - 1)
};

template <int HD, int GN>
__device__ __forceinline__ void load_tile(Tile<HD, GN>& x, const Kv4AttnArgs& a, const int32_t* table, int g, int key0,
                                          int n, int i, int t) {
    constexpr int kSteps = HD / 32;
    const int index = key0 >> a.s.page_log2;
    const bool inside = key0 < n;
    int page = inside && index < a.width ? table[index] : -1;
    const bool there = page >= 0 && page < a.s.num_pages;
    page = there ? page : 0;
    const int tok = key0 & (a.s.page() - 1);
    const uint8_t* block = a.cache + ((int64_t)page * a.s.kvh + g) * a.s.block();
    const uint8_t* kc = block + (tok + i) * (HD / 2) + t * (HD / 8);
    if constexpr (kSteps == 4) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(kc);
#pragma unroll
        for (int s = 0; s < 4; ++s) x.kw[s] = w[s];
    } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(kc);
        x.kw[0] = w.x;
        x.kw[1] = w.y;
    }
    const uint8_t* ks = block + 2 * a.s.k_bytes() + (tok + i) * (4 * GN);
    typedef half_t pairs_t __attribute__((ext_vector_type(2 * GN)));
    const pairs_t kz = *reinterpret_cast<const pairs_t*>(ks);
#pragma unroll
    for (int q = 0; q < GN; ++q) x.ks[q] = half2_t{kz[2 * q], kz[2 * q + 1]};
    const int tb = (tok >> 2) + t;
    const int j8 = HD == 128 ? i : i >> 1;
    x.vw = *reinterpret_cast<const u32x4*>(block + a.s.k_bytes() + (tb * (HD / 8) + j8) * 16);
    const uint8_t* vs = block + 2 * a.s.k_bytes() + a.s.scale_bytes() + tb * (16 * GN);
    x.vs = *reinterpret_cast<const half4_t*>(vs + 16 * (8 * j8 / (HD / GN)));
    x.vz = *reinterpret_cast<const half4_t*>(vs + 16 * (i < GN ? i : GN - 1) + 8);
    if (inside && !there) {            // a page outside the cache: NaN for the queries that see it
#pragma unroll
        for (int q = 0; q < GN; ++q) x.ks[q] = half2_t{(half_t)NAN, (half_t)NAN};
    }
    if (!there || key0 + 16 > n) {     // tokens past the length may hold anything
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (!there || key0 + 4 * t + r >= n) {
                x.vs[r] = (half_t)0.0f;
                x.vz[r] = (half_t)0.0f;
            }
        }
    }
}

// One workgroup: an item's tokens of one kv head for up to 16 columns, 32
// tokens per wave and pass.  S^T = K Q^T puts a column in each MFMA column, so one
// exponential covers four tokens of every column, and the result is already
// the B operand of O^T = V^T P^T (its k order, tokens 4 t + r of two tiles, is V's
// as loaded).  V's row order in that product is free: lane i takes the columns
// i VC .. i VC + VC - 1 of its tokens and supplies one of them to each of VC
// products.  The waves' results meet once, at the end.
template <int HD, int GN, bool BF16>
__global__ __launch_bounds__(kThreads) void awq_kv4_decode_kernel(Kv4AttnArgs a) {
    constexpr int kSteps = HD / 32;
    constexpr int VC = HD / 16;            // V columns per lane
    constexpr int G = HD / GN;
    constexpr int kStride = HD + 4;        // floats per column of the reduction buffer
    __shared__ int64_t sums[kWaves];
    __shared__ Item item_lds;
    __shared__ float m_lds[kWaves][kCols], l_lds[kWaves][kCols];
    __shared__ int lim_lds[kCols];
    __shared__ __align__(16) float o_lds[kWaves][kCols][kStride];

    if (!find_item<false>(a, blockIdx.x, &item_lds, sums)) return;
    const Item it = uniform(&item_lds);
    const int g = blockIdx.y, group = a.nh / a.s.kvh;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, t = lane >> 4;
    const int block = it.rel % it.blocks, split = it.rel / it.blocks;
    const int live_rows = it.rows < a.max_query ? it.rows : a.max_query;
    const int c0 = block * kCols, cols = live_rows * group - c0 < kCols ? live_rows * group - c0 : kCols;
    const int n = walked(a, it.len);

    // This lane's column: row c / group of the request, head c % group.
    const int c = c0 + (col < cols ? col : 0);
    const int row = c / group, head = g * group + c % group;
    const int64_t pos = (int64_t)it.len - it.rows + row;
    const int lim = pos < 0 ? 0 : pos + 1 < n ? (int)(pos + 1) : n;   // tokens it sees
    // Rows grow along the columns: the block's first sees the fewest tokens, its last the most.
    const int lim_min = __builtin_amdgcn_readlane(lim, 0);
    const int lim_max = __builtin_amdgcn_readlane(lim, cols - 1);
    const int start = split * it.chunk;
    const int end = lim_max < start + it.chunk ? lim_max : start + it.chunk;

    half8_t q[kSteps], qz = {};
    int exp;                               // of the row's power of two
    {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(it.row0 + row) * a.ld + (int64_t)head * HD;
        float x[kSteps][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            load8<BF16>(src + 32 * s + 8 * t, x[s]);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[s][e]));
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        exp = kQExp - __builtin_amdgcn_frexp_expf(mx);
        exp = exp < 100 ? exp : 100;
        const float up = __builtin_ldexpf(1.0f, exp);
        float sum[GN];
#pragma unroll
        for (int i = 0; i < GN; ++i) sum[i] = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[s][e] = (half_t)(x[s][e] * up);
                sum[32 * s / G] += (float)q[s][e];
            }
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < GN; ++i) {
            sum[i] += __shfl_xor(sum[i], 16);
            sum[i] += __shfl_xor(sum[i], 32);
            if (t == i) mine = sum[i];
        }
#pragma unroll
        for (int e = 0; e < 3; ++e) {      // 33 bits
            qz[e] = (half_t)mine;
            mine -= (float)qz[e];
        }
    }

    // exp(scale x) = exp2(x factor); the scores here are 2^exp times as large.
    // Every exponent is a difference of scores first: what they were rounded to
    // on the way must be the same wherever two meet.
    const float factor = a.scale * 1.4426950408889634f, unit = __builtin_ldexpf(factor, -exp);
    float m = -INFINITY;                   // of column `col`
    floatx4 acc[VC], acc_z = {0.f, 0.f, 0.f, 0.f};   // acc_z: rows 0 .. GN - 1 the groups' zeros, row 4 the sum
#pragma unroll
    for (int v = 0; v < VC; ++v) acc[v] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int32_t* table = a.tables + (int64_t)it.b * a.width;
    Tile<HD, GN> x[2];
    int key0 = start + kWaveKeys * wave;
    if (key0 < end) {
        load_tile(x[0], a, table, g, key0, n, col, t);
        load_tile(x[1], a, table, g, key0 + 16, n, col, t);
    }
    for (; key0 < end; key0 += kKeys) {
        Tile<HD, GN> y[2];
        if (key0 + kKeys < end) {          // the next pass's, in flight under this one
            load_tile(y[0], a, table, g, key0 + kKeys, n, col, t);
            load_tile(y[1], a, table, g, key0 + kKeys + 16, n, col, t);
        }
        floatx4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            half8_t z = {};
#pragma unroll
            for (int i = 0; i < GN; ++i)
                if (t == i) z[0] = z[1] = z[2] = x[h].ks[i].y;
            s[h] = mfma16x16x32(z, qz, floatx4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                const half_t sc = x[h].ks[32 * st / G].x;
                const half2_t s2 = {sc, sc};
                half2_t o[4];
                scaled_codes(x[h].kw[st], s2, times_minus16(s2), o);
                const half8_t k = {o[0].x, o[0].y, o[1].x, o[1].y, o[2].x, o[2].y, o[3].x, o[3].y};
                s[h] = mfma16x16x32(k, q[st], s[h]);
            }
        }
        if (key0 + kWaveKeys > lim_min) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (key0 + 16 * h + 4 * t + r >= lim) s[h][r] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[h][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx);
        const float ref = mn == -INFINITY ? 0.0f : mn;   // nothing yet: every exponential is 0
        if (__any(mn > m)) {
            const float alpha = __builtin_amdgcn_exp2f((m - ref) * unit);
            acc_z *= alpha;
#pragma unroll
            for (int v = 0; v < VC; ++v) acc[v] *= alpha;
        }
        m = mn;
        float p[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) p[4 * h + r] = __builtin_amdgcn_exp2f((s[h][r] - ref) * unit);
        half8_t phi, plo;
        split16(p, kPExp, phi, plo);

        // The zeros' rows and the row of ones.
        half8_t z = {};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const half_t fill = (half_t)(col == 4 ? 1.0f : 0.0f);
            z[r] = col < GN ? x[0].vz[r] : fill;
            z[4 + r] = col < GN ? x[1].vz[r] : fill;
        }
        acc_z = mfma16x16x32(z, plo, acc_z);
        acc_z = mfma16x16x32(z, phi, acc_z);
        half2_t pairs[4][VC];              // [tokens 2 k, 2 k + 1 of the two tiles][column]
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Tile<HD, GN>& y0 = x[k >> 1];
            const uint32_t w0 = y0.vw[2 * (k & 1)], w1 = y0.vw[2 * (k & 1) + 1];
            const half2_t s2 = {y0.vs[2 * (k & 1)], y0.vs[2 * (k & 1) + 1]}, m16 = times_minus16(s2);
            if constexpr (VC == 8) {
                half2_t o[4];
                scaled_codes(__builtin_amdgcn_perm(w1, w0, 0x05040100u), s2, m16, o);   // columns 0 .. 3
#pragma unroll
                for (int u = 0; u < 4; ++u) pairs[k][u] = o[u];
                scaled_codes(__builtin_amdgcn_perm(w1, w0, 0x07060302u), s2, m16, o);   // columns 4 .. 7
#pragma unroll
                for (int u = 0; u < 4; ++u) pairs[k][4 + u] = o[u];
            } else {                       // 4 columns a lane: the word's lower half or its upper one
                scaled_codes(__builtin_amdgcn_perm(w1, w0, col & 1 ? 0x07060302u : 0x05040100u), s2, m16, pairs[k]);
            }
        }
#pragma unroll
        for (int v = 0; v < VC; ++v) {
            const half8_t w = {pairs[0][v].x, pairs[0][v].y, pairs[1][v].x, pairs[1][v].y,
                               pairs[2][v].x, pairs[2][v].y, pairs[3][v].x, pairs[3][v].y};
            acc[v] = mfma16x16x32(w, plo, acc[v]);
            acc[v] = mfma16x16x32(w, phi, acc[v]);
        }
        x[0] = y[0];
        x[1] = y[1];
    }

    // This lane: rows 4 t + r of each product, i.e. columns VC (4 t + r) + v of column `col`.
    float zero[GN];
#pragma unroll
    for (int i = 0; i < GN; ++i) zero[i] = __shfl(acc_z[i], col);
    const float l = __shfl(acc_z[0], 16 + col);
    if (t == 0) {
        m_lds[wave][col] = __builtin_ldexpf(m, -exp);   // of the scores themselves
        l_lds[wave][col] = l;
        if (wave == 0) lim_lds[col] = lim;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int v = 0; v < VC; v += 4) {
            const int d = VC * (4 * t + r) + v;
            float z = zero[0];
#pragma unroll
            for (int i = 1; i < GN; ++i)
                if (d >= i * G) z = zero[i];
            *reinterpret_cast<floatx4*>(&o_lds[wave][col][d]) =
                floatx4{acc[v][r] + z, acc[v + 1][r] + z, acc[v + 2][r] + z, acc[v + 3][r] + z};
        }
    __syncthreads();
    for (int i = threadIdx.x; i < cols * HD; i += kThreads) {
        const int k = i / HD, d = i - k * HD;
        float mx = m_lds[0][k];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, m_lds[w][k]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, ls = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float al = __builtin_amdgcn_exp2f((m_lds[w][k] - ref) * factor);
            sum = fmaf(al, o_lds[w][k][d], sum);
            ls = fmaf(al, l_lds[w][k], ls);
        }
        if (it.splits == 1) {
            const int cc = c0 + k, r = cc / group, h = g * group + cc % group;
            const float y = lim_lds[k] == 0 ? 0.0f : sum / ls;
            reinterpret_cast<uint16_t*>(a.out)[((int64_t)(it.row0 + r) * a.nh + h) * HD + d] = to16<BF16>(y);
        } else {
            float* dst = a.part + (((int64_t)blockIdx.x * a.s.kvh + g) * kCols + k) * (HD + 2);
            dst[d] = sum;
            if (d == 0) {
                dst[HD] = mx;
                dst[HD + 1] = ls;
            }
        }
    }
}

// out[row, head] = sum of its items' parts, each weighted by exp2(its maximum -
// the overall maximum).  One workgroup per row and kv head.  Rows that see no
// token, and rows of no request, are set to zero here.
template <int HD, bool BF16>
__global__ __launch_bounds__(kThreads) void awq_kv4_combine_kernel(Kv4AttnArgs a) {
    __shared__ int64_t sums[kWaves];
    __shared__ Item item_lds;
    const int row = blockIdx.x, g = blockIdx.y, group = a.nh / a.s.kvh;
    const bool found = find_item<true>(a, row, &item_lds, sums);
    const Item it = uniform(&item_lds);
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + ((int64_t)row * a.nh + g * group) * HD;
    if (!found || it.splits == 0) {
        for (int i = threadIdx.x; i < group * HD; i += kThreads) out[i] = 0;
        return;
    }
    const int r = row - it.row0;
    if (it.splits == 1 || r >= a.max_query) return;
    const float factor = a.scale * 1.4426950408889634f;
    const bool blind = (int64_t)it.len - it.rows + r < 0;
    for (int i = threadIdx.x; i < group * HD; i += kThreads) {
        const int c = r * group + i / HD, d = i % HD;
        const int64_t step = (int64_t)it.blocks * a.s.kvh * kCols * (HD + 2);
        const float* base = a.part + (((int64_t)(it.base + c / kCols) * a.s.kvh + g) * kCols + c % kCols) * (HD + 2);
        float mx = -INFINITY;
        for (int s = 0; s < it.splits; ++s) mx = fmaxf(mx, base[s * step + HD]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, l = 0.0f;
        for (int s = 0; s < it.splits; ++s) {
            const float w = __builtin_amdgcn_exp2f((base[s * step + HD] - ref) * factor);
            sum = fmaf(w, base[s * step + d], sum);
            l = fmaf(w, base[s * step + HD + 1], l);
        }
        out[i] = to16<BF16>(blind ? 0.0f : sum / l);
    }
}

int64_t most_items(const Kv4AttnArgs& a) {
    const int64_t rows = (int64_t)a.requests * a.max_query < a.total ? (int64_t)a.requests * a.max_query : a.total;
    return items_per_head(a.s.kvh) + a.requests + rows * (a.nh / a.s.kvh) / kCols;
}

template <int HD, int GN, bool BF16>
hipError_t launch(const Kv4AttnArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((awq_kv4_decode_kernel<HD, GN, BF16>), dim3((unsigned)most_items(a), a.s.kvh), dim3(kThreads), 0,
                       stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((awq_kv4_combine_kernel<HD, BF16>), dim3(a.total, a.s.kvh), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

size_t kv4_attn_workspace(int requests, int total, int max_query, int nh, int kvh, int hd) {
    Kv4AttnArgs a = {};
    a.requests = requests;
    a.total = total;
    a.max_query = max_query;
    a.nh = nh;
    a.s.kvh = kvh;
    return (size_t)most_items(a) * kvh * kCols * (hd + 2) * sizeof(float);
}

hipError_t launch_kv4_attention(const Kv4AttnArgs& a, bool bf16, hipStream_t stream) {
    using std::integral_constant;
    auto typed = [&](auto hd, auto gn) {
        return bf16 ? launch<hd(), gn(), true>(a, stream) : launch<hd(), gn(), false>(a, stream);
    };
    constexpr integral_constant<int, 1> c1;
    constexpr integral_constant<int, 2> c2;
    constexpr integral_constant<int, 4> c4;
    constexpr integral_constant<int, 64> c64;
    constexpr integral_constant<int, 128> c128;
    if (a.s.hd == 64) return a.s.groups == 1 ? typed(c64, c1) : typed(c64, c2);
    return a.s.groups == 1 ? typed(c128, c1) : a.s.groups == 2 ? typed(c128, c2) : typed(c128, c4);
}

}  // namespace awq
