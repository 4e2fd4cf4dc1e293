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
// q is scaled by its row's power of two and held in fp16, to 2^-32 of the row's largest
// value (fp16 rows below 2^8 exactly); the probabilities are fp32 and enter as two fp16 parts, hi and lo.
// Outputs are as far from the 64-bit result as plain fp32 torch's (2.1e-4 of their
// norm in fp16, 1.7e-3 in bf16: the output's own rounding).
//
// Three launches at most: requests of few columns (decode), requests of many (tiles), and the
// joining of what was split along the tokens.  28 heads of 128 over 4 kv heads, groups
// of 64, pages of 64, graph replays, us: one request of 1100 tokens 10.4, 64 of up to
// 4096 (2190 on average) 36, 16 of up to 16000 31; prompts of 256, 1024, 1777 and 4096
// tokens 21, 40, 78 and 277 (434 TFLOP/s of useful work).  Past 64 requests every wave's search for
// its item takes over: 256 of up to 2048 tokens 73, 1024 of up to 512 139, 4096 of up to 256 1130.
#include "awq_serve_walk.h"

namespace awq {
namespace {

static_assert(kKeys == kWaveKeys * kWaves && kTileCols == 16 * kWaves, "awq_serve_items.h");

constexpr int kPExp = 14;              // the probabilities' scale before they are split: 2^14
constexpr int kQExp = 8;               // q's largest value lies in 2^7 .. 2^8: a group's sum stays below 2^15

// ---- pieces of both kernels ---------------------------------------------------------

// Maximum over the four lanes that share a column (lane, lane + 16, + 32, + 48).
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
// The running maximum is raised only where a score passes it by more than this
// (in powers of two): probabilities of up to 2^1.5, scaled by 2^14, still fit fp16,
// and most passes do without the cross-lane maximum and the rescaling.
constexpr float kSlack = 1.5f;

// 0x4C004C00 in a VGPR, opaque to the optimiser (awq_device.h magic_vgpr): the
// and-or below stays one instruction.
constexpr uint32_t kBase16 = 0x4C004C00u;
__device__ __forceinline__ uint32_t base16_vgpr() {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)kBase16, (int)kBase16, 0x111, 0xF, 0xF, false);
}
// Eight codes of a word times a scale, exact: nibble u and nibble u + 4 make
// pair u.  A nibble in bits 6 .. 9 of 0x4C00 is fp16 16 + code; (16 + code) s - 16 s
// is rounded once, to a value that needs no rounding.
__device__ __forceinline__ void scaled_codes(uint32_t w, uint32_t base, half2_t s, half2_t minus16s, half2_t (&o)[4]) {
    constexpr uint32_t kMask = 0x03C003C0u;
    o[0] = __builtin_elementwise_fma(as_h2(and_or(w << 6, kMask, base)), s, minus16s);
    o[1] = __builtin_elementwise_fma(as_h2(and_or(w << 2, kMask, base)), s, minus16s);
    o[2] = __builtin_elementwise_fma(as_h2(and_or(w >> 2, kMask, base)), s, minus16s);
    o[3] = __builtin_elementwise_fma(as_h2(and_or(w >> 6, kMask, base)), s, minus16s);
}
__device__ __forceinline__ half2_t times_minus16(half2_t s) { return s * half2_t{(half_t)-16.0f, (half_t)-16.0f}; }

template <int GN>
struct PairsOf {
    typedef half_t type __attribute__((ext_vector_type(2 * GN)));
};

// A column's query as the B operand of the k-steps: lane (column, t) holds
// columns 32 s + 8 t + e of the head, times the power of two that brings the row's
// largest value to 2^7 .. 2^8 (2^15 times at most, which is exact for whatever is
// smaller).  The groups' sums come from the matrix cores too, as products with rows
// of ones, and enter in three fp16 parts (33 bits), lane t those of group t.
// Returns the exponent of the row's power of two.
template <int HD, int GN, bool BF16>
__device__ __forceinline__ int load_query(const uint16_t* src, int col, int t, half8_t (&q)[HD / 32], half8_t& qz) {
    constexpr int kSteps = HD / 32, G = HD / GN;
    int exp;
    if constexpr (BF16) {
        float x[kSteps][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            load8<true>(src + 32 * s + 8 * t, x[s]);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[s][e]));
        }
        exp = kQExp - __builtin_amdgcn_frexp_expf(column_max(mx));
        exp = exp < 100 ? exp : 100;
        const float up = __builtin_ldexpf(1.0f, exp);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[s][e] = (half_t)(x[s][e] * up);
    } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const half8_t*>(src + 32 * s + 8 * t);
        half2_t mx = {};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                mx = __builtin_elementwise_max(mx, as_h2(as_u32(half2_t{q[s][e], q[s][e + 1]}) & 0x7FFF7FFFu));
        exp = kQExp - __builtin_amdgcn_frexp_expf(column_max(fmaxf((float)mx.x, (float)mx.y)));
        exp = exp < 15 ? exp : 15;
        const half_t up = (half_t)__builtin_ldexpf(1.0f, exp);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] *= up;
    }
    floatx4 sums = {0.f, 0.f, 0.f, 0.f};   // row g: group g
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const half_t one = (half_t)(col == 32 * s / G ? 1.0f : 0.0f);
        sums = mfma16x16x32(half8_t{one, one, one, one, one, one, one, one}, q[s], sums);
    }
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < GN; ++i) {
        const float sum = __shfl(sums[i], col);
        if (t == i) mine = sum;
    }
    qz = half8_t{};
#pragma unroll
    for (int e = 0; e < 3; ++e) {
        qz[e] = (half_t)mine;
        mine -= (float)qz[e];
    }
    return exp;
}

// What one of a row's scaled scores counts in powers of two.  Kept finite: bf16 queries near 2^127
// under a large scale pass fp32 here, and a difference of zero times infinity would be NaN.
__device__ __forceinline__ float score_unit(float factor, int exp) {
    return fminf(__builtin_ldexpf(factor, -exp), __FLT_MAX__);
}

// Tells the scheduler how to mix READS reads of LDS and MFMAS products: FIRST reads, then
// one after every EACH products.
template <int READS, int MFMAS, int EACH, int FIRST>
__device__ __forceinline__ void ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
    constexpr int kRest = READS - FIRST;
#pragma unroll
    for (int i = 0; i < kRest; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MFMAS > EACH * kRest ? MFMAS - EACH * kRest : 1, 0);
}

// ---- few columns: decode ---------------------------------------------------------------

// One workgroup: an item's tokens of one kv head for up to 16 columns, 32
// tokens per wave and pass.  S^T = K Q^T puts a column in each MFMA column, so one
// exponential covers four tokens of every column, and the result is already
// the B operand of O^T = V^T P^T (its k order, tokens 4 t + r of two tiles, is V's
// as loaded).  V's row order in that product is free: lane i takes the columns
// i VC .. i VC + VC - 1 of its tokens and supplies one of them to each of VC
// products.  K's registers are loaded again as soon as its product is made, V's
// likewise: each is in flight under the other half of the pass, without a second
// set of registers.  The waves' results meet once, at the end.
//
// What bounds it: at one request latency -- 7.2 us of launch, item, page, codes and
// the waves' meeting, one after another; at 64 requests of up to 4096 tokens (85 MB
// of codes and scales, 30 us) the start and end of a workgroup, 9 us, and the vector
// unit in between: 300 instructions a wave for 32 tokens, a third of them the
// multiplying out of 8192 codes, against 28 products.  Three waves a SIMD (146 to 163
// registers; four spilled 44 to 68 bytes).  A second set of K and V registers, and a page number
// loaded in the pass before, were slower when they were tried.
template <int HD, int GN, bool BF16>
__global__ __launch_bounds__(kThreads, 3) void awq_kv4_decode_kernel(Kv4AttnArgs a) {
    constexpr int kSteps = HD / 32;
    constexpr int VC = HD / 16;            // V columns per lane
    constexpr int G = HD / GN;
    constexpr int kStride = HD + 4;        // floats per column of the reduction buffer
    __shared__ float m_lds[kWaves][kCols], l_lds[kWaves][kCols];
    __shared__ int lim_lds[kCols];
    __shared__ __align__(16) float o_lds[kWaves][kCols][kStride];

    Item it;
    if (!find_item<kCols, kKeys>(a, blockIdx.x, a.decode_target, it)) {
        if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) fill_rows(a);   // the grid's last column has no item
        return;
    }
    write_records(a, it, false);
    const int g = blockIdx.y, group = a.nh / a.s.kvh;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, t = lane >> 4;
    const int block = it.rel % it.blocks, split = it.rel / it.blocks;
    const int all_cols = columns(a, it.r.rows), c0 = block * kCols;
    const int cols = all_cols - c0 < kCols ? all_cols - c0 : kCols;
    const int n = walked(a, it.r.len);
    // The block's last column sees the most tokens.
    const int64_t last_pos = (int64_t)it.r.len - it.r.rows + (c0 + cols - 1) / group;
    const int lim_max = last_pos < 0 ? 0 : last_pos + 1 < n ? (int)(last_pos + 1) : n;
    const int start = split * it.chunk;
    const int end = item_end(start, it.chunk, lim_max);

    // What this lane reads of 16 tokens, from where they begin in the codes and in the scales.
    const int j8 = HD == 128 ? col : col >> 1;
    const uint32_t k_ofs = col * (HD / 2) + t * (HD / 8), v_ofs = a.s.k_bytes() + (t * (HD / 8) + j8) * 16;
    const uint32_t ks_ofs = col * (4 * GN), vs_ofs = a.s.scale_bytes() + t * (16 * GN) + 16 * (8 * j8 / G);
    const uint32_t vz_ofs = a.s.scale_bytes() + t * (16 * GN) + 16 * (col < GN ? col : GN - 1) + 8;
    struct Place {                         // of 16 tokens
        const uint8_t *codes, *scales;
        bool there;
    };
    auto place = [&](int page, int key) {
        Place p;
        p.there = page >= 0 && page < a.s.num_pages;
        const int tok = key & (a.s.page() - 1);
        const uint8_t* block_at = a.cache + ((int64_t)(p.there ? page : 0) * a.s.kvh + g) * a.s.block();
        p.codes = block_at + tok * (HD / 2);
        p.scales = block_at + 2 * a.s.k_bytes() + tok * (4 * GN);
        return p;
    };
    uint32_t kw[2][kSteps];                // token col, columns 32 s + 8 t .. of K
    half2_t ks[2][GN];                     // its (scale, zero)
    u32x4 vw[2];                           // tokens 4 t .. 4 t + 3, eight columns of V around VC col
    half4_t vs[2], vz[2];                  // their scales in these columns' group; the zeros of group min(col, GN - 1)
    auto load_k = [&](const Place (&p)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (kSteps == 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(p[h].codes + k_ofs);
#pragma unroll
                for (int s = 0; s < 4; ++s) kw[h][s] = w[s];
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2*>(p[h].codes + k_ofs);
                kw[h][0] = w.x;
                kw[h][1] = w.y;
            }
            const auto kz = *reinterpret_cast<const typename PairsOf<GN>::type*>(p[h].scales + ks_ofs);
#pragma unroll
            for (int i = 0; i < GN; ++i) ks[h][i] = half2_t{kz[2 * i], kz[2 * i + 1]};
        }
    };
    auto load_v = [&](const Place (&p)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            vw[h] = *reinterpret_cast<const u32x4*>(p[h].codes + v_ofs);
            vs[h] = *reinterpret_cast<const half4_t*>(p[h].scales + vs_ofs);
            vz[h] = *reinterpret_cast<const half4_t*>(p[h].scales + vz_ofs);
        }
    };

    int key0 = start + kWaveKeys * wave;
    Pages64 pages = {a.tables + (int64_t)it.b * a.width, 0, 0};
    pages.fetch(a, key0, n);
    Place now[2];
    now[0] = place(pages.page(a, key0, n), key0);
    now[1] = place(pages.page(a, key0 + 16, n), key0 + 16);
    if (key0 < end) {
        load_k(now);
        load_v(now);
    }

    // This lane's column: row c / group of the request, head c % group.
    const int c = c0 + (col < cols ? col : 0);
    const int row = c / group, head = g * group + c % group;
    const int64_t pos = (int64_t)it.r.len - it.r.rows + row;
    const int lim = pos < 0 ? 0 : pos + 1 < n ? (int)(pos + 1) : n;   // tokens it sees
    const int lim_min = __builtin_amdgcn_readlane(lim, 0);            // rows grow along the columns
    half8_t q[kSteps], qz;
    const int exp = load_query<HD, GN, BF16>(
        reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(it.r.row0 + row) * a.ld + (int64_t)head * HD, col, t, q, qz);
    // exp(scale x) = exp2(x factor); the scores here are 2^exp times as large.
    // Every exponent is a difference of scores first: what they were rounded to
    // on the way must be the same wherever two meet.
    const float factor = a.scale * 1.4426950408889634f, unit = score_unit(factor, exp);
    const uint32_t base = base16_vgpr();
    // Rows GN .. 15 of the zeros' block: a row of ones at 4, the rest zero.
    const uint32_t z_mask = col < GN ? 0xFFFFFFFFu : 0u, z_fill = col == 4 ? 0x3C003C00u : 0u;

    float m = -INFINITY;                   // of column `col`
    floatx4 acc[VC], acc_z = {0.f, 0.f, 0.f, 0.f};   // acc_z: rows 0 .. GN - 1 the groups' zeros, row 4 the sum
#pragma unroll
    for (int v = 0; v < VC; ++v) acc[v] = floatx4{0.f, 0.f, 0.f, 0.f};
    while (key0 < end) {
        const bool more = key0 + kKeys < end;
        Place next[2];
        const int key1 = more ? key0 + kKeys : key0;
        next[0] = place(pages.page(a, key1, n), key1);
        next[1] = place(pages.page(a, key1 + 16, n), key1 + 16);

        if (!now[0].there || !now[1].there) {   // a page outside the cache: NaN for the queries that see it
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (!now[h].there)
#pragma unroll
                    for (int i = 0; i < GN; ++i) ks[h][i] = half2_t{(half_t)NAN, (half_t)NAN};
        }
        floatx4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            half8_t z = {};
#pragma unroll
            for (int i = 0; i < GN; ++i)
                if (t == i) z[0] = z[1] = z[2] = ks[h][i].y;
            s[h] = mfma16x16x32(z, qz, floatx4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                const half_t sc = ks[h][32 * st / G].x;
                const half2_t s2 = {sc, sc};
                half2_t o[4];
                scaled_codes(kw[h][st], base, s2, times_minus16(s2), o);
                const half8_t k = {o[0].x, o[0].y, o[1].x, o[1].y, o[2].x, o[2].y, o[3].x, o[3].y};
                s[h] = mfma16x16x32(k, q[st], s[h]);
            }
        }
        if (more) load_k(next);
        if (key0 + kWaveKeys > lim_min) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (key0 + 16 * h + 4 * t + r >= lim) s[h][r] = -INFINITY;
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int r = 1; r < 4; ++r) mx = fmaxf(mx, fmaxf(s[0][r], s[1][r]));
        if (__any((mx - m) * unit > kSlack)) {
            const float mn = fmaxf(m, column_max(mx));
            const float alpha = __builtin_amdgcn_exp2f(mn == -INFINITY ? 0.0f : (m - mn) * unit);
            acc_z *= alpha;
#pragma unroll
            for (int v = 0; v < VC; ++v) acc[v] *= alpha;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.0f : m;     // nothing yet: every exponential is 0
        float p[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) p[4 * h + r] = __builtin_amdgcn_exp2f((s[h][r] - ref) * unit);
        half8_t phi, plo;
        split16(p, kPExp, phi, plo);

        if (!now[0].there || !now[1].there || key0 + kWaveKeys > n) {   // tokens past the length may hold anything
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!now[h].there || key0 + 16 * h + 4 * t + r >= n) vs[h][r] = vz[h][r] = (half_t)0.0f;
        }
        union {
            uint32_t w[4];
            half8_t h;
        } z;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x2 w = __builtin_bit_cast(u32x2, vz[h]);
            z.w[2 * h] = (w.x & z_mask) | z_fill;
            z.w[2 * h + 1] = (w.y & z_mask) | z_fill;
        }
        acc_z = mfma16x16x32(z.h, plo, acc_z);
        acc_z = mfma16x16x32(z.h, phi, acc_z);
        // Four columns at a time: the words' lower halves, then their upper ones
        // (heads of 64: a lane has four columns, one half or the other).
#pragma unroll
        for (int part = 0; part < VC / 4; ++part) {
            const uint32_t half = VC == 8 ? (part ? 0x07060302u : 0x05040100u) : (col & 1 ? 0x07060302u : 0x05040100u);
            half2_t pairs[4][4];           // [tokens 2 k, 2 k + 1 of the two tiles][column]
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const half4_t sv = vs[k >> 1];
                const half2_t s2 = {sv[2 * (k & 1)], sv[2 * (k & 1) + 1]};
                scaled_codes(__builtin_amdgcn_perm(vw[k >> 1][2 * (k & 1) + 1], vw[k >> 1][2 * (k & 1)], half), base, s2,
                             times_minus16(s2), pairs[k]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const half8_t w = {pairs[0][u].x, pairs[0][u].y, pairs[1][u].x, pairs[1][u].y,
                                   pairs[2][u].x, pairs[2][u].y, pairs[3][u].x, pairs[3][u].y};
                floatx4& d = acc[4 * part + u];
                d = mfma16x16x32(w, plo, d);
                d = mfma16x16x32(w, phi, d);
            }
        }
        if (more) load_v(next);
        now[0] = next[0];
        now[1] = next[1];
        key0 += kKeys;
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
            reinterpret_cast<uint16_t*>(a.out)[((int64_t)(it.r.row0 + r) * a.nh + h) * HD + d] = to16<BF16>(y);
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

// ---- many columns: tiles ---------------------------------------------------------------

// Place of a token within its 64-token tile of the transposed V: the S^T product
// leaves lane group t with tokens 4 t .. 4 t + 3 of each 16-token block, and the P V
// product wants 8 consecutive k per lane: 8 consecutive places hold tokens
// 4 t .. 4 t + 3 of two neighbouring blocks.  Four neighbouring tokens (block of
// four tb) stay together, at place 32 (tb / 8) + 8 (tb % 4) + 4 (tb / 4 % 2).

// Swizzle of a row's 16-byte chunks in LDS, K: 16 rows' same chunk is what one
// operand read fetches, and the rows start on the same bank.
template <int CHUNKS>
__device__ __forceinline__ int k_chunk(int row, int chunk) {
    return chunk ^ (row & (CHUNKS < 16 ? CHUNKS - 1 : 15));
}
// V: reads as K's; writes go to the same chunk of rows that are 8 apart.
__device__ __forceinline__ int v_chunk(int row, int chunk) { return chunk ^ ((row ^ (row >> 3)) & 7); }

// One workgroup: 16 columns of one kv head per wave, over an item's tokens in tiles of
// 64.  The tile's codes are multiplied out once per workgroup, exactly, into LDS --
// K as it is, V transposed, its zeros and a row of ones as rows of their own -- and
// every wave reads its operands there.  The codes of the next tile are on their way
// in registers meanwhile.  One LDS buffer and two barriers a tile: the room goes to
// a third workgroup on the CU, which has work while the others wait (two buffers and two
// workgroups: 105 us at a prompt of 1777 tokens, then 97).
//
// What bounds it: at 4096 tokens the issue of vector instructions beside the
// products, some 380 a wave and tile -- sixteen scores a lane with their exponentials
// and two parts, 130 to multiply the codes out -- against 56 products; LDS is
// busy 40 % of the time.  At 1777 the 780 workgroups, of 1 to 28 tiles, are nearly all resident at
// once (768 places): the CUs whose three have the most tiles end last.  128 columns a workgroup, in two column blocks a wave or in eight
// waves, multiply out half as much and were slower (107 and 116 us against 97 and 105): fewer, coarser
// workgroups, and no registers to read operands ahead.
// ONE_PAGE: pages of 64 tokens and more, where a tile lies in one of them and its
// address is the workgroup's, not a lane's.
template <int HD, int GN, bool ONE_PAGE, bool BF16>
__global__ __launch_bounds__(kThreads, GN == 4 ? 2 : 3) void awq_kv4_tile_kernel(Kv4AttnArgs a) {
    constexpr int kSteps = HD / 32, kDb = HD / 16, kChunks = HD / 8, G = HD / GN;
    constexpr int kRows = HD + 16;                       // of the transposed V: columns, zeros, ones
    constexpr int kK = kTileKeys * HD, kV = kRows * kTileKeys, kZ = kTileKeys * 4;   // halfs
    __shared__ __align__(16) half_t buf[kK + kV + kZ];

    Item it;
    const int tid = threadIdx.x, lane = tid & 63;
    if (!find_item<kTileCols, kTileKeys>(a, blockIdx.x, a.tile_target, it)) {
        if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && a.limit == 0) fill_rows(a);
        return;
    }
    write_records(a, it, true);
    const int g = blockIdx.y, group = a.nh / a.s.kvh;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, t = lane >> 4;
    // The last blocks, which see the most tokens, start first.
    const int block = it.blocks - 1 - it.rel % it.blocks, split = it.rel / it.blocks;
    const int all_cols = columns(a, it.r.rows), c0 = block * kTileCols;
    const int n = walked(a, it.r.len);
    auto limit_of = [&](int c) {                         // tokens that a column sees
        const int64_t pos = (int64_t)it.r.len - it.r.rows + c / group;
        return pos < 0 ? 0 : pos + 1 < n ? (int)(pos + 1) : n;
    };
    const int c_last = c0 + kTileCols < all_cols ? c0 + kTileCols - 1 : all_cols - 1;
    const int start = split * it.chunk, lim_wg = limit_of(c_last);
    const int end = item_end(start, it.chunk, lim_wg);
    const int tiles = end > start ? (end - start + kTileKeys - 1) / kTileKeys : 0;
    Pages64 window = {a.tables + (int64_t)it.b * a.width, 0, 0};
    window.fetch(a, start, n);

    // Rows of the zeros' block that no tile writes: ones at 4, else zero; zeros of no group.
    for (int i = tid; i < 16 * kTileKeys + kZ; i += kThreads) {
        const int r = i / kTileKeys;
        if (i < 16 * kTileKeys) {
            if (r >= GN) buf[kK + HD * kTileKeys + i] = (half_t)(r == 4 ? 1.0f : 0.0f);
        } else if (i % 4 >= GN) {
            buf[kK + kV + i - 16 * kTileKeys] = (half_t)0.0f;
        }
    }

    // What this thread brings of a tile: of K the words of token k_tok and lane group
    // k_t; of V eight columns of four tokens (heads of 64: half of the threads).
    const int k_tok = tid >> 2, k_t = tid & 3;
    const int v_tb = tid / kChunks, v_j = tid % kChunks, v_g = 8 * v_j / G;
    const bool has_v = v_tb < kTileKeys / 4;
    typedef uint32_t words_t __attribute__((ext_vector_type(kSteps)));
    words_t kw;
    typename PairsOf<GN>::type ks;
    u32x4 vw;
    half4_t vs, vz;
    struct Pages {
        int k, v;                                        // of this thread's token of K, of its four of V
    };
    auto pages = [&](int key) {
        if constexpr (ONE_PAGE) {
            const int p = window.page(a, key, n);
            return Pages{p, p};
        } else {
            if (((key + kTileKeys - 1) >> a.s.page_log2) - window.first >= 64) window.fetch(a, key, n);
            return Pages{__shfl(window.entry, ((key + k_tok) >> a.s.page_log2) - window.first),
                         has_v ? __shfl(window.entry, ((key + 4 * v_tb) >> a.s.page_log2) - window.first) : -1};
        }
    };
    auto there = [&](int page) { return page >= 0 && page < a.s.num_pages; };
    auto block_of = [&](int page) { return a.cache + ((int64_t)(there(page) ? page : 0) * a.s.kvh + g) * a.s.block(); };
    const uint32_t k_ofs = k_t * (HD / 8), v_ofs = a.s.k_bytes() + v_j * 16;
    const uint32_t ks_ofs = 2 * a.s.k_bytes(), vs_ofs = 2 * a.s.k_bytes() + a.s.scale_bytes() + v_g * 16;
    auto load = [&](int key, Pages p) {
        // The token of the page that the tile or the thread begins with, and the thread's after it.
        const int in = ONE_PAGE ? key & (a.s.page() - 1) : 0;
        const uint8_t* kb = block_of(p.k);
        const uint8_t* vb = ONE_PAGE ? kb : block_of(p.v);
        const uint32_t k_in = ONE_PAGE ? k_tok : (key + k_tok) & (a.s.page() - 1);
        const uint32_t v_in = ONE_PAGE ? v_tb : ((key + 4 * v_tb) & (a.s.page() - 1)) >> 2;
        const uint8_t* kp = kb + in * (HD / 2);
        kw = *reinterpret_cast<const words_t*>(kp + k_in * (HD / 2) + k_ofs);
        ks = *reinterpret_cast<const typename PairsOf<GN>::type*>(kb + in * (4 * GN) + k_in * (4 * GN) + ks_ofs);
        if (has_v) {
            vw = *reinterpret_cast<const u32x4*>(vb + in * (HD / 2) + v_in * (kChunks * 16) + v_ofs);
            const uint8_t* sp = vb + in * (4 * GN) + v_in * (16 * GN) + vs_ofs;
            vs = *reinterpret_cast<const half4_t*>(sp);
            vz = *reinterpret_cast<const half4_t*>(sp + 8);
        }
    };
    const uint32_t base = base16_vgpr();
    const int v_place = 4 * (v_tb >> 3) + (v_tb & 3), v_sub = 4 * (v_tb >> 2 & 1);
    auto store = [&](int key, Pages p) {
        half_t *lk = buf, *lv = lk + kK, *lz = lv + kV;
        if (!there(p.k)) {                               // outside the cache: NaN for the queries that see it
#pragma unroll
            for (int i = 0; i < 2 * GN; ++i) ks[i] = (half_t)NAN;
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const half_t sc = ks[2 * (32 * j / G)];
            const half2_t s2 = {sc, sc};
            half2_t o[4];
            scaled_codes(kw[j], base, s2, times_minus16(s2), o);
            *reinterpret_cast<half8_t*>(lk + k_tok * HD + 8 * k_chunk<kChunks>(k_tok, 4 * j + k_t)) =
                half8_t{o[0].x, o[0].y, o[1].x, o[1].y, o[2].x, o[2].y, o[3].x, o[3].y};
        }
        half_t zk = ks[1];
#pragma unroll
        for (int i = 1; i < GN; ++i)
            if (k_t == i) zk = ks[2 * i + 1];
        if (k_t < GN) lz[k_tok * 4 + k_t] = zk;
        if (has_v) {
            if (!there(p.v) || key + kTileKeys > n) {    // tokens past the length may hold anything
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!there(p.v) || key + 4 * v_tb + r >= n) vs[r] = vz[r] = (half_t)0.0f;
            }
            const half2_t s01 = {vs[0], vs[1]}, s23 = {vs[2], vs[3]};
            const half2_t m01 = times_minus16(s01), m23 = times_minus16(s23);
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const uint32_t half = part ? 0x07060302u : 0x05040100u;
                half2_t p01[4], p23[4];
                scaled_codes(__builtin_amdgcn_perm(vw[1], vw[0], half), base, s01, m01, p01);
                scaled_codes(__builtin_amdgcn_perm(vw[3], vw[2], half), base, s23, m23, p23);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int d = 8 * v_j + 4 * part + u;
                    *reinterpret_cast<half4_t*>(lv + d * kTileKeys + 8 * v_chunk(d, v_place) + v_sub) =
                        half4_t{p01[u].x, p01[u].y, p23[u].x, p23[u].y};
                }
            }
            if (8 * v_j % G == 0) {
                const int d = HD + v_g;
                *reinterpret_cast<half4_t*>(lv + d * kTileKeys + 8 * v_chunk(d, v_place) + v_sub) = vz;
            }
        }
    };

    Pages now = {-1, -1};                                // of the tile in registers
    if (tiles > 0) {
        now = pages(start);
        load(start, now);
    }

    half8_t q[kSteps], qz;
    const int local = 16 * wave + col, c = c0 + local, cc = c < all_cols ? c : all_cols - 1;
    const int lim = limit_of(cc);
    const int exp = load_query<HD, GN, BF16>(reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(it.r.row0 + cc / group) * a.ld +
                                                 (int64_t)(g * group + cc % group) * HD, col, t, q, qz);
    const float factor = a.scale * 1.4426950408889634f, unit = score_unit(factor, exp);
    const int lim_min = __builtin_amdgcn_readlane(lim, 0), lim_max = __builtin_amdgcn_readlane(lim, 15);

    float m = -INFINITY;
    floatx4 acc[kDb + 1];                                // [kDb]: rows 0 .. GN - 1 the groups' zeros, row 4 the sum
#pragma unroll
    for (int d = 0; d <= kDb; ++d) acc[d] = floatx4{0.f, 0.f, 0.f, 0.f};
    // Operand addresses: the swizzles only flip bits that the rows' starts leave free.
    const uint32_t k_at = col * HD + 8 * k_chunk<kChunks>(col, t);
    const uint32_t v_at = kK + col * kTileKeys + 8 * v_chunk(col, t);   // row 16 d + col flips by 2 d
    for (int tile = 0; tile < tiles; ++tile) {
        const int key0 = start + tile * kTileKeys;
        if (tile) lds_barrier();                         // every wave has read the tile before
        store(key0, now);
        if (tile + 1 < tiles) {                          // the next tile's codes, in flight under this one
            now = pages(key0 + kTileKeys);
            load(key0 + kTileKeys, now);
        }
        lds_barrier();
        if (key0 >= lim_max) continue;                   // past every column of this wave
        // 32 tokens at a time: half the scores are alive.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            floatx4 s[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int kb = 2 * h + b;
                const half_t zk = buf[kK + kV + (16 * kb + col) * 4 + t];
                const half8_t z = {zk, zk, zk, 0, 0, 0, 0, 0};
                s[b] = mfma16x16x32(z, qz, floatx4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int st = 0; st < kSteps; ++st)
                    s[b] = mfma16x16x32(*reinterpret_cast<const half8_t*>(buf + (k_at ^ (32 * st)) + 16 * kb * HD), q[st], s[b]);
            }
            // Operands are read several products ahead (the scheduler by itself keeps
            // two in flight, and waits for LDS at every product): first the scores'
            // alone, then the first half's sums with the second half's scores.
            if (h == 0) ahead<2 * kSteps + 2, 2 * (kSteps + 1), 1, 5>();
            else ahead<kDb + 1 + 2 * kSteps + 2, 2 * (kDb + 1) + 2 * (kSteps + 1), 2, 4>();
            if (key0 + 32 * h + 32 > lim_min) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key0 + 32 * h + 16 * b + 4 * t + r >= lim) s[b][r] = -INFINITY;
            }
            float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
            for (int r = 1; r < 4; ++r) mx = fmaxf(mx, fmaxf(s[0][r], s[1][r]));
            if (__any((mx - m) * unit > kSlack)) {
                const float mn = fmaxf(m, column_max(mx));
                const float alpha = __builtin_amdgcn_exp2f(mn == -INFINITY ? 0.0f : (m - mn) * unit);
#pragma unroll
                for (int d = 0; d <= kDb; ++d) acc[d] *= alpha;
                m = mn;
            }
            const float ref = m == -INFINITY ? 0.0f : m;     // nothing yet: every exponential is 0
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f((s[j >> 2][j & 3] - ref) * unit);
            half8_t phi, plo;
            split16(p, kPExp, phi, plo);
#pragma unroll
            for (int d = 0; d <= kDb; ++d) {
                const half8_t v = *reinterpret_cast<const half8_t*>(buf + (v_at ^ (32 * h) ^ (16 * (d & 3))) + 16 * d * kTileKeys);
                acc[d] = mfma16x16x32(v, plo, acc[d]);
                acc[d] = mfma16x16x32(v, phi, acc[d]);
            }
            if (h == 1) ahead<kDb + 1, 2 * (kDb + 1), 2, 4>();
        }
    }

    float zero[GN];
#pragma unroll
    for (int j = 0; j < GN; ++j) zero[j] = __shfl(acc[kDb][j], col);
    const float l = __shfl(acc[kDb][0], 16 + col);
    if (c >= all_cols) return;
    if (it.splits == 1) {
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) +
                        ((int64_t)(it.r.row0 + c / group) * a.nh + g * group + c % group) * HD + 4 * t;
#pragma unroll
        for (int d = 0; d < kDb; ++d) {
            uint32_t w[2];
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const float z = zero[16 * d / G];
                const float y0 = lim == 0 ? 0.0f : (acc[d][r] + z) / l, y1 = lim == 0 ? 0.0f : (acc[d][r + 1] + z) / l;
                w[r / 2] = (uint32_t)to16<BF16>(y0) | ((uint32_t)to16<BF16>(y1) << 16);
            }
            *reinterpret_cast<u32x2*>(dst + 16 * d) = u32x2{w[0], w[1]};
        }
    } else {
        float* dst = a.tile_part + (((int64_t)blockIdx.x * a.s.kvh + g) * kTileCols + local) * (HD + 2);
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
            for (int r = 0; r < 4; r += 2)
                *reinterpret_cast<float2*>(dst + 16 * d + 4 * t + r) =
                    float2{acc[d][r] + zero[16 * d / G], acc[d][r + 1] + zero[16 * d / G]};
        if (t == 0) {
            dst[HD] = __builtin_ldexpf(m, -exp);
            dst[HD + 1] = l;
        }
    }
}

// ---- joining the items of a row -----------------------------------------------------

template <int HD, int WAVES, bool BF16>
__global__ __launch_bounds__(kThreads) void awq_kv4_combine_kernel(Kv4AttnArgs a) {
    combine_items<HD, WAVES, BF16>(a);
}

// ---- launches ----------------------------------------------------------------------------

template <int HD, int GN, bool BF16>
hipError_t launch(Kv4AttnArgs a, hipStream_t stream) {
    const AttentionPlan p = attention_plan(a.requests, a.total, a.max_query, a.nh / a.s.kvh, a.s.kvh);
    a.limit = p.limit;
    a.decode_target = p.decode_target;
    a.tile_target = p.tile_target;
    a.records = reinterpret_cast<i32x4*>(a.part);
    a.part += (size_t)a.total * (sizeof(i32x4) / sizeof(float));
    a.tile_part = a.part + p.decode_items * a.s.kvh * kCols * (HD + 2);
    if (p.decode) {
        hipLaunchKernelGGL((awq_kv4_decode_kernel<HD, GN, BF16>), dim3((unsigned)p.decode_items, a.s.kvh), dim3(kThreads),
                           0, stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.tile) {
        auto kernel = a.s.page() >= kTileKeys ? awq_kv4_tile_kernel<HD, GN, true, BF16> : awq_kv4_tile_kernel<HD, GN, false, BF16>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)p.tile_items, a.s.kvh), dim3(kThreads), 0, stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.combine) {
        const int64_t all = (int64_t)a.total * a.nh, groups = all <= kFewUnits ? all : (all + 3) / 4;
        auto kernel = all <= kFewUnits ? awq_kv4_combine_kernel<HD, 4, BF16> : awq_kv4_combine_kernel<HD, 1, BF16>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(groups < kCombineGroups ? groups : kCombineGroups)), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace

size_t kv4_attn_workspace(int requests, int total, int max_query, int nh, int kvh, int hd) {
    return part_bytes(attention_plan(requests, total, max_query, nh / kvh, kvh), total, kvh, hd + Kv4AttnArgs::kExtra);
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
