// Attention over the 16-bit paged cache (include/awq_serving.h:
// awq_serve_kv16_attention): o = softmax(score(q K^T)) V for the rows of many
// requests, each over its own pages, GQA heads; the score is scale x, capped by
// c tanh(x / c), less slope |i - j|, and a row sees tokens lo .. hi - 1 of a window,
// a document or a prefix.
//
// Both kernels form S^T = K Q^T: an MFMA column is a (row, head) pair, so that the
// running maximum and sum of a column live in the lanes that hold its scores, and
// the probabilities are already the B operand of O^T = V^T P^T (the k order of that
// product, tokens, is V's as it is read).  Rows and the heads that share a kv head are
// one axis of columns: K and V of a token are read once for all of them.
#include "awq_serve_walk.h"

namespace awq {
namespace {

constexpr int k16Cols = Kv16AttnArgs::kTileCols;
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// ---- 16-bit operands of either type, eight in four words ---------------------------

template <bool BF16>
__device__ __forceinline__ floatx16 mfma32(u32x4 a, u32x4 b, floatx16 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
// Two values rounded to nearest.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    if constexpr (BF16)
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, bf16x2));
    else
        return as_u32(__builtin_convertvector(f2{x, y}, half2_t));
}
template <bool BF16>
__device__ __forceinline__ float low16(uint32_t w) {
    if constexpr (BF16) return __builtin_bit_cast(float, w << 16);
    else return (float)as_h2(w).x;
}
template <bool BF16>
__device__ __forceinline__ float high16(uint32_t w) {
    if constexpr (BF16) return __builtin_bit_cast(float, w & 0xFFFF0000u);
    else return (float)as_h2(w).y;
}
template <bool BF16>
constexpr uint32_t kOnes = BF16 ? 0x3F803F80u : 0x3C003C00u;
template <bool BF16>
constexpr uint32_t kExponents = BF16 ? 0x7F807F80u : 0x7C007C00u;

// Largest exponent field of each half: all ones where a value is not finite.
template <bool BF16>
__device__ __forceinline__ uint32_t exponents(uint32_t most, uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most),
                                                                  __builtin_bit_cast(u16x2, w & kExponents<BF16>)));
}
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint32_t most) {
    constexpr uint32_t kLow = kExponents<BF16> & 0xFFFFu;
    return (most & 0xFFFFu) == kLow || (most >> 16) == kLow;
}
// The same words with 0 in the place of values that are not finite.
template <bool BF16>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    constexpr uint32_t kLow = kExponents<BF16> & 0xFFFFu, kHigh = kExponents<BF16> & 0xFFFF0000u;
    return ((w & kLow) == kLow ? 0u : w & 0xFFFFu) | ((w & kHigh) == kHigh ? 0u : w & 0xFFFF0000u);
}

// The probabilities' scale in powers of two, and how far above it a score may lie before the running maximum is
// raised: of 32 columns one or another passes its maximum in many tiles, and each time the sums are rescaled.
// fp16 holds values up to 2^16 and 11 bits down to 2^-14: 2^8 leaves both room for 2^7.5 above and
// all bits down to 2^-22 of the maximum; bf16 has the range of fp32, and 2^-32, 2^-16 with what lies above, keeps the sums of
// values near its largest inside fp32 for 2^16 tokens of one weight, and 2^94 of range below.
template <bool BF16>
constexpr float kPScale = BF16 ? -32.0f : 8.0f;
template <bool BF16>
constexpr float kSlack16 = BF16 ? 16.0f : 7.5f;

// bf16 queries are brought to at most 2^8 by a power of two, so that a sum of products
// stays inside fp32 for keys of ordinary size; fp16's are inside it as they are.  Returns the power's exponent.
// mx: largest value of the row.  scale: of scores that meet the distance's part as they are, 0 of others (plain ones count by
// their differences, capped ones end at the cap).  Such scores are formed, and under scales that would bring what multiplies
// the products past 2^126 the query stays larger instead, up to 2^108.
__device__ __forceinline__ int query_exp(float mx, float scale) {
    int exp = 8 - __builtin_amdgcn_frexp_expf(mx);
    const int over = scale > 0.0f ? __builtin_amdgcn_frexp_expf(scale) - exp - 126 : 0;
    exp += over < 0 ? 0 : over < 100 ? over : 100;
    return exp < 100 ? exp : 100;
}
__device__ __forceinline__ u32x4 scaled_bf16(u32x4 w, float up) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2<true>(low16<true>(w[i]) * up, high16<true>(w[i]) * up);
    return w;
}
// What multiplies a product of the scaled query: kept finite (an infinity times a product of 0 is NaN) and above zero
// (a masked score times it is -infinity; 2^-149 of any product is nothing beside 1).
__device__ __forceinline__ float unit_of(float factor, int exp) {
    return fminf(fmaxf(__builtin_ldexpf(factor, -exp), 0x1p-149f), __FLT_MAX__);
}

// c tanh(x / c) as c - 2 c / (1 + e^(2 x / c)): in absolute terms it errs by a few 2^-24 c, nothing beside the
// probabilities' rounding while c is below 2^9; above, where small scores matter beside a large cap, the series
// to 1e-8 of the value below c / 4.
constexpr float kPlainCap = 512.0f;
__device__ __forceinline__ float capped(float x, float c, float inv) {
    const float u = x * inv, u2 = u * u;
    const float e = __builtin_amdgcn_exp2f(u * 2.8853900817779268f);
    const float far = fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    if (c <= kPlainCap) return c * far;
    const float near = u * fmaf(u2, fmaf(u2, fmaf(u2, fmaf(u2, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return c * (fabsf(u) < 0.25f ? near : far);
}
// A sum of rounded probabilities, two a word.
template <bool BF16>
__device__ __forceinline__ float add2(uint32_t p, float sum) {
    if constexpr (BF16)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), __builtin_bit_cast(bf16x2, kOnes<true>), sum, false);
    else
        return __builtin_amdgcn_fdot2(as_h2(p), as_h2(kOnes<false>), sum, false);
}

// ---- few columns: decode ---------------------------------------------------------------

// One workgroup: an item's tokens of one kv head for up to 16 columns, 32 tokens per
// wave and pass.  Lane (i, t) of K holds token i, columns 32 s + 8 t ..; of V the columns
// VC i .. VC i + VC - 1 of tokens 4 t .. 4 t + 3 of both halves, turned into the A operands of VC products
// by byte permutations: V's row order in the result is free.  K's registers are loaded
// again as soon as its products are made, V's likewise.  The waves meet once, at the end.
// The probabilities enter in two 16-bit parts: the products wait for memory anyway.
//
// What bounds it: with many tokens memory.  64 requests of up to 4096 tokens, 28 heads of 128 over 4, are 288 MB in 61 us
// with the joining launch, 4.7 TB/s of the 6.2 that reads alone reach (45 us where the cache of 256 MB holds most of it);
// with few the chain of lengths, page, K, V, parts: one of 1100 tokens takes 7.2 us and the joining launch 3.9.
// About 512, 768, 1024 and 1536 items took 65.8, 66.0, 67.1 and 66.0 us there, 26.6, 26.3, 27.9 and 29.5 for 4 requests of up
// to 16384 tokens.
//
// Three waves a SIMD, 170 registers each, but for heads of 128 in fp16 with shaped scores, which would spill (175).  With
// two, a window of 4096 over 8 requests, 32 heads over 8, took 30.7 us for 27.9.
template <int HD, bool BF16, bool SHAPED>
__global__ __launch_bounds__(kThreads, HD == 128 && !BF16 && SHAPED ? 2 : 3) void awq_kv16_decode_kernel(Kv16AttnArgs a) {
    constexpr int kSteps = HD / 32;
    constexpr int VC = HD / 16;            // V columns per lane
    constexpr int VW = VC / 2;             // words of them
    constexpr int kStride = HD + 4;        // floats per column of the reduction buffer
    typedef uint32_t vwords __attribute__((ext_vector_type(VW)));
    __shared__ float m_lds[kWaves][kCols], l_lds[kWaves][kCols], unit_lds[kCols];
    __shared__ int seen_lds[kCols];
    __shared__ __align__(16) float o_lds[kWaves][kCols][kStride];

    Item it;
    uint32_t head_of;
    const int kvh = a.s.kvh, item = (int)div_by(blockIdx.x, (uint32_t)kvh, a.kvh_inv, head_of), g = (int)head_of;
    if (!find_item<kCols, kKeys>(a, item, a.decode_target, it)) {
        if (blockIdx.x == gridDim.x - 1) fill_rows(a);   // the grid's last workgroup has no item
        return;
    }
    if (g == 0) write_records(a, it, false);
    const int group = a.heads_each;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, t = lane >> 4;
    const int block = it.rel % it.blocks, split = it.rel / it.blocks;
    const int all_cols = columns(a, it.r.rows), c0 = block * kCols;
    const int cols = all_cols - c0 < kCols ? all_cols - c0 : kCols;
    const int n = walked(a, it.r.len);

    // This lane's column: row c / group of the request, head c % group; the tokens it sees, and
    // those that all columns and that any column sees (columns that see none do not count).
    const int c = c0 + (col < cols ? col : 0);
    const int row = c / group, head = g * group + c % group;
    const auto sees = a.range(it.b, it.r.row0, it.r.rows, it.r.len, row);
    const bool blind = sees.hi == 0;
    int lo_min = blind ? n : sees.lo, lo_max = blind ? 0 : sees.lo, hi_min = blind ? n : sees.hi, hi_max = sees.hi;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        lo_min = min(lo_min, __shfl_xor(lo_min, d));
        lo_max = max(lo_max, __shfl_xor(lo_max, d));
        hi_min = min(hi_min, __shfl_xor(hi_min, d));
        hi_max = max(hi_max, __shfl_xor(hi_max, d));
    }
    lo_min = __builtin_amdgcn_readfirstlane(lo_min);
    lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    hi_min = __builtin_amdgcn_readfirstlane(hi_min);
    hi_max = __builtin_amdgcn_readfirstlane(hi_max);
    int start = it.first + split * it.chunk;
    const int end = item_end(start, it.chunk, hi_max);
    if (start < lo_min) start = lo_min / kWaveKeys * kWaveKeys;

    struct Place {                         // of 16 tokens
        const uint16_t* at;
        bool there;
    };
    auto place = [&](int page, int key) {
        Place p;
        p.there = page >= 0 && page < a.s.num_pages;
        p.at = a.cache + ((int64_t)(p.there ? page : 0) * kvh + g) * a.s.block() + (key & (a.s.page() - 1)) * HD;
        return p;
    };
    u32x4 kw[2][kSteps];                   // token col, columns 32 s + 8 t .. of K
    vwords vw[2][4];                       // tokens 4 t + r, columns VC col .. of V
    const uint32_t k_ofs = col * HD + 8 * t, v_ofs = (HD << a.s.page_log2) + 4 * t * HD + VC * col;
    auto load_k = [&](const Place (&p)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) kw[h][s] = *reinterpret_cast<const u32x4*>(p[h].at + k_ofs + 32 * s);
    };
    auto load_v = [&](const Place (&p)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) vw[h][r] = *reinterpret_cast<const vwords*>(p[h].at + v_ofs + r * HD);
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

    u32x4 q[kSteps];
    const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(it.r.row0 + row) * a.ld + (int64_t)head * HD + 8 * t;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
    int exp = 0;
    if constexpr (BF16) {
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(fabsf(low16<true>(q[s][i])), fabsf(high16<true>(q[s][i]))));
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        exp = query_exp(fmaxf(mx, __shfl_xor(mx, 32)), SHAPED && a.softcap == 0.0f ? a.scale : 0.0f);
        const float up = __builtin_ldexpf(1.0f, exp);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] = scaled_bf16(q[s], up);
    }
    // Shaped scores are in their own unit, plain ones products of the scaled query:
    // every exponent is a difference of scores first, so that what they were rounded to on the way is
    // the same wherever two meet.
    const float unit = SHAPED ? kLog2e : unit_of(a.scale * kLog2e, exp);
    const float natural = unit_of(a.scale, exp), inv_cap = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
    const float slope = SHAPED && a.slopes ? a.slopes[head] : 0.0f;
    const int pos = it.r.len - it.r.rows + row;          // of a row that sees a token: 0 or more

    float m = -INFINITY, l = 0.0f;
    floatx4 acc[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) acc[v] = floatx4{0.f, 0.f, 0.f, 0.f};
    while (key0 < end) {
        const bool more = key0 + kKeys < end;
        Place next[2];
        const int key1 = more ? key0 + kKeys : key0;
        next[0] = place(pages.page(a, key1, n), key1);
        next[1] = place(pages.page(a, key1 + 16, n), key1 + 16);

        floatx4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s[h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < kSteps; ++st) s[h] = mfma16<BF16>(kw[h][st], q[st], s[h]);
        }
        if (more) load_k(next);
        if constexpr (SHAPED) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = s[h][r] * natural;
                    if (a.softcap > 0.0f) x = capped(x, a.softcap, inv_cap);
                    s[h][r] = fmaf(-slope, fabsf((float)(pos - (key0 + 16 * h + 4 * t + r))), x);
                }
        }
        const bool gone = !now[0].there || !now[1].there;
        if (gone || key0 < lo_max || key0 + kWaveKeys > hi_min) {
            // Some column does not see all of these tokens.  A page outside the cache, or a value that is
            // not finite: NaN for the rows that see its token, and no product of it for the others.
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = key0 + 16 * h + 4 * t + r;
                    uint32_t most = 0;
#pragma unroll
                    for (int w = 0; w < VW; ++w) most = exponents<BF16>(most, vw[h][r][w]);
                    const bool odd = !now[h].there || (__ballot(not_finite<BF16>(most)) >> (16 * t) & 0xFFFFu) != 0;
                    s[h][r] = key < sees.lo || key >= sees.hi ? -INFINITY : odd ? NAN : s[h][r];
                    if (odd) vw[h][r] = vwords{};
                }
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int r = 1; r < 4; ++r) mx = fmaxf(mx, fmaxf(s[0][r], s[1][r]));
        if (__any((mx - m) * unit > kSlack16<BF16>)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            const float mn = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)));
            const float alpha = __builtin_amdgcn_exp2f(mn == -INFINITY ? 0.0f : (m - mn) * unit);
            l *= alpha;
#pragma unroll
            for (int v = 0; v < VC; ++v) acc[v] *= alpha;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.0f : m;     // nothing yet: every exponential is 0
        float p_scale = kPScale<BF16>;
        asm("" : "+s"(p_scale));                         // in a scalar register: a vector one is one too many
        float p[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[4 * h + r] = __builtin_amdgcn_exp2f(fmaf(s[h][r] - ref, unit, p_scale));
                l += p[4 * h + r];
            }
        u32x4 phi, plo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            phi[i] = pack2<BF16>(p[2 * i], p[2 * i + 1]);
            plo[i] = pack2<BF16>(p[2 * i] - low16<BF16>(phi[i]), p[2 * i + 1] - high16<BF16>(phi[i]));
        }
#pragma unroll
        for (int v = 0; v < VC; ++v) {
            constexpr uint32_t kLow = 0x05040100u, kHigh = 0x07060302u;
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = __builtin_amdgcn_perm(vw[i >> 1][2 * (i & 1) + 1][v / 2], vw[i >> 1][2 * (i & 1)][v / 2], v & 1 ? kHigh : kLow);
            acc[v] = mfma16<BF16>(w, plo, acc[v]);
            acc[v] = mfma16<BF16>(w, phi, acc[v]);
        }
        if (more) load_v(next);
        now[0] = next[0];
        now[1] = next[1];
        key0 += kKeys;
    }

    // This lane: rows 4 t + r of each product, i.e. columns VC (4 t + r) + v of column `col`.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (t == 0) {
        m_lds[wave][col] = m;
        l_lds[wave][col] = l;
        if (wave == 0) {
            seen_lds[col] = sees.hi;
            unit_lds[col] = unit;
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int v = 0; v < VC; v += 4)
            *reinterpret_cast<floatx4*>(&o_lds[wave][col][VC * (4 * t + r) + v]) =
                floatx4{acc[v][r], acc[v + 1][r], acc[v + 2][r], acc[v + 3][r]};
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
            const float al = __builtin_amdgcn_exp2f((m_lds[w][k] - ref) * unit_lds[k]);
            sum = fmaf(al, o_lds[w][k][d], sum);
            ls = fmaf(al, l_lds[w][k], ls);
        }
        if (it.splits == 1) {
            const int cc = c0 + k, r = cc / group, h = g * group + cc % group;
            const float y = seen_lds[k] == 0 ? 0.0f : sum / ls;
            reinterpret_cast<uint16_t*>(a.out)[((int64_t)(it.r.row0 + r) * a.nh + h) * HD + d] = to16<BF16>(y);
        } else {
            float* dst = a.part + (((int64_t)item * kvh + g) * kCols + k) * (HD + a.kExtra);
            dst[d] = sum;
            if (d == 0) {
                dst[HD] = mx;
                dst[HD + 1] = ls;
                dst[HD + 2] = unit_lds[k];
            }
        }
    }
}

// ---- many columns: tiles ---------------------------------------------------------------

// Two and four direct loads to neighbouring kilobytes of LDS, from as many of memory: the instruction's offset counts in
// both, and M0 is written once (awq_device.h, buffer_load_lds_x4).
__device__ __forceinline__ void buffer_load_lds_2x4(u32x4 rsrc, uint32_t v0, uint32_t v1, uint32_t lds_base) {
    asm volatile(
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %2, 0 offen lds\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen offset:1024 lds"
        :
        : "v"(v0), "v"(v1), "s"(rsrc), "s"(lds_base)
        : "memory", "m0");
}
__device__ __forceinline__ void buffer_load_lds_4x4(u32x4 rsrc, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3,
                                                    uint32_t lds_base) {
    asm volatile(
        "s_mov_b32 m0, %5\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %4, 0 offen lds\n\t"
        "buffer_load_dwordx4 %1, %4, 0 offen offset:1024 lds\n\t"
        "buffer_load_dwordx4 %2, %4, 0 offen offset:2048 lds\n\t"
        "buffer_load_dwordx4 %3, %4, 0 offen offset:3*1024 lds"
        :
        : "v"(v0), "v"(v1), "v"(v2), "v"(v3), "s"(rsrc), "s"(lds_base)
        : "memory", "m0");
}
// The 16-byte chunks of a token's row in LDS are swizzled by this.  An operand of K is
// one chunk of 32 tokens, a transposing read of V four neighbouring chunks of four
// tokens each: both touch every bank once.
template <int HD>
__device__ __forceinline__ constexpr int swizzle(int token) {
    return HD == 128 ? (token & 3) << 2 | (token >> 2 & 3) : (token >> 1 & 1) << 2 | (token >> 2 & 3);
}

// Over some columns: the first and the last of their first tokens, and of the ends of what they see.  (Columns that see none
// count in lo_max and hi_max alone, as 0.)
struct Span {
    int lo_min, lo_max, hi_min, hi_max;
};
// Of rows r0 .. r1 of a request, where no row has a first token of its own: both ends go up with the rows, and rows before the
// request's first token see none.  Scalar work: over the lanes, and with the query asked for
// after it, a prompt of 256 rows took 16.4 us for 14.3.
__device__ __forceinline__ Span rising_span(const Kv16AttnArgs& a, const Item& it, int n, int r0, int r1, int prefix) {
    const int none = it.r.rows - it.r.len;
    if (r0 < none) r0 = none;
    if (r0 > r1) return Span{n, 0, n, 0};
    const auto x = a.seen(it.r.rows, it.r.len, r0, prefix, 0), y = a.seen(it.r.rows, it.r.len, r1, prefix, 0);
    return Span{x.lo, y.lo, x.hi, y.hi};
}
template <class Op>
__device__ __forceinline__ int wave_int(int v, Op op) {
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true));   // row_half_mirror
    v = op(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true));   // row_mirror
    auto row = [&](int lane) { return __builtin_amdgcn_readlane(v, lane); };
    return op(op(row(0), row(16)), op(row(32), row(48)));
}
__device__ __forceinline__ Span wave_span(const Span& s) {
    auto least = [](int x, int y) { return x < y ? x : y; };
    auto most = [](int x, int y) { return x > y ? x : y; };
    return Span{wave_int(s.lo_min, least), wave_int(s.lo_max, most), wave_int(s.hi_min, least), wave_int(s.hi_max, most)};
}

// One workgroup: 128 columns of one kv head, 32 a wave, over an item's tokens in tiles of
// 64.  K and V go from memory to LDS without passing registers, the next tile's under
// this one's products: two buffers and one barrier a tile.  V is transposed as it is
// read (ds_read_b64_tr_b16).  Of a tile the scores' maximum comes first; then each exponential is taken under a
// product of the next tile's scores, which need the matrix unit and not these registers.  Products of 32 columns
// because a wave then reads each operand of K and V once for 32 columns: with 16, LDS would give them at
// twice the rate it has.
//
// What bounds it: instructions.  The 64 x 32 exponentials and the steps around them take a wave as long as its
// products, and two waves of a SIMD overlap the two only in part.  A prompt of 6001 rows, 28 heads of 128 over 4,
// is 258 GFLOP in 305 us, 847 TFLOP/s, where a large product of a library reaches 1158; of zeros, at the clock that less power
// allows, it took 252.  Before its first tile a workgroup spends 4 us on its item, the rows' ranges, the query and the table,
// so with few tiles the time is that: 256 rows take 14.3 us, 1024 32.
//
// PARTS = 2: two groups of four waves take every other tile and meet through LDS, where whole workgroups of
// four would be one round and leave CUs half empty (attention_plan16).  Prompts of 1200 / 1777 / 2300 rows: 29 / 41 / 62 us
// against 35 / 50 / 67; with 6001, 325 against 305, for eight waves meet at each barrier.
template <int HD, bool BF16, bool SHAPED, int PARTS>
__global__ __launch_bounds__(256 * PARTS, 2) void awq_kv16_tile_kernel(Kv16AttnArgs a) {
    constexpr int kKS = HD / 16;                         // k-steps of S
    constexpr int kDb = HD / 32;                         // blocks of V's columns
    constexpr int kChunks = HD / 8;
    constexpr int kLoads = 16 * HD * 2 / 1024;           // of a wave: 16 tokens of K or V
    constexpr int kHalf = kTileKeys * HD;                // elements of K or V in a buffer
    // [group of waves][stage]; at the end the second group's sums
    __shared__ __align__(1024) uint16_t kv_lds[PARTS][2][2 * kHalf];
    __shared__ __align__(8) uint16_t odd_lds[PARTS][2][4];

    Item it;
    uint32_t head_of;
    const int kvh = a.s.kvh, item = (int)div_by(blockIdx.x, (uint32_t)kvh, a.kvh_inv, head_of), g = (int)head_of;
    if (!find_item<k16Cols, kTileKeys>(a, item, a.tile_target, it)) {
        if (blockIdx.x == gridDim.x - 1 && a.limit == 0) fill_rows(a);
        return;
    }
    if (g == 0) write_records(a, it, true);
    const int group = a.heads_each;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3), part = PARTS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int col = lane & 31, half = lane >> 5;
    // The last blocks, which see the most tokens, start first.
    const int split = it.rel / it.blocks, block = it.blocks - 1 - (it.rel - split * it.blocks);
    const int all_cols = columns(a, it.r.rows), c0 = block * k16Cols;
    const int n = walked(a, it.r.len);

    const int last = all_cols - 1, local = 32 * wave + col, c = c0 + local, cc = min(c, last);
    auto over_group = [&](int column, uint32_t& rest) { return (int)div_by((uint32_t)column, (uint32_t)group, a.heads_inv, rest); };
    auto row_of = [&](int column) {
        uint32_t rest;
        return over_group(column, rest);
    };
    uint32_t in_group;
    const int row = over_group(cc, in_group), head = g * group + (int)in_group;
    // Loads come back in order: what says which tokens are seen first, then the table, then this lane's query, columns
    // 16 s + 8 half .. of the head, then the tiles.
    const int prefix = a.prefix ? a.prefix[it.b] : 0;
    int first_of = 0, first_two[2] = {};                 // of this lane's column; of two of the workgroup's 128
    if (a.first) {
        first_of = a.first[it.r.row0 + row];
#pragma unroll
        for (int i = 0; i < 2; ++i) first_two[i] = a.first[it.r.row0 + row_of(min(c0 + 64 * i + lane, last))];
    }
    // The table's entries from a tile's first page on are a lane's each, 64 of them; `lost` has a bit for
    // those of the request's tokens that are no page of the cache.  First those from the item's begin on, which its
    // first tile may lie behind.
    int start = it.first + split * it.chunk;
    const int32_t* table = a.tables + (int64_t)it.b * a.width;
    const int log2 = a.s.page_log2;
    const int held = (n + a.s.page() - 1) >> log2;       // pages of the request's tokens, one past the table's too
    int first = 0, entry = 0;
    uint64_t lost = 0;
    auto ask = [&](int key0) {
        first = __builtin_amdgcn_readfirstlane(key0 >> log2);
        const int index = first + lane;
        entry = index < min(a.width, held) ? table[index] : -1;
    };
    auto look = [&] {
        const bool there = (uint32_t)entry < (uint32_t)a.s.num_pages;
        lost = __ballot(!there && first + lane < held);
        entry = there ? entry : 0;
    };
    ask(start);
    u32x4 q[kKS];
    {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(it.r.row0 + row) * a.ld + (int64_t)head * HD + 8 * half;
#pragma unroll
        for (int s = 0; s < kKS; ++s) q[s] = *reinterpret_cast<const u32x4*>(src + 16 * s);
        __builtin_amdgcn_sched_barrier(0);
    }
    const auto sees = a.seen(it.r.rows, it.r.len, row, prefix, first_of);
    const bool blind = sees.hi == 0;
    // What the workgroup's columns see, and the wave's.
    Span wg, mine;
    if (a.first) {
        wg = Span{n, 0, n, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {                    // (the last column again past it)
            const auto r = a.seen(it.r.rows, it.r.len, row_of(min(c0 + 64 * i + lane, last)), prefix, first_two[i]);
            wg = Span{r.hi ? min(wg.lo_min, r.lo) : wg.lo_min, max(wg.lo_max, r.lo), r.hi ? min(wg.hi_min, r.hi) : wg.hi_min,
                      max(wg.hi_max, r.hi)};
        }
        wg = wave_span(wg);
        mine = wave_span(Span{blind ? n : sees.lo, sees.lo, blind ? n : sees.hi, sees.hi});
    } else {
        const int w0 = c0 + 32 * wave;
        wg = rising_span(a, it, n, row_of(c0), row_of(min(c0 + k16Cols - 1, last)), prefix);
        mine = rising_span(a, it, n, row_of(min(w0, last)), row_of(min(w0 + 31, last)), prefix);
    }
    const int wg_lo_max = wg.lo_max, wg_hi_min = wg.hi_min;
    const int lo_min = mine.lo_min, lo_max = mine.lo_max, hi_min = mine.hi_min, hi_max = mine.hi_max;
    const int end = item_end(start, it.chunk, wg.hi_max);
    if (start < wg.lo_min) start = wg.lo_min / kTileKeys * kTileKeys;
    const int all_tiles = end > start ? (end - start + kTileKeys - 1) / kTileKeys : 0;
    // Tile `tile` of this group is the (PARTS tile + part)-th.
    const int steps = (all_tiles + PARTS - 1) / PARTS, tiles = (all_tiles + PARTS - 1 - part) / PARTS;
    start += part * kTileKeys;
    constexpr int kStep = PARTS * kTileKeys;

    // Loads: wave w brings tokens 16 w .. of the tile.  A place past the
    // last token, or in a page outside the cache, lies past its resource's end and reads as zeros.
    look();
    const uint64_t cache_g = reinterpret_cast<uint64_t>(a.cache) + 2 * g * a.s.block();
    const uint32_t page_bytes = (uint32_t)(2 * kvh * a.s.block());      // of all heads: 2^29 at most
    const int r0 = lane / kChunks;                       // a load's rows begin with this lane's token
    const uint32_t l_ofs = r0 * (HD * 2) + ((lane % kChunks) ^ swizzle<HD>(r0)) * 16;
    const uint32_t k_to = lds_addr(&kv_lds[0][0][0]) + part * (8 * kHalf) + wave * (16 * HD * 2), v_to = k_to + 2 * kHalf;
    struct Place {                                       // of this wave's tokens of a tile
        uint64_t at;
        int tokens;
        uint32_t gone;                                   // the tile's blocks of 16 tokens in pages outside the cache, a bit each
    };
    auto locate = [&](int key0) {
        if (((key0 + kTileKeys - 1) >> log2) - first >= 64) {
            ask(key0);
            look();
        }
        const int key = key0 + 16 * wave, left = n - key;
        Place p = {0, left < 16 ? (left > 0 ? left : 0) : 16, 0};
        if (lost) {
#pragma unroll
            for (int j = 0; j < 4; ++j) p.gone |= (uint32_t)(lost >> (((key0 + 16 * j) >> log2) - first) & 1) << j;
            p.tokens = p.gone >> wave & 1 ? 0 : p.tokens;
        }
        p.tokens = __builtin_amdgcn_readfirstlane(p.tokens);
        const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(entry, (key >> log2) - first);
        p.at = cache_g + (uint64_t)page * page_bytes + (uint32_t)((key & (a.s.page() - 1)) * (HD * 2));
        return p;
    };
    auto load = [&](uint64_t at, int tokens, uint32_t to) {
        u32x4 r = raw_rsrc(reinterpret_cast<const void*>(at), tokens * (HD * 2));
#pragma unroll
        for (int i = 0; i < 3; ++i) r[i] = (uint32_t)__builtin_amdgcn_readfirstlane(r[i]);   // (the same for the wave)
        constexpr uint32_t kFlip = HD == 128 ? 16 : 32;  // the swizzle of the tokens of a load after
        if constexpr (kLoads == 4)
            buffer_load_lds_4x4(r, l_ofs, l_ofs ^ kFlip, l_ofs ^ (2 * kFlip), l_ofs ^ (3 * kFlip), to);
        else
            buffer_load_lds_2x4(r, l_ofs, l_ofs ^ kFlip, to);
    };
    auto load_k = [&](const Place& p, int stage) { load(p.at, p.tokens, k_to + stage * (4 * kHalf)); };
    auto load_v = [&](const Place& p, int stage) { load(p.at + ((HD * 2) << log2), p.tokens, v_to + stage * (4 * kHalf)); };
    int exp = 0;
    if constexpr (BF16) {
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < kKS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(fabsf(low16<true>(q[s][i])), fabsf(high16<true>(q[s][i]))));
        exp = query_exp(fmaxf(mx, __shfl_xor(mx, 32)), SHAPED && a.softcap == 0.0f ? a.scale : 0.0f);
        const float up = __builtin_ldexpf(1.0f, exp);
#pragma unroll
        for (int s = 0; s < kKS; ++s) q[s] = scaled_bf16(q[s], up);
    }
    Place now = {}, next = {};                           // of this tile and the next
    if (tiles > 0) {
        now = locate(start);
        load_k(now, 0);
        load_v(now, 0);
    }
    if (tiles > 1) {
        next = locate(start + kStep);
        load_k(next, 1);
    }

    // Shaped scores are formed in powers of two, plain ones are products of the scaled query.
    const float unit = SHAPED ? 1.0f : unit_of(a.scale * kLog2e, exp);
    const float natural = unit_of(a.scale, exp), inv_cap = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
    const float cap2 = a.softcap * kLog2e, cap_in = fminf(unit_of(a.scale, exp) * inv_cap * 2.8853900817779268f, __FLT_MAX__);
    const float slope = SHAPED && a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    const float natural2 = fminf(natural * kLog2e, __FLT_MAX__);
    const int pos = it.r.len - it.r.rows + row;
    wait_vm_stores();                                    // the first tiles
    lds_barrier();

    // Operand addresses: token col (+ 32) and chunk 2 s + half of K; of V, lane 4 m + j of
    // 16 supplies four columns of token 4 half + m, and its group's other half of the 32 columns.
    const uint32_t k_at = lds_addr(&kv_lds[0][0][0]) + part * (8 * kHalf) + col * (HD * 2) + (half ^ swizzle<HD>(col)) * 16;
    const int vm = 4 * half + (lane >> 2 & 3), vj = lane & 3;
    const uint32_t v_at = lds_addr(&kv_lds[0][0][0]) + part * (8 * kHalf) + 2 * kHalf + vm * (HD * 2) + ((2 * (lane >> 4 & 1) + (vj >> 1)) ^ swizzle<HD>(vm)) * 16 + (vj & 1) * 8;

    // A score s counts 2^(s unit + ref), scaled by kPScale: the sum is one fused step, rounded once.  Where ref is
    // large (`big`, for the whole wave) its own rounding would show; there it is (s - m) unit.
    constexpr float kBig = 256.0f, kMost = kPScale<BF16> + kSlack16<BF16>;
    float ref = 0.0f, m = 0.0f, l = 0.0f;
    bool some = false, big = false;                      // some: the column has met a score
    floatx16 acc[kDb];
#pragma unroll
    for (int d = 0; d < kDb; ++d) acc[d] = floatx16{};
    floatx16 s[2];
    // Operands are read two steps ahead of their products, and fences keep it so: the scheduler by itself reads
    // each right before its product and waits for LDS every time.
    u32x4 kf[2][2];
    // Addresses of a stage are formed from one opaque register each tile: sixteen of them, hoisted, would be too many.
    typedef const __attribute__((address_space(3))) u32x4* lds16;
    auto in_stage = [&](uint32_t at, int stage) {
        at += stage * (4 * kHalf);
        asm volatile("" : "+v"(at));
        return at;
    };
    auto read_k = [&](uint32_t at, int st) {             // of one k-step, both blocks of 32 tokens
#pragma unroll
        for (int b = 0; b < 2; ++b) kf[st % 2][b] = *(lds16)(uintptr_t)((at ^ (32 * st)) + b * (32 * HD * 2));
    };
    auto score = [&](uint32_t at, int st) {
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = mfma32<BF16>(kf[st % 2][b], q[st], st ? s[b] : floatx16{});
        if (st + 2 < kKS) read_k(at, st + 2);
    };
    auto all_scores = [&](int stage) {
        const uint32_t at = in_stage(k_at, stage);
        read_k(at, 0);
        read_k(at, 1);
#pragma unroll
        for (int st = 0; st < kKS; ++st) {
            score(at, st);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (tiles > 0) all_scores(0);
    for (int tile = 0; tile < tiles; ++tile) {
        const int key0 = start + tile * kStep;
        char* v_base = reinterpret_cast<char*>(&kv_lds[part][tile & 1][kHalf]);
        Place after = {};
        if (tile + 2 < tiles) after = locate(key0 + 2 * kStep);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // what this wave has under way: the tile's V, the next one's K
        // Where some column does not see all of the tile's tokens, a value of V that is not finite must
        // not meet its probability of zero: each wave takes such values out of the tokens it
        // brought, and the rows that see them get NaN by their scores.
        const bool edge = key0 < wg_lo_max || key0 + kTileKeys > wg_hi_min;
        if (edge) {
            constexpr int kRows = 1024 / (HD * 2);       // tokens of a read
            uint32_t odd = 0;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                u32x4* at = reinterpret_cast<u32x4*>(v_base + wave * (16 * HD * 2) + 1024 * i + 16 * lane);
                u32x4 w = *at;
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) most = exponents<BF16>(most, w[j]);
                const uint64_t hit = __ballot(not_finite<BF16>(most));
                if (hit) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = finite_part<BF16>(w[j]);
                    *at = w;
#pragma unroll
                    for (int j = 0; j < kRows; ++j)
                        if (hit >> (kChunks * j) & ((1u << kChunks) - 1)) odd |= 1u << (kRows * i + j);
                }
            }
            if (lane == 0) odd_lds[part][tile & 1][wave] = (uint16_t)odd;
        }
        lds_barrier();                                   // the next tile's K and this one's V are there, the others read by all
        const bool more = tile + 1 < tiles;
        const int stage = (tile + 1) & 1;
        if (tile + 2 < tiles) load_k(after, tile & 1);
        if (more) load_v(next, stage);
        const uint32_t gone = now.gone;
        now = next;
        next = after;
        if (key0 >= hi_max || key0 + kTileKeys <= lo_min) {   // nothing for this wave
            if (more) all_scores(stage);
            continue;
        }
        uint64_t bad = 0;                                // tokens that give NaN, a bit each
        if (edge) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(&odd_lds[part][tile & 1][0]);
            bad = (uint64_t)__builtin_amdgcn_readfirstlane(w.y) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane(w.x);
        }
        if (gone) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (gone >> j & 1) bad |= 0xFFFFull << (16 * j);
        }
        if constexpr (SHAPED) {
            if (a.softcap == 0.0f) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i / 16][i % 16] *= natural2;
            } else if (a.softcap <= kPlainCap) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float e = __builtin_amdgcn_exp2f(s[i / 16][i % 16] * cap_in);
                    s[i / 16][i % 16] = fmaf(-2.0f * cap2, __builtin_amdgcn_rcpf(e + 1.0f), cap2);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    s[i / 16][i % 16] = capped(s[i / 16][i % 16] * natural, a.softcap, inv_cap) * kLog2e;
                    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // few at a time: registers
                }
            }
            if (a.slopes) {
                const float far = (float)(pos - key0 - 4 * half);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    s[i / 16][i % 16] = fmaf(-slope, fabsf(far - (float)(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4)), s[i / 16][i % 16]);
            }
        }
        if (key0 + kTileKeys > hi_min) {
            const int end = sees.hi - key0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 32; ++i)
                s[i / 16][i % 16] = 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4 < end ? s[i / 16][i % 16] : -INFINITY;
        }
        if (key0 < lo_max) {
            const int begin = sees.lo - key0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 32; ++i)
                s[i / 16][i % 16] = 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4 >= begin ? s[i / 16][i % 16] : -INFINITY;
        }
        if (bad) {
            const uint64_t mine = bad >> (4 * half);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int in = 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4, key = key0 + in + 4 * half;
                if (mine >> in & 1 && key >= sees.lo && key < sees.hi) s[i / 16][i % 16] = NAN;
            }
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fmaxf(s[0][i], s[1][i]));
        if (__any(!some || big || fmaf(mx, unit, ref) > kMost)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            float alpha = 1.0f;
            if (!some) {
                if (mx != -INFINITY) {
                    m = mx;
                    ref = kPScale<BF16> - mx * unit;
                    some = true;
                }
            } else if (big) {
                const float to = fmaxf(m, mx);
                alpha = __builtin_amdgcn_exp2f((m - to) * unit);
                m = to;
            } else {
                const float up = fmaf(mx, unit, ref) - kPScale<BF16>, to = ref - up;
                m = up > 0.0f ? mx : (kPScale<BF16> - ref) / unit;
                alpha = up > 0.0f ? __builtin_amdgcn_exp2f(to - ref) : 1.0f;
                ref = up > 0.0f ? to : ref;
            }
            big = big || __any(fabsf(ref) > kBig);
            l *= alpha;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < kDb; ++d) {
                acc[d] *= alpha;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        float y[32];
        if (!big) {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = SHAPED ? s[i / 16][i % 16] + ref : fmaf(s[i / 16][i % 16], unit, ref);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = fmaf(s[i / 16][i % 16] - m, unit, kPScale<BF16>);
        }
        const uint32_t k_now = in_stage(k_at, stage), v_now = in_stage(v_at, tile & 1);
        if (more) {
            read_k(k_now, 0);
            if (!SHAPED) read_k(k_now, 1);               // (shaped scores have more else in registers)
        }
        // V's operands: product j is of k-step j / kDb and column block j % kDb.
        constexpr int kProducts = 4 * kDb, kAhead = 4;
        u32x4 vf[kAhead];
        auto read_v = [&](int j) {
            typedef __attribute__((address_space(3))) s16x4* lds4;
            const uint32_t at = 16 * (j / kDb) * (HD * 2), flip = 64 * (j % kDb);
            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)((v_now ^ flip) + at)));
            const u32x2 z = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)((v_now ^ flip ^ 32) + at + 8 * (HD * 2))));
            vf[j % kAhead] = u32x4{x.x, x.y, z.x, z.y};
        };
        // The exponentials under the next tile's scores, then the sums.  A probability is rounded to the cache's type, once, half a
        // step as the result's own rounding, and the rounded ones are summed.  One part / two: the results are off from 64 bits by
        // 0.00026 / 0.00021 in fp16 (the plain form by 0.00021), 0.00170 / 0.00162 in bf16; a prompt of 6001 rows takes 302 / 385 us,
        // of 1777 42 / 50, 2500 rows of packed documents 32 / 36.
        u32x4 p[4];
        auto weigh = [&](int i) {
            const uint32_t w = pack2<BF16>(__builtin_amdgcn_exp2f(y[i]), __builtin_amdgcn_exp2f(y[i + 1]));
            l = add2<BF16>(w, l);
            p[i / 8][i % 8 / 2] = w;
        };
        constexpr int kEach = 32 / kKS;                  // probabilities of a k-step
        if (more) {
            if (SHAPED) read_k(k_now, 1);
#pragma unroll
            for (int st = 0; st < kKS; ++st) {
                score(k_now, st);
#pragma unroll
                for (int i = 0; i < kEach; i += 2) weigh(kEach * st + i);
                if (st >= kKS - 2)
#pragma unroll
                    for (int j = 0; j < kAhead / 2; ++j) read_v(kAhead / 2 * (st - kKS + 2) + j);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // Opaque: what both branches have in common must not be moved before them, away from the products.
#pragma unroll
            for (int i = 0; i < 32; ++i) asm volatile("" : "+v"(y[i]));
#pragma unroll
            for (int i = 0; i < 32; i += 2) weigh(i);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) read_v(j);
        }
#pragma unroll
        for (int j = 0; j < kProducts; ++j) {
            acc[j % kDb] = mfma32<BF16>(vf[j % kAhead], p[j / kDb], acc[j % kDb]);
            if (j + kAhead < kProducts) read_v(j + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    float most = !some ? -INFINITY : big ? m : (kPScale<BF16> - ref) / unit;
    if constexpr (PARTS == 2) {
        // The groups meet: the second's sums through LDS, each weighted by its reference.
        floatx4* meet = reinterpret_cast<floatx4*>(&kv_lds[0][0][0]) + wave * (64 * (4 * kDb + 1)) + lane;
        static_assert(sizeof(kv_lds) >= 4 * 64 * (4 * kDb + 1) * sizeof(floatx4), "room for a group's sums");
        if (tiles < steps) lds_barrier();                // the other group has one more
        if (steps > 0) {
            lds_barrier();                               // the last tiles are read by all
            if (part == 1) {
#pragma unroll
                for (int d = 0; d < kDb; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        meet[64 * (4 * d + j)] = floatx4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
                meet[64 * 4 * kDb] = floatx4{most, l, ref, big ? 1.0f : 0.0f};
            }
            lds_barrier();
        }
        if (part == 1) return;
        if (steps > 0) {
            const floatx4 other = meet[64 * 4 * kDb];
            // Powers of two that bring each group's sums to the larger reference.  (One without a score has sums of
            // 0, or of NaN.)
            float up = 0.0f;
            if (some && other[0] != -INFINITY) up = big || other[3] != 0.0f ? (other[0] - most) * unit : ref - other[2];
            const float mine = __builtin_amdgcn_exp2f(-fmaxf(up, 0.0f)), add = __builtin_amdgcn_exp2f(fminf(up, 0.0f));
            most = fmaxf(most, other[0]);
            l = l * mine + other[1] * add;
#pragma unroll
            for (int d = 0; d < kDb; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const floatx4 o = meet[64 * (4 * d + j)];
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[d][4 * j + r] = acc[d][4 * j + r] * mine + o[r] * add;
                }
        }
    }
    l += __shfl_xor(l, 32);
    if (c >= all_cols) return;
    // This lane: columns 32 d + 8 j + 4 half + r of the head.
    if (it.splits == 1) {
        const float inv = 1.0f / l;
        // Halves of a wave trade every other four columns: eight neighbouring ones a lane.
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + ((int64_t)(it.r.row0 + row) * a.nh + head) * HD + 8 * half;
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = 4 * j + 2 * i;
                    w[i] = blind ? 0u : pack2<BF16>(acc[d][at] * inv, acc[d][at + 1] * inv);
                }
                const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                *reinterpret_cast<u32x4*>(dst + 32 * d + 8 * j) = u32x4{x[0], y[0], x[1], y[1]};
            }
    } else {
        float* dst = a.tile_part + (((int64_t)item * kvh + g) * k16Cols + local) * (HD + a.kExtra);
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<floatx4*>(dst + 32 * d + 8 * j + 4 * half) =
                    floatx4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
        if (half == 0) *reinterpret_cast<floatx4*>(dst + HD) = floatx4{most, l, unit, 0.0f};
    }
}

// ---- joining the items of a row -----------------------------------------------------

template <int HD, int WAVES, bool BF16>
__global__ __launch_bounds__(kThreads) void awq_kv16_combine_kernel(Kv16AttnArgs a) {
    combine_items<HD, WAVES, BF16>(a);
}

// ---- launches ----------------------------------------------------------------------------

template <int HD, bool BF16, bool SHAPED>
hipError_t launch(Kv16AttnArgs a, hipStream_t stream) {
    const AttentionPlan16 p = attention_plan16(a.requests, a.total, a.max_query, a.nh / a.s.kvh, a.s.kvh);
    a.limit = p.limit;
    a.decode_target = p.decode_target;
    a.tile_target = p.tile_target;
    a.combine = p.combine;
    a.heads_each = a.nh / a.s.kvh;
    a.heads_inv = div_inverse((uint32_t)a.heads_each);
    a.kvh_inv = div_inverse((uint32_t)a.s.kvh);
    a.records = reinterpret_cast<i32x4*>(a.part);
    a.part += (size_t)a.total * (sizeof(i32x4) / sizeof(float));
    a.tile_part = a.part + p.decode_items * a.s.kvh * kCols * (HD + a.kExtra);
    if (p.decode) {
        hipLaunchKernelGGL((awq_kv16_decode_kernel<HD, BF16, SHAPED>), dim3((unsigned)(p.decode_items * a.s.kvh)), dim3(kThreads), 0,
                           stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.tile) {
        auto kernel = p.tile_parts == 2 ? awq_kv16_tile_kernel<HD, BF16, SHAPED, 2> : awq_kv16_tile_kernel<HD, BF16, SHAPED, 1>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(p.tile_items * a.s.kvh)), dim3(256 * p.tile_parts), 0, stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.combine) {
        const int64_t all = (int64_t)a.total * a.nh, groups = all <= kFewUnits ? all : (all + 3) / 4;
        auto kernel = all <= kFewUnits ? awq_kv16_combine_kernel<HD, 4, BF16> : awq_kv16_combine_kernel<HD, 1, BF16>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(groups < kCombineGroups ? groups : kCombineGroups)), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace

// A launch holds 2^32 threads.
bool kv16_attn_fits(int requests, int total, int max_query, int nh, int kvh) {
    const AttentionPlan16 p = attention_plan16(requests, total, max_query, nh / kvh, kvh);
    return (p.decode_items > p.tile_items ? p.decode_items : p.tile_items) * kvh < ((int64_t)1 << 32) / 512;
}

size_t kv16_attn_workspace(int requests, int total, int max_query, int nh, int kvh, int hd) {
    return part_bytes(attention_plan16(requests, total, max_query, nh / kvh, kvh), total, kvh, hd + Kv16AttnArgs::kExtra);
}

hipError_t launch_kv16_attention(const Kv16AttnArgs& a, bool bf16, hipStream_t stream) {
    auto typed = [&](auto hd, auto type) {
        return a.shaped() ? launch<hd(), type(), true>(a, stream) : launch<hd(), type(), false>(a, stream);
    };
    constexpr std::integral_constant<int, 64> c64;
    constexpr std::integral_constant<int, 128> c128;
    if (a.s.hd == 64) return bf16 ? typed(c64, std::true_type{}) : typed(c64, std::false_type{});
    return bf16 ? typed(c128, std::true_type{}) : typed(c128, std::false_type{});
}

}  // namespace awq
