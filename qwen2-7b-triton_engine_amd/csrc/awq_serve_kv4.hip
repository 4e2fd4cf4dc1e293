// The 4-bit paged KV cache's write and read (include/awq_serving.h:
// awq_serve_kv4_append, awq_serve_kv4_gather).
//
// A group of G columns x of one token's head is held as
//   zero = fp16(min x),  r = (max x - zero) / 15,  scale = r rounded UP to 7
//   significant bits,  code = round((x - zero) / scale) in 0 .. 15.
// Rounded up, 15 scales reach the maximum; with 7 bits, code * scale (4 + 7 bits)
// is exact in fp16, so attention multiplies the matrix cores' operands out
// without a rounding.  It costs a step that is at most 1/64 coarser.
//
// What bounds them: at a decode step's few tokens latency, at a prompt's the start and end of
// workgroups and the loads, 80 bytes of cos, sin and RoPE partner for 16 of the row.  Eight
// columns a thread: one 16-byte load of the row, one of its RoPE partner, one
// 32-bit word of codes out.  k and v of a head go through the same lanes, since
// a token's head is stored as NaN when either cannot be held.  The arithmetic
// is unfused fp32 in the order of the formulas (contraction is off): codes are
// decided at the middle between two values, where one more or less rounding
// moves a value by a whole step.  For the same reason the quotients are true
// divisions, not products with a reciprocal.
// Measured in a graph, 28 query and 4 kv heads of 128, groups of 64, us: append 4.3 for 64 tokens,
// 11.7 for 2011 (9.2 without RoPE; a copy of its rows takes 6.0), gather 2.7 and 3.9.
#include "awq_serving.h"

#pragma clang fp contract(off)

namespace awq {
namespace {

constexpr int kThreads = 256;
constexpr float kMaxScale = 4032.0f;   // 16 of them, which attention forms, still fit fp16

// Minimum and maximum over each 2^STEPS neighbouring lanes (4, 8 or 16).
template <int LANES>
__device__ __forceinline__ void lanes_min_max(float& lo, float& hi) {
    auto step = [&](float l, float h) {
        lo = fminf(lo, l);
        hi = fmaxf(hi, h);
    };
    step(dpp_move<0xB1>(lo), dpp_move<0xB1>(hi));                                   // quad_perm [1,0,3,2]
    step(dpp_move<0x4E>(lo), dpp_move<0x4E>(hi));                                   // quad_perm [2,3,0,1]
    if constexpr (LANES >= 8) step(dpp_move<0x141>(lo), dpp_move<0x141>(hi));       // row_half_mirror
    if constexpr (LANES >= 16) step(dpp_move<0x140>(lo), dpp_move<0x140>(hi));      // row_mirror
}

struct Coded {
    half_t scale, zero;
    uint32_t code[8];
    bool held;                         // fp16 holds the group, and all of it is finite
};

// This lane's eight columns of a group of 8 LANES.
template <int LANES>
__device__ __forceinline__ Coded quantise(const float (&x)[8]) {
    float lo = x[0], hi = x[0];
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
        finite = finite && fabsf(x[e]) < INFINITY;   // false for a NaN
    }
    lanes_min_max<LANES>(lo, hi);
    Coded c;
    c.zero = (half_t)lo;
    const float z = (float)c.zero;
    const float r = fmaxf((hi - z) / 15.0f, 0.0f);
    float s = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, r) + 0x1FFFFu) & ~0x1FFFFu);
    if (s < 0x1p-17f) s = __builtin_ceilf(s * 0x1p24f) * 0x1p-24f;   // fp16's steps are coarser there
    c.held = finite && fabsf(z) < INFINITY && s <= kMaxScale;
    c.scale = (half_t)s;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = s > 0.0f ? __builtin_rintf((x[e] - z) / s) : 0.0f;
        c.code[e] = (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f);
    }
    return c;
}

// Threads: hd / 8 lanes for each (token, head): the query heads, then the kv
// heads (k and v together).
template <int HD, int G, bool BF16>
__global__ __launch_bounds__(kThreads) void awq_kv4_append_kernel(Kv4AppendArgs a, uint32_t heads, uint32_t inv) {
    constexpr int L = HD / 8;          // lanes of a head
    constexpr int kGroups = HD / G;
    const int64_t unit64 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
    const bool live = unit64 < (int64_t)a.tokens * heads;
    const uint32_t unit = live ? (uint32_t)unit64 : 0;
    const int j = threadIdx.x % L, d0 = 8 * j;
    uint32_t h;
    const uint32_t tok = div_by(unit, heads, inv, h);
    const int pos = a.positions[tok];
    const bool on_table = pos >= 0 && pos < a.max_pos;
    const uint16_t* row = reinterpret_cast<const uint16_t*>(a.qkv) + (int64_t)tok * a.ld;
    const bool is_q = h < (uint32_t)a.nh;
    const uint16_t* head = row + (int64_t)h * HD;   // k heads follow the query heads

    float x[8], y[8];
    load8<BF16>(head + d0, x);
    if (a.cos) {
        const bool low = j < L / 2;
        load8<BF16>(head + (low ? d0 + HD / 2 : d0 - HD / 2), y);
        const int64_t at = (int64_t)(on_table ? pos : 0) * HD + d0;
        const floatx4* c = reinterpret_cast<const floatx4*>(a.cos + at);
        const floatx4* s = reinterpret_cast<const floatx4*>(a.sin + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float p = low ? -y[e] : y[e];
            x[e] = x[e] * c[e / 4][e % 4] + p * s[e / 4][e % 4];
        }
    }
    if (is_q) {
        if (!on_table) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = NAN;
        }
        if (live) store8<BF16>(reinterpret_cast<uint16_t*>(a.q) + ((int64_t)tok * a.nh + h) * HD + d0, x);
    }
    // A query head beside a kv head in one wave goes along for the cross-lane
    // steps and stores nothing.
    if (__all(is_q)) return;
    const int g = is_q ? 0 : (int)h - a.nh;
    load8<BF16>(row + (int64_t)(a.nh + a.s.kvh + g) * HD + d0, y);
    const Coded k = quantise<G / 8>(x), v = quantise<G / 8>(y);
    const uint64_t bad = __ballot(!k.held || !v.held);
    const int first = (threadIdx.x & 63) / L * L;
    const bool held = ((bad >> first) & ((1ull << L) - 1)) == 0;
    const int slot = a.slots[tok];
    if (!live || is_q || !on_table || slot < 0 || (slot >> a.s.page_log2) >= a.s.num_pages) return;
    const int in_page = slot & (a.s.page() - 1);
    uint8_t* block = a.cache + ((int64_t)(slot >> a.s.page_log2) * a.s.kvh + g) * a.s.block();
    uint32_t kw = 0, vw = 0;
    if (held) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            kw |= k.code[e] << (4 * (e / 2 + 4 * (e % 2)));
            vw |= v.code[e] << (4 * e);
        }
    }
    uint32_t* kc = reinterpret_cast<uint32_t*>(block);
    uint32_t* vc = reinterpret_cast<uint32_t*>(block + a.s.k_bytes());
    kc[in_page * (HD / 8) + (j & 3) * (HD / 32) + (j >> 2)] = kw;
    vc[((in_page >> 2) * (HD / 8) + j) * 4 + (in_page & 3)] = vw;
    if (j % (G / 8) == 0) {
        const int gi = j / (G / 8);
        const half_t nan = (half_t)NAN;
        half2_t* ks = reinterpret_cast<half2_t*>(block + 2 * a.s.k_bytes());
        half_t* vs = reinterpret_cast<half_t*>(block + 2 * a.s.k_bytes() + a.s.scale_bytes());
        ks[in_page * kGroups + gi] = held ? half2_t{k.scale, k.zero} : half2_t{nan, nan};
        vs += ((in_page >> 2) * kGroups + gi) * 8 + (in_page & 3);
        vs[0] = held ? v.scale : (half_t)0.0f;
        vs[4] = held ? v.zero : (half_t)0.0f;
    }
}

template <int HD, int G, bool BF16>
__global__ __launch_bounds__(kThreads) void awq_kv4_gather_kernel(Kv4GatherArgs a, uint32_t inv) {
    constexpr int L = HD / 8, kGroups = HD / G;
    const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
    if (unit >= (int64_t)a.tokens * a.s.kvh) return;
    const int j = threadIdx.x % L;
    uint32_t g;
    const uint32_t tok = div_by((uint32_t)unit, a.s.kvh, inv, g);
    const int slot = a.slots[tok];
    float k[8], v[8];
    if (slot < 0 || (slot >> a.s.page_log2) >= a.s.num_pages) {
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = v[e] = NAN;
    } else {
        const int in_page = slot & (a.s.page() - 1), gi = j / (G / 8);
        const uint8_t* block = a.cache + ((int64_t)(slot >> a.s.page_log2) * a.s.kvh + g) * a.s.block();
        const uint32_t kw = reinterpret_cast<const uint32_t*>(block)[in_page * (HD / 8) + (j & 3) * (HD / 32) + (j >> 2)];
        const uint32_t vw =
            reinterpret_cast<const uint32_t*>(block + a.s.k_bytes())[((in_page >> 2) * (HD / 8) + j) * 4 + (in_page & 3)];
        const half2_t ks = reinterpret_cast<const half2_t*>(block + 2 * a.s.k_bytes())[in_page * kGroups + gi];
        const half_t* vs = reinterpret_cast<const half_t*>(block + 2 * a.s.k_bytes() + a.s.scale_bytes()) +
                           ((in_page >> 2) * kGroups + gi) * 8 + (in_page & 3);
        const float k_scale = (float)ks.x, k_zero = (float)ks.y, v_scale = (float)vs[0], v_zero = (float)vs[4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            k[e] = (float)((kw >> (4 * (e / 2 + 4 * (e % 2)))) & 15u) * k_scale + k_zero;
            v[e] = (float)((vw >> (4 * e)) & 15u) * v_scale + v_zero;
        }
    }
    const int64_t at = unit * HD + 8 * j;
    store8<BF16>(reinterpret_cast<uint16_t*>(a.k) + at, k);
    store8<BF16>(reinterpret_cast<uint16_t*>(a.v) + at, v);
}

// f(head size, group size, bf16) with all three as constants.
template <typename F>
hipError_t with_shape(const Kv4Shape& s, bool bf16, F f) {
    using std::integral_constant;
    auto typed = [&](auto hd, auto g) {
        return bf16 ? f(hd, g, std::true_type{}) : f(hd, g, std::false_type{});
    };
    constexpr integral_constant<int, 32> c32;
    constexpr integral_constant<int, 64> c64;
    constexpr integral_constant<int, 128> c128;
    const int group = s.hd / s.groups;
    if (s.hd == 64) return group == 32 ? typed(c64, c32) : typed(c64, c64);
    return group == 32 ? typed(c128, c32) : group == 64 ? typed(c128, c64) : typed(c128, c128);
}

}  // namespace

hipError_t launch_kv4_append(const Kv4AppendArgs& a, bool bf16, hipStream_t stream) {
    const uint32_t heads = (uint32_t)(a.nh + a.s.kvh);
    const int64_t threads = (int64_t)a.tokens * heads * (a.s.hd / 8);
    return with_shape(a.s, bf16, [&](auto hd, auto g, auto type) {
        hipLaunchKernelGGL((awq_kv4_append_kernel<hd(), g(), type()>), dim3((unsigned)((threads + kThreads - 1) / kThreads)),
                           dim3(kThreads), 0, stream, a, heads, div_inverse(heads));
        return hipGetLastError();
    });
}

hipError_t launch_kv4_gather(const Kv4GatherArgs& a, bool bf16, hipStream_t stream) {
    const int64_t threads = (int64_t)a.tokens * a.s.kvh * (a.s.hd / 8);
    return with_shape(a.s, bf16, [&](auto hd, auto g, auto type) {
        hipLaunchKernelGGL((awq_kv4_gather_kernel<hd(), g(), type()>), dim3((unsigned)((threads + kThreads - 1) / kThreads)),
                           dim3(kThreads), 0, stream, a, div_inverse(a.s.kvh));
        return hipGetLastError();
    });
}

}  // namespace awq
