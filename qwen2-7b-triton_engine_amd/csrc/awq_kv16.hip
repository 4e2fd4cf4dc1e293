// The 16-bit paged KV cache's write (include/awq_serving.h: awq_serve_kv16_append).
//
// What bounds it: at a decode step's few tokens latency, at a prompt's the bytes.  A thread
// has eight columns of a head's lower half and the eight that RoPE pairs them with, so
// that a row is read once, and that of kHeads heads of its token, which share cos
// and sin in registers.
#include "awq_serving.h"

namespace awq {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;

template <int HD, bool BF16>
__global__ __launch_bounds__(kThreads) void awq_kv16_append_kernel(Kv16AppendArgs a, uint32_t parts, uint32_t inv) {
    constexpr int L = HD / 16;         // lanes of a head
    const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
    if (unit >= (int64_t)a.tokens * parts) return;
    const int d0 = 8 * (threadIdx.x % L);
    uint32_t part;
    const uint32_t tok = div_by((uint32_t)unit, parts, inv, part);
    const int heads = a.nh + 2 * a.s.kvh, h0 = (int)part * kHeads;
    const uint16_t* row = reinterpret_cast<const uint16_t*>(a.qkv) + (int64_t)tok * a.ld + d0;
    u32x4 lo[kHeads], hi[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const uint16_t* src = row + (int64_t)(h0 + i < heads ? h0 + i : h0) * HD;
        lo[i] = *reinterpret_cast<const u32x4*>(src);
        hi[i] = *reinterpret_cast<const u32x4*>(src + HD / 2);
    }
    const int pos = a.positions[tok], slot = a.slots[tok];
    const bool on_table = pos >= 0 && pos < a.max_pos;
    const bool stored = on_table && slot >= 0 && (slot >> a.s.page_log2) < a.s.num_pages;
    float c[2][8], s[2][8];
    if (a.cos && h0 < a.nh + a.s.kvh) {
        const int64_t at = (int64_t)(on_table ? pos : 0) * HD + d0;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const floatx4 cw = *reinterpret_cast<const floatx4*>(a.cos + at + half * (HD / 2) + e);
                const floatx4 sw = *reinterpret_cast<const floatx4*>(a.sin + at + half * (HD / 2) + e);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[half][e + i] = cw[i];
                    s[half][e + i] = sw[i];
                }
            }
    }
    const int in_page = slot & (a.s.page() - 1);
    uint16_t* page = a.cache + (int64_t)(stored ? slot >> a.s.page_log2 : 0) * a.s.kvh * a.s.block() + (int64_t)in_page * HD + d0;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = h0 + i;
        if (h >= heads) break;
        if (a.cos && h < a.nh + a.s.kvh) {
            float x[8], y[8], u[8], v[8];
            load8<BF16>(&lo[i], x);
            load8<BF16>(&hi[i], y);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                u[e] = x[e] * c[0][e] - y[e] * s[0][e];
                v[e] = y[e] * c[1][e] + x[e] * s[1][e];
            }
            store8<BF16>(&lo[i], u);
            store8<BF16>(&hi[i], v);
        }
        uint16_t* dst;
        if (h < a.nh) {
            if (!on_table) lo[i] = hi[i] = u32x4{0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu};   // NaN in both types
            dst = reinterpret_cast<uint16_t*>(a.q) + ((int64_t)tok * a.nh + h) * HD + d0;
        } else {
            if (!stored) break;
            const int g = h - a.nh < a.s.kvh ? h - a.nh : h - a.nh - a.s.kvh;
            dst = page + g * a.s.block() + (h - a.nh < a.s.kvh ? 0 : HD << a.s.page_log2);
        }
        *reinterpret_cast<u32x4*>(dst) = lo[i];
        *reinterpret_cast<u32x4*>(dst + HD / 2) = hi[i];
    }
}

}  // namespace

hipError_t launch_kv16_append(const Kv16AppendArgs& a, bool bf16, hipStream_t stream) {
    const uint32_t parts = (uint32_t)((a.nh + 2 * a.s.kvh + kHeads - 1) / kHeads);
    const int64_t threads = (int64_t)a.tokens * parts * (a.s.hd / 16);
    auto kernel = a.s.hd == 64 ? (bf16 ? awq_kv16_append_kernel<64, true> : awq_kv16_append_kernel<64, false>)
                               : (bf16 ? awq_kv16_append_kernel<128, true> : awq_kv16_append_kernel<128, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, a, parts,
                       div_inverse(parts));
    return hipGetLastError();
}

}  // namespace awq
