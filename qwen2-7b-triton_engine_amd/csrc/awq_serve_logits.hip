// A step's logits under penalties, biases and a grammar's mask, and their
// greedy token (include/awq_serving.h: awq_serve_logits):
//   x / or * repetition, x - frequency n, x - presence, x + bias, -inf; argmax.
//
// What bounds it: memory -- the logits in and out once; for one row the
// latency of two launches.  The penalties need to know how often each token
// occurs in the row's history.  A counter per token in memory would be a
// second tensor as large as the logits, to be kept from step to step; here a
// workgroup has a stretch of the vocabulary, counts the history's tokens that
// fall into it in LDS (integers: the order of the atomics does not matter)
// and then passes over its logits.  The history is read once per stretch, out
// of the caches.  Of a token biased twice the last entry counts, found the
// same way as the largest index.
#include "awq_serving.h"

#pragma clang fp contract(off)   // each step rounds as the same step in torch does

namespace awq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kInPrompt = 0x80000000u;   // of a counter; the rest counts generated tokens
constexpr uint32_t kMinusInf = 0x007FFFFFu;   // order_of(-inf)

// Unsigned integers in the order of the floats: -inf lowest, NaN highest, the
// two zeros equal.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (!(x == x)) return 0xFFFFFFFFu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) {
        const uint64_t o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}

// VEC neighbouring logits as fp32, and back rounded once (x becomes what was stored).
template <int DT, int VEC>
__device__ __forceinline__ void load_logits(const void* p, int64_t at, float (&x)[VEC]) {
    if constexpr (DT == AWQ_SERVE_FP32) {
        const float* f = reinterpret_cast<const float*>(p) + at;
        if constexpr (VEC == 8) {
            const floatx4 lo = reinterpret_cast<const floatx4*>(f)[0], hi = reinterpret_cast<const floatx4*>(f)[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = lo[e];
                x[4 + e] = hi[e];
            }
        } else {
            x[0] = f[0];
        }
    } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + at;
        if constexpr (VEC == 8)
            load8<DT == AWQ_SERVE_BF16>(h, x);
        else if constexpr (DT == AWQ_SERVE_BF16)
            x[0] = __builtin_bit_cast(float, (uint32_t)h[0] << 16);
        else
            x[0] = (float)__builtin_bit_cast(half_t, h[0]);
    }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_logits(void* p, int64_t at, float (&x)[VEC]) {
    if constexpr (DT == AWQ_SERVE_FP32) {
        float* f = reinterpret_cast<float*>(p) + at;
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            if constexpr (VEC == 8) *reinterpret_cast<floatx4*>(f + e) = floatx4{x[e], x[e + 1], x[e + 2], x[e + 3]};
            else f[0] = x[0];
        }
    } else {
        constexpr bool BF16 = DT == AWQ_SERVE_BF16;
        uint16_t* h = reinterpret_cast<uint16_t*>(p) + at;
        uint16_t r[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            r[e] = to16<BF16>(x[e]);
            if constexpr (BF16) x[e] = __builtin_bit_cast(float, (uint32_t)r[e] << 16);
            else x[e] = (float)__builtin_bit_cast(half_t, r[e]);
        }
        if constexpr (VEC == 8) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (uint32_t)r[2 * e] | ((uint32_t)r[2 * e + 1] << 16);
            *reinterpret_cast<u32x4*>(h) = w;
        } else {
            h[0] = r[0];
        }
    }
}

// One workgroup: the stretch blockIdx.x of CH logits of row blockIdx.y.
template <int DT, int VEC, int CH>
__global__ __launch_bounds__(kThreads) void awq_logits_kernel(LogitsArgs a) {
    __shared__ __align__(16) uint32_t seen[CH];     // the history's tokens
    __shared__ __align__(16) uint32_t entry[CH];    // 1 + the last bias entry, 0: none
    __shared__ uint64_t best[kWaves];
    const int row = blockIdx.y, tid = threadIdx.x;
    const int v0 = blockIdx.x * CH;
    const int n = a.vocab - v0 < CH ? a.vocab - v0 : CH;
    const bool history = a.tokens != nullptr, biases = a.bias_start != nullptr;
    if (history || biases) {
        for (int i = 4 * tid; i < CH; i += 4 * kThreads) {
            *reinterpret_cast<u32x4*>(&seen[i]) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(&entry[i]) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
    }
    if (history) {
        const int64_t len = a.lengths[row] < a.width ? a.lengths[row] : a.width;
        const int64_t prompt = a.prompt_lens[row];
        auto count = [&](int64_t i, int64_t token) {
            const uint64_t at = (uint64_t)(token - v0);
            if (at >= (uint64_t)n) return;
            if (i < prompt) atomicOr(&seen[at], kInPrompt);
            else atomicAdd(&seen[at], 1u);
        };
        auto scan = [&](auto* text) {
            text += (int64_t)row * a.width;
            int64_t i = tid;
            for (; i + 7 * kThreads < len; i += 8 * kThreads) {   // eight loads in flight
                int64_t t[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) t[u] = text[i + u * kThreads];
#pragma unroll
                for (int u = 0; u < 8; ++u) count(i + u * kThreads, t[u]);
            }
            for (; i < len; i += kThreads) count(i, text[i]);
        };
        if (a.token_bytes == 8) scan(reinterpret_cast<const int64_t*>(a.tokens));
        else scan(reinterpret_cast<const int32_t*>(a.tokens));
    }
    if (biases) {
        int lo = a.bias_start[row], hi = a.bias_start[row + 1];
        lo = lo < 0 ? 0 : lo;
        hi = hi < a.bias_count ? hi : a.bias_count;
        for (int i = lo + tid; i < hi; i += kThreads) {
            const uint32_t at = (uint32_t)(a.bias_tokens[i] - v0);
            if (at < (uint32_t)n) atomicMax(&entry[at], (uint32_t)i + 1u);
        }
    }
    if (history || biases) __syncthreads();

    const float rep = history && a.repetition ? a.repetition[row] : 1.0f;
    const float pres = history && a.presence ? a.presence[row] : 0.0f;
    const float freq = history && a.frequency ? a.frequency[row] : 0.0f;
    const uint32_t* mask = a.mask ? a.mask + (int64_t)row * ((a.vocab + 31) / 32) + v0 / 32 : nullptr;
    uint64_t top = 0;
    for (int i = VEC * tid; i < n; i += VEC * kThreads) {
        float x[VEC];
        load_logits<DT, VEC>(a.logits, (int64_t)row * a.ld + v0 + i, x);
        uint32_t allowed = 0xFFu;
        if (mask) allowed = mask[i / 32] >> (i % 32);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (history) {
                const uint32_t s = seen[i + e];
                if (s) x[e] = x[e] > 0.0f ? x[e] / rep : x[e] * rep;
                const uint32_t times = s & ~kInPrompt;
                if (times) {
                    x[e] = x[e] - freq * (float)times;
                    x[e] = x[e] - pres;
                }
            }
            if (biases) {
                const uint32_t b = entry[i + e];
                if (b) x[e] = x[e] + a.bias_values[b - 1];
            }
            if (!((allowed >> e) & 1u)) x[e] = -INFINITY;
        }
        store_logits<DT, VEC>(a.out, (int64_t)row * a.vocab + v0 + i, x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const uint64_t key = ((uint64_t)order_of(x[e]) << 32) | (0xFFFFFFFFu - (uint32_t)(v0 + i + e));
            top = key > top ? key : top;
        }
    }
    top = wave_max64(top);
    if ((tid & 63) == 0) best[tid >> 6] = top;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = best[w] > top ? best[w] : top;
        a.keys[(int64_t)row * gridDim.x + blockIdx.x] = top;
    }
}

// The row's largest key: one wave a row.
__global__ __launch_bounds__(64) void awq_greedy_kernel(const uint64_t* __restrict__ keys, int64_t* __restrict__ next,
                                                        int stretches) {
    uint64_t top = 0;
    for (int i = threadIdx.x; i < stretches; i += 64) {
        const uint64_t k = keys[(int64_t)blockIdx.x * stretches + i];
        top = k > top ? k : top;
    }
    top = wave_max64(top);
    if (threadIdx.x == 0)
        next[blockIdx.x] = (uint32_t)(top >> 32) == kMinusInf ? -1 : (int64_t)(0xFFFFFFFFu - (uint32_t)top);
}

constexpr int kShort = 2048, kLong = 8192;

// Short stretches where long ones would leave CUs without work.
int stretch_of(int rows, int vocab) { return (int64_t)rows * ((vocab + kLong - 1) / kLong) >= 512 ? kLong : kShort; }

template <int DT, int VEC>
void launch(const LogitsArgs& a, hipStream_t stream) {
    const int ch = stretch_of(a.rows, a.vocab);
    const dim3 grid((a.vocab + ch - 1) / ch, a.rows);
    if (ch == kLong) hipLaunchKernelGGL((awq_logits_kernel<DT, VEC, kLong>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((awq_logits_kernel<DT, VEC, kShort>), grid, dim3(kThreads), 0, stream, a);
}

}  // namespace

size_t logits_workspace(int rows, int vocab) {
    const int ch = stretch_of(rows, vocab);
    return (size_t)rows * ((vocab + ch - 1) / ch) * sizeof(uint64_t);
}

hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
    // Eight logits a thread where every row starts on 16 bytes and ends on a whole piece.
    const int bytes = a.dtype == AWQ_SERVE_FP32 ? 4 : 2;
    const bool wide = a.vocab % 8 == 0 && (a.ld * bytes) % 16 == 0 &&
                      ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0;
    using std::integral_constant;
    auto typed = [&](auto dt) {
        if (wide) launch<dt(), 8>(a, stream);
        else launch<dt(), 1>(a, stream);
    };
    if (a.dtype == AWQ_SERVE_FP16) typed(integral_constant<int, AWQ_SERVE_FP16>{});
    else if (a.dtype == AWQ_SERVE_BF16) typed(integral_constant<int, AWQ_SERVE_BF16>{});
    else typed(integral_constant<int, AWQ_SERVE_FP32>{});
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int ch = stretch_of(a.rows, a.vocab);
    hipLaunchKernelGGL(awq_greedy_kernel, dim3(a.rows), dim3(64), 0, stream, a.keys, a.next, (a.vocab + ch - 1) / ch);
    return hipGetLastError();
}

}  // namespace awq
