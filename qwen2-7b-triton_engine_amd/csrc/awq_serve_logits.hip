// A step's logits under penalties, biases and a grammar's mask, and their
// greedy token (include/awq_serving.h: awq_serve_logits):
//   x / or * repetition, x - frequency n, x - presence, x + bias, -inf; argmax.
//
// What it cannot do without is the logits in and out once.  The penalties need to know how often each token
// occurs in the row's history.  A counter per token in memory would be a
// second tensor as large as the logits, to be kept from step to step; here a
// workgroup has a stretch of the vocabulary, counts the history's tokens that
// fall into it in LDS (integers: the order of the atomics does not matter) and
// lists each at its first count.  Of a token biased twice the last entry counts, found
// as the largest index.  The listed tokens, few among many, get their new
// logits by one thread each; then the stretch passes through, its logits loaded
// before the counting began.  The history is read once per stretch, out of the caches.
// What bounds it, both launches in a graph, us: one row of 152064 logits 7.6, the latency of
// two launches; sixty-four with histories of 4096 26.5 (41 MB in and out: 6.6 at the memory's
// rate), some 500 vector instructions a wave, half of them the history's tokens, which each of the
// row's 38 stretches looks at, and chains of LDS latencies between barriers.  With a
// counter and a bias entry read for every logit 45.  A fourth workgroup on a CU (4032 logits
// each) changed nothing; a wave that gathers its tokens of the stretch before it counts them was
// faster where histories are long (eight rows of 50257 with 16000: 13.5 -> 11.6) and slower for
// one row (7.0 -> 7.2).
#include "awq_serving.h"

#pragma clang fp contract(off)   // each step rounds as the same step in torch does

namespace awq {
namespace {

constexpr int kThreads = 512;
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

// Eight neighbouring logits as they lie in memory, at any alignment of theirs
// (vocabularies are odd, rows are strided), and as fp32.
template <int DT>
struct Piece {
    static constexpr int kWords = DT == AWQ_SERVE_FP32 ? 8 : 4;
    static constexpr int kBytes = DT == AWQ_SERVE_FP32 ? 4 : 2;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const uint8_t* p) { __builtin_memcpy(w, p, sizeof(w)); }
    __device__ __forceinline__ void store(uint8_t* p) const { __builtin_memcpy(p, w, sizeof(w)); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (DT == AWQ_SERVE_FP32) x[e] = __builtin_bit_cast(float, w[e]);
            else if constexpr (DT == AWQ_SERVE_BF16) x[e] = __builtin_bit_cast(float, e % 2 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
            else x[e] = (float)as_h2(w[e / 2])[e % 2];
        }
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {   // values that the type holds
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (DT == AWQ_SERVE_FP32) w[i] = __builtin_bit_cast(uint32_t, x[i]);
            else if constexpr (DT == AWQ_SERVE_BF16)
                w[i] = __builtin_bit_cast(uint32_t, x[2 * i]) >> 16 | (__builtin_bit_cast(uint32_t, x[2 * i + 1]) & 0xFFFF0000u);
            else w[i] = as_u32(half2_t{(half_t)x[2 * i], (half_t)x[2 * i + 1]});
        }
    }
};
template <int DT>
__device__ __forceinline__ float load_one(const uint8_t* p) {
    if constexpr (DT == AWQ_SERVE_FP32) return *reinterpret_cast<const float*>(p);
    const uint16_t h = *reinterpret_cast<const uint16_t*>(p);
    if constexpr (DT == AWQ_SERVE_BF16) return __builtin_bit_cast(float, (uint32_t)h << 16);
    return (float)__builtin_bit_cast(half_t, h);
}
template <int DT>
__device__ __forceinline__ void store_one(uint8_t* p, float x) {
    if constexpr (DT == AWQ_SERVE_FP32) *reinterpret_cast<float*>(p) = x;
    else *reinterpret_cast<uint16_t*>(p) = to16<DT == AWQ_SERVE_BF16>(x);
}
// x rounded to the type.
template <int DT>
__device__ __forceinline__ float rounded(float x) {
    if constexpr (DT == AWQ_SERVE_FP32) return x;
    const uint16_t h = to16<DT == AWQ_SERVE_BF16>(x);
    if constexpr (DT == AWQ_SERVE_BF16) return __builtin_bit_cast(float, (uint32_t)h << 16);
    return (float)__builtin_bit_cast(half_t, h);
}

// Logits of a workgroup, eight a thread.  Shorter stretches read the history more often, longer
// ones leave a CU one workgroup (LDS).  1024 / 4096 / 8192 logits, us: one row of 152064 6.97 /
// 6.93 / 8.05, eight with histories of 4096 12.8 / 8.9 / 9.6, sixty-four 60 / 26 / 37; eight
// of 50257 with 16000 12.4 / 13.6 / 15.2.
constexpr int kStretch = 8 * kThreads;
int stretches(int vocab) { return (vocab + kStretch - 1) / kStretch; }

// One workgroup: the stretch blockIdx.x of row blockIdx.y.
template <int DT>
__global__ __launch_bounds__(kThreads) void awq_logits_kernel(LogitsArgs a) {
    constexpr int kBytes = Piece<DT>::kBytes;
    __shared__ __align__(16) uint32_t word[kStretch];   // counts of the history's tokens, then the new logits
    __shared__ __align__(16) uint32_t entry[kStretch];  // 1 + the last bias entry, 0: none
    __shared__ uint32_t touched[kStretch / 32];     // bit of each token with a new logit
    __shared__ uint16_t list[kStretch];             // those tokens
    __shared__ int listed;
    __shared__ uint64_t best[kWaves];
    const int row = blockIdx.y, tid = threadIdx.x;
    const int v0 = blockIdx.x * kStretch;
    const int n = a.vocab - v0 < kStretch ? a.vocab - v0 : kStretch;
    const uint8_t* in = reinterpret_cast<const uint8_t*>(a.logits) + ((int64_t)row * a.ld + v0) * kBytes;
    uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + ((int64_t)row * a.vocab + v0) * kBytes;
    const int first = 8 * tid;                      // of the thread's eight
    Piece<DT> x;
    if (first + 8 <= n) x.load(in + (int64_t)first * kBytes);
    const uint32_t* mask = a.mask ? a.mask + (int64_t)row * ((a.vocab + 31) / 32) + v0 / 32 : nullptr;

    // Everything that hangs on nothing else is loaded at once: a workgroup is a
    // chain of latencies, the row's numbers, its history, the listed logits.
    const bool history = a.tokens != nullptr, biases = a.bias_start != nullptr;
    int64_t len = history ? a.lengths[row] : 0;
    const int64_t prompt = history ? a.prompt_lens[row] : 0;
    const int bias_from = biases ? a.bias_start[row] : 0, bias_to = biases ? a.bias_start[row + 1] : 0;
    const float rep = history && a.repetition ? a.repetition[row] : 1.0f;
    const float pres = history && a.presence ? a.presence[row] : 0.0f;
    const float freq = history && a.frequency ? a.frequency[row] : 0.0f;
    len = len < a.width ? len : a.width;
    // Both ends within the entries, and unsigned: with a thread's or a stride's number on top a
    // start near 2^31 must not come out below the end.
    const uint32_t bias_hi = bias_to < 0 ? 0 : bias_to < a.bias_count ? bias_to : a.bias_count;
    const uint32_t bias_lo = bias_from < 0 ? 0 : (uint32_t)bias_from < bias_hi ? bias_from : bias_hi;
    constexpr int kFlight = 8;                      // tokens of a thread in flight
    int64_t t[kFlight];
    const bool wide_ids = a.token_bytes == 8;
    auto fetch = [&](int64_t i0) {
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int64_t i = i0 + u * kThreads, at = (int64_t)row * a.width + i;
            t[u] = i >= len ? -1 : wide_ids ? reinterpret_cast<const int64_t*>(a.tokens)[at]
                                            : (int64_t)reinterpret_cast<const int32_t*>(a.tokens)[at];
        }
    };
    if (len > 0) fetch(tid);
    const int first_bias = bias_lo + tid < bias_hi ? a.bias_tokens[bias_lo + tid] : -1;

    for (int i = 4 * tid; i < kStretch; i += 4 * kThreads) {
        *reinterpret_cast<u32x4*>(&word[i]) = u32x4{0, 0, 0, 0};
        *reinterpret_cast<u32x4*>(&entry[i]) = u32x4{0, 0, 0, 0};
    }
    for (int i = tid; i < kStretch / 32; i += kThreads) touched[i] = 0;
    if (tid == 0) listed = 0;
    __syncthreads();
    for (int64_t i0 = tid; i0 < len; i0 += kFlight * kThreads) {
        if (i0 != tid) fetch(i0);
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const uint64_t at = (uint64_t)(t[u] - v0);
            if (at >= (uint64_t)n) continue;
            const uint32_t before = i0 + u * kThreads < prompt ? atomicOr(&word[at], kInPrompt) : atomicAdd(&word[at], 1u);
            if (before == 0) list[atomicAdd(&listed, 1)] = (uint16_t)at;
        }
    }
    __syncthreads();
    if (bias_lo < bias_hi) {
        for (uint32_t i = bias_lo + tid; i < bias_hi; i += kThreads) {
            const uint32_t at = (uint32_t)((i == bias_lo + tid ? first_bias : a.bias_tokens[i]) - v0);
            if (at >= (uint32_t)n) continue;
            if (atomicMax(&entry[at], i + 1u) == 0 && word[at] == 0) list[atomicAdd(&listed, 1)] = (uint16_t)at;
        }
        __syncthreads();
    }

    for (int i = tid; i < listed; i += kThreads) {
        const int at = list[i];
        const uint32_t s = word[at], b = entry[at], times = s & ~kInPrompt;
        float y = load_one<DT>(in + (int64_t)at * kBytes);
        if (s) y = y > 0.0f ? y / rep : y * rep;
        if (times) {
            y = y - freq * (float)times;
            y = y - pres;
        }
        if (b) y = y + a.bias_values[b - 1];
        word[at] = __builtin_bit_cast(uint32_t, rounded<DT>(y));
        atomicOr(&touched[at / 32], 1u << (at % 32));
    }
    // In place what follows overwrites what is read above (and only that).
    __syncthreads();

    uint64_t top_key = 0;
    auto see = [&](float v, int at) {               // by key: ties, zeros and NaN in order
        const uint64_t key = ((uint64_t)order_of(v) << 32) | (0xFFFFFFFFu - (uint32_t)(v0 + at));
        top_key = key > top_key ? key : top_key;
    };
    if (first < n) {
        const uint32_t changed = touched[first / 32] >> (first % 32) & 0xFFu;
        const uint32_t allowed = mask ? mask[first / 32] >> (first % 32) : 0xFFu;
        if (first + 8 > n) {                        // the vocabulary's last piece, one by one
            for (int at = first; at < n; ++at) {
                const int e = at - first;
                float y = changed >> e & 1 ? __builtin_bit_cast(float, word[at]) : load_one<DT>(in + (int64_t)at * kBytes);
                if (!(allowed >> e & 1)) y = -INFINITY;
                store_one<DT>(out + (int64_t)at * kBytes, y);
                see(y, at);
            }
        } else {
            float y[8];
            x.get(y);
            if (changed) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (changed >> e & 1) y[e] = __builtin_bit_cast(float, word[first + e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] = allowed >> e & 1 ? y[e] : -INFINITY;
                see(y[e], first + e);
            }
            x.set(y);
            x.store(out + (int64_t)first * kBytes);
        }
    }
    top_key = wave_max64(top_key);
    if ((tid & 63) == 0) best[tid >> 6] = top_key;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top_key = best[w] > top_key ? best[w] : top_key;
        a.keys[(int64_t)row * gridDim.x + blockIdx.x] = top_key;
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

}  // namespace

size_t logits_workspace(int rows, int vocab) { return (size_t)rows * stretches(vocab) * sizeof(uint64_t); }

hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
    auto kernel = a.dtype == AWQ_SERVE_FP16   ? awq_logits_kernel<AWQ_SERVE_FP16>
                  : a.dtype == AWQ_SERVE_BF16 ? awq_logits_kernel<AWQ_SERVE_BF16>
                                              : awq_logits_kernel<AWQ_SERVE_FP32>;
    hipLaunchKernelGGL(kernel, dim3(stretches(a.vocab), a.rows), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(awq_greedy_kernel, dim3(a.rows), dim3(64), 0, stream, a.keys, a.next, stretches(a.vocab));
    return hipGetLastError();
}

}  // namespace awq
