// Internal interface of the serving operators (include/awq_serving.h): argument
// blocks of their launchers, and what their kernels share.
#pragma once

#include "../../include/awq_serving.h"
#include "awq_kernels.h"
#include "awq_serve_items.h"

namespace awq {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct PageStepArgs {
    const int32_t* state;       // [requests + 1]: lengths, free pages
    const int32_t* tokens;      // [requests]: new tokens (step), tokens kept (release)
    int32_t* tables;            // [requests, width]
    int32_t* free_pages;        // [capacity]
    int32_t *new_state, *query_start, *slots, *positions, *failed;
    int requests, total, width, capacity, page_log2;
};
hipError_t launch_page_step(const PageStepArgs& a, hipStream_t stream);
hipError_t launch_page_release(const PageStepArgs& a, hipStream_t stream);

// One layer's cache: where the parts of a block begin (include/awq_serving.h).
struct Kv4Shape {
    int kvh, hd, groups, page_log2, num_pages;
    __host__ __device__ int page() const { return 1 << page_log2; }
    __host__ __device__ int k_bytes() const { return page() * hd / 2; }               // K codes; V codes alike
    __host__ __device__ int scale_bytes() const { return page() * groups * 4; }       // K scales; V scales alike
    __host__ __device__ int block() const { return 2 * (k_bytes() + scale_bytes()); }
};

struct Kv4AppendArgs {
    const void* qkv;            // [tokens, ...], ld elements from row to row
    int64_t ld;
    uint8_t* cache;
    const int32_t *slots, *positions;
    const float *cos, *sin;     // [max_pos, hd], or null: no rotation
    void* q;                    // [tokens, nh * hd]
    int tokens, nh, max_pos;
    Kv4Shape s;
};
hipError_t launch_kv4_append(const Kv4AppendArgs& a, bool bf16, hipStream_t stream);
struct Kv4GatherArgs {
    const uint8_t* cache;
    const int32_t* slots;
    void *k, *v;                // [tokens, kvh, hd]
    int tokens;
    Kv4Shape s;
};
hipError_t launch_kv4_gather(const Kv4GatherArgs& a, bool bf16, hipStream_t stream);

struct Kv4AttnArgs {
    const void* q;              // [total, nh * hd], ld elements from row to row
    int64_t ld;
    const uint8_t* cache;
    const int32_t *tables, *seq_lens, *query_start;
    float* part;
    void* out;                  // [total, nh * hd]
    int requests, total, max_query, nh, width;
    float scale;
    Kv4Shape s;
    // set by the launch
    float* tile_part;
    i32x4* records;             // [total]: what the combining launch has to know of a row
    int limit;                  // columns up to which a request is the decode kernel's
    int decode_target, tile_target;   // items of one kv head that the kernels aim at
    // what awq_serve_walk.h asks for
    static constexpr int kTileCols = 64, kExtra = 2;
    static constexpr bool kEven = false, combine = true;
    __device__ __forceinline__ int group() const { return nh / s.kvh; }
    __device__ __forceinline__ int least_steps(int steps, bool) const { return steps; }
    __device__ __forceinline__ int first_key(int, int) const { return 0; }
    __device__ __forceinline__ bool sees_none(int, int, int rows, int len, int i) const { return (int64_t)len - rows + i < 0; }
    __device__ __forceinline__ float factor(const float*) const { return scale * 1.4426950408889634f; }
};
size_t kv4_attn_workspace(int requests, int total, int max_query, int nh, int kvh, int hd);
hipError_t launch_kv4_attention(const Kv4AttnArgs& a, bool bf16, hipStream_t stream);

// One layer's 16-bit cache: [num_pages][kvh][K, V][page][hd].
struct Kv16Shape {
    int kvh, hd, page_log2, num_pages;
    __host__ __device__ int page() const { return 1 << page_log2; }
    __host__ __device__ int64_t block() const { return (int64_t)(hd * 2) << page_log2; }   // elements of a page and head
};

struct Kv16AppendArgs {
    const void* qkv;            // [tokens, ...], ld elements from row to row
    int64_t ld;
    uint16_t* cache;
    const int32_t *slots, *positions;
    const float *cos, *sin;     // [max_pos, hd], or null: no rotation
    void* q;                    // [tokens, nh * hd]
    int tokens, nh, max_pos;
    Kv16Shape s;
};
hipError_t launch_kv16_append(const Kv16AppendArgs& a, bool bf16, hipStream_t stream);

struct Kv16AttnArgs {
    const void* q;              // [total, nh * hd], ld elements from row to row
    int64_t ld;
    const uint16_t* cache;
    const int32_t *tables, *seq_lens, *query_start;
    const float* slopes;        // [nh], or null
    const int32_t* prefix;      // [requests], or null
    const int32_t* first;       // [total], or null
    float* part;
    void* out;                  // [total, nh * hd]
    int requests, total, max_query, nh, width;
    int window;                 // tokens that a row sees back from itself, 0: all
    float scale, softcap;       // softcap 0: none
    Kv16Shape s;
    // set by the launch
    float* tile_part;
    i32x4* records;             // [total]
    int limit, decode_target, tile_target;
    bool combine;               // whether the joining launch follows
    int heads_each;             // nh / kvh
    uint32_t heads_inv, kvh_inv;   // div_inverse of it and of kvh
    // what awq_serve_walk.h asks for
    static constexpr int kTileCols = kTile16Cols, kExtra = 4;   // maximum, sum, unit, nothing
    static constexpr bool kEven = true;
    __device__ __forceinline__ int group() const { return heads_each; }
    __device__ __forceinline__ int least_steps(int steps, bool prompts) const { return least_tile_steps(steps, prompts); }
    __device__ __forceinline__ int first_key(int rows, int len) const {
        return first_token(window, rows, len, walked_tokens(width, s.page_log2, len));
    }
    // Tokens lo .. hi - 1 that the i-th row of request b sees; none: 0 and 0.  Of a table
    // that is too short its first missing token is the last one: it gives NaN.
    struct Range {
        int lo, hi;
    };
    // of request b's prefix p and the row's first token f; 0: none
    __device__ __forceinline__ Range seen(int rows, int len, int i, int p, int f) const {
        const int64_t pos = (int64_t)len - rows + i;
        int64_t lo = window ? pos - window + 1 : 0, hi = pos + 1;
        hi = hi > p ? hi : p < len ? p : len;
        lo = lo > f ? lo : f;
        lo = lo > 0 ? lo : 0;
        if (pos < 0 || lo >= hi) return Range{0, 0};
        const int n = walked_tokens(width, s.page_log2, len);
        return Range{lo < n ? (int)lo : n - 1, hi < n ? (int)hi : n};
    }
    __device__ __forceinline__ Range range(int b, int row0, int rows, int len, int i) const {
        return seen(rows, len, i, prefix ? prefix[b] : 0, first ? first[row0 + i] : 0);
    }
    __device__ __forceinline__ bool sees_none(int b, int row0, int rows, int len, int i) const {
        return range(b, row0, rows, len, i).hi == 0;
    }
    // Scores that are capped or carry a bias are scaled before, plain ones after their differences.
    __host__ __device__ bool shaped() const { return softcap > 0.0f || slopes; }
    __device__ __forceinline__ float factor(const float* extra) const { return extra[2]; }
};
bool kv16_attn_fits(int requests, int total, int max_query, int nh, int kvh);
size_t kv16_attn_workspace(int requests, int total, int max_query, int nh, int kvh, int hd);
hipError_t launch_kv16_attention(const Kv16AttnArgs& a, bool bf16, hipStream_t stream);

struct LogprobsArgs {
    const void* hidden;         // [tokens, k], ld elements from row to row
    int64_t ld;
    const void* weight;         // [vocab, k]
    const void* targets;        // [tokens] of token_bytes
    int token_bytes;
    float *logprobs, *lse;      // [tokens]
    float* part;                // [vocabulary tiles][tokens] (maximum, sum)
    int tokens, vocab, k;
    float* chosen;              // set by the launch: [tokens], the targets' logits
};
size_t logprobs_workspace(int tokens, int vocab);
hipError_t launch_logprobs(LogprobsArgs a, bool bf16, hipStream_t stream);

struct LogitsArgs {
    const void* logits;
    int64_t ld;
    void* out;
    int64_t* next;
    int rows, vocab, dtype;
    const void* tokens;
    int token_bytes;
    int64_t width;
    const int32_t *lengths, *prompt_lens;
    const float *repetition, *presence, *frequency;
    const int32_t *bias_start, *bias_tokens;
    const float* bias_values;
    int bias_count;
    const uint32_t* mask;
    uint64_t* keys;
};
size_t logits_workspace(int rows, int vocab);
hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream);

// ---- what the kernels share ---------------------------------------------------

// Activations of 16 bits: eight of them as fp32 and back, rounded to nearest.
template <bool BF16>
__device__ __forceinline__ void load8(const void* p, float (&x)[8]) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (BF16) {
            x[2 * e] = __builtin_bit_cast(float, w[e] << 16);
            x[2 * e + 1] = __builtin_bit_cast(float, w[e] & 0xFFFF0000u);
        } else {
            const half2_t h = as_h2(w[e]);
            x[2 * e] = (float)h.x;
            x[2 * e + 1] = (float)h.y;
        }
    }
}
template <bool BF16>
__device__ __forceinline__ uint16_t to16(float x) {
    if constexpr (BF16)
        return __builtin_bit_cast(uint16_t, (__bf16)x);
    else
        return __builtin_bit_cast(uint16_t, (half_t)x);
}
template <bool BF16>
__device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)to16<BF16>(x[2 * e]) | ((uint32_t)to16<BF16>(x[2 * e + 1]) << 16);
    *reinterpret_cast<u32x4*>(p) = w;
}

constexpr float kLog2e = 1.4426950408889634f;

// A product of 16-bit operands of either type, eight in four words.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
template <bool BF16>
__device__ __forceinline__ floatx4 mfma16(u32x4 a, u32x4 b, floatx4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return mfma16x16x32(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c);
}

// A barrier for LDS alone: loads from memory stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Sum of a 64-bit value over the lanes below this one and itself.
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t o = __shfl_up(v, d);
        if ((int)(threadIdx.x & 63) >= d) v += o;
    }
    return v;
}
// The same of 32-bit values by DPP steps, without the LDS pipe.
__device__ __forceinline__ int wave_scan32(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);    // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast:31 into rows 2 and 3
    return v;
}
// Largest of a value of 0 or more over the lanes below this one and itself.
__device__ __forceinline__ int wave_scan_max(int v) {
    auto step = [&](int o) { v = o > v ? o : v; };
    step(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true));
    step(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true));
    step(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true));
    step(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true));
    step(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    return v;
}
// The sums over a workgroup of WAVES waves, and the whole in `all`.  Values of at
// most 2^24 + 1: a wave's sum fits 32 bits, the waves' are added in 64.
// lds: free for use before the call and after it.
template <int WAVES>
__device__ __forceinline__ int64_t block_scan(int v, int (&lds)[WAVES], int64_t& all) {
    const int wave = threadIdx.x >> 6;
    const int upto = wave_scan32(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) lds[wave] = upto;
    __syncthreads();
    all = 0;
    int64_t before = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += lds[w];
        all += lds[w];
    }
    return before + upto;
}

}  // namespace awq
