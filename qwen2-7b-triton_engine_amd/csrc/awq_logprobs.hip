// Log-probabilities of given tokens under the output projection, without its logits
// (include/awq_serving.h: awq_serve_logprobs): with z = W h,
//   lse = log sum exp z,  logprob = z[target] - lse.
//
// A matrix product whose result stays in registers: a workgroup has a tile of
// vocabulary rows times tokens, and leaves of each of its tokens the largest logit and the sum of
// exponentials over the tile's rows -- 8 bytes for BV logits -- and the target's logit where it is
// in the tile.  A second launch joins the tiles.  Z = W H^T puts a token in each MFMA
// column, so that its maximum and sum are a lane's own up to two cross-lane steps.
//
// What bounds it: with up to 128 tokens the weight's bytes, read once.  152064 rows of 3584 are 1.09 GB: one token 182 us
// (6.0 TB/s), 64 209, 128 245.  With many the product: 2047 tokens are 2.23 TFLOP in 1927 us, 1158 TFLOP/s (1881 to 1951 from
// run to run), where a library's product of the same sizes takes 1799 (1240) and leaves 622 MB of logits; power holds the clock at
// 1.8 GHz.  Between them, at 256 tokens, both: 349 us.
#include "awq_serving.h"

namespace awq {
namespace {

constexpr int kBK = 64;                // k of a step: rows of 128 bytes in LDS

// WV x WT waves of FV x FT blocks of 16 vocabulary rows x 16 tokens, S stages of LDS.
template <int WV, int WT, int FV, int FT, int S, int PER_CU>
struct LpTile {
    static constexpr int kWV = WV, kWT = WT, kFV = FV, kFT = FT, kS = S, kPerCu = PER_CU;
    static constexpr int kWaves = WV * WT, kThreads = 64 * kWaves;
    static constexpr int BV = 16 * FV * WV, BT = 16 * FT * WT;
    static constexpr int kWBlocks = BV / 8, kHBlocks = BT / 8;     // of 8 rows: one load of a wave each
    static constexpr int kWLoads = (kWBlocks + kWaves - 1) / kWaves, kHLoads = (kHBlocks + kWaves - 1) / kWaves;
    static constexpr int kLoads = kWLoads + kHLoads;
    static constexpr int kStage = (BV + BT) * kBK * 2;
};

// The 16-byte chunks of a row are swizzled: 16 rows' same chunk, an operand's read, touches every bank once.
__device__ __forceinline__ constexpr int lp_swizzle(int row) { return row >> 1 & 7; }

struct LpGrid {
    int v_tiles, t_tiles, group, per_xcd;   // token tiles side by side in a group
};

template <class L, bool BF16>
__global__ __launch_bounds__(L::kThreads, L::kPerCu * L::kWaves / 4) void awq_logprobs_kernel(LogprobsArgs a, LpGrid grid) {
    constexpr int FV = L::kFV, FT = L::kFT, S = L::kS;
    static_assert((S - 1) * L::kLoads <= 63, "vmcnt holds 6 bits");
    static_assert(L::BT <= L::kThreads, "a thread joins a token's waves");
    __shared__ __align__(1024) unsigned char smem[S * L::kStage];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroups go round the XCDs: each gets a range of vocabulary tiles of its own, all token
    // tiles of a group beside each other, so that a weight passes one XCD's cache once.
    const int seq = (int)(blockIdx.x & 7) * grid.per_xcd + (int)(blockIdx.x >> 3);
    if (seq >= grid.v_tiles * grid.t_tiles) return;
    const int group = seq / (grid.v_tiles * grid.group), in = seq - group * (grid.v_tiles * grid.group);
    const int left = grid.t_tiles - group * grid.group, width = left < grid.group ? left : grid.group;
    const int vt = in / width, tt = group * grid.group + in % width;
    const int v0 = vt * L::BV, t0 = tt * L::BT;

    const int rows_v = min(L::BV, a.vocab - v0), rows_t = min(L::BT, a.tokens - t0);
    const u32x4 rw = raw_rsrc(reinterpret_cast<const uint16_t*>(a.weight) + (int64_t)v0 * a.k, (uint32_t)rows_v * a.k * 2);
    const u32x4 rh = raw_rsrc(reinterpret_cast<const uint16_t*>(a.hidden) + (int64_t)t0 * a.ld,
                              (uint32_t)(((int64_t)(rows_t - 1) * a.ld + a.k) * 2));
    // A load brings 8 rows of 128 bytes; block b of them has rows 8 b ..
    uint32_t w_ofs[L::kWLoads], h_ofs[L::kHLoads];
    const uint32_t lds0 = lds_addr(smem);
    const int lr = lane >> 3, slot = lane & 7;
#pragma unroll
    for (int i = 0; i < L::kWLoads; ++i) {
        const int row = 8 * min(wave * L::kWLoads + i, L::kWBlocks - 1) + lr;
        w_ofs[i] = (uint32_t)row * a.k * 2 + (slot ^ lp_swizzle(row)) * 16;
    }
#pragma unroll
    for (int i = 0; i < L::kHLoads; ++i) {
        const int row = 8 * min(wave * L::kHLoads + i, L::kHBlocks - 1) + lr;
        h_ofs[i] = (uint32_t)row * (uint32_t)a.ld * 2 + (slot ^ lp_swizzle(row)) * 16;
    }
    auto issue = [&](int step) {
        const uint32_t to = lds0 + step % S * L::kStage, k = step * (kBK * 2);
#pragma unroll
        for (int i = 0; i < L::kWLoads; ++i)
            buffer_load_lds_x4(rw, w_ofs[i], k, to + 1024 * min(wave * L::kWLoads + i, L::kWBlocks - 1));
#pragma unroll
        for (int i = 0; i < L::kHLoads; ++i)
            buffer_load_lds_x4(rh, h_ofs[i], k, to + L::BV * 128 + 1024 * min(wave * L::kHLoads + i, L::kHBlocks - 1));
    };
    const int steps = a.k / kBK;
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
        if (i < steps) issue(i);

    const int col = lane & 15, kb = lane >> 4, wv = wave % L::kWV, wt = wave / L::kWV;
    const uint32_t frag = col * 128 + ((kb ^ lp_swizzle(col)) * 16);   // of k-half 1: ^ 64
    floatx4 acc[FV][FT];
#pragma unroll
    for (int v = 0; v < FV; ++v)
#pragma unroll
        for (int t = 0; t < FT; ++t) acc[v][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int step = 0; step < steps; ++step) {
        const int after = steps - 1 - step;              // steps whose loads may stay in flight: S - 2, fewer at the end
        wait_batches<L::kLoads, S - 2>(after < S - 2 ? after : S - 2);
        lds_barrier();                                   // the step is there, and the stage before it read by all
        if (step + S - 1 < steps) issue(step + S - 1);
        const unsigned char* st = smem + step % S * L::kStage;
        u32x4 w[2][FV], x[2][FT];
        auto read = [&](int h) {
#pragma unroll
            for (int v = 0; v < FV; ++v) w[h][v] = *reinterpret_cast<const u32x4*>(st + (wv * FV + v) * 2048 + (frag ^ (64 * h)));
#pragma unroll
            for (int t = 0; t < FT; ++t)
                x[h][t] = *reinterpret_cast<const u32x4*>(st + L::BV * 128 + (wt * FT + t) * 2048 + (frag ^ (64 * h)));
        };
        // The second half's operands are read under the first's products, and a wave that has all of its operands goes
        // before one that is reading: 2047 tokens 1951 us for 2019 without, 512 535 for 561 (in turn, in one run).
        read(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h == 0) read(1);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int t = 0; t < FT; ++t)
#pragma unroll
                for (int v = 0; v < FV; ++v) acc[v][t] = mfma16<BF16>(w[h][v], x[h][t], acc[v][t]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Lane (col, kb) holds of token col of block t the rows 16 v + 4 kb + r.
    const int row0 = v0 + 16 * FV * wv + 4 * kb;
    float2* part = reinterpret_cast<float2*>(a.part);
    __syncthreads();                                     // the stages are read: their room holds the waves' sums
    float2* red = reinterpret_cast<float2*>(smem);       // [WV][BT]
#pragma unroll
    for (int t = 0; t < FT; ++t) {
        const int token = t0 + 16 * (wt * FT + t) + col;
        int64_t want = -1;
        if (token < a.tokens) want = a.token_bytes == 8 ? reinterpret_cast<const int64_t*>(a.targets)[token]
                                                        : reinterpret_cast<const int32_t*>(a.targets)[token];
        const int64_t at = want - row0;
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < FV; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (at == 16 * v + r && want < a.vocab) a.chosen[token] = acc[v][t][r];
                if (row0 + 16 * v + r >= a.vocab) acc[v][t][r] = -INFINITY;
                m = fmaxf(m, acc[v][t][r]);
            }
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const float ref = m == -INFINITY ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < FV; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[v][t][r] - ref) * kLog2e);
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (kb == 0) red[wv * L::BT + 16 * (wt * FT + t) + col] = float2{m, s};
    }
    __syncthreads();
    if (threadIdx.x < L::BT && t0 + (int)threadIdx.x < a.tokens) {
        float m = -INFINITY, s = 0.0f;
#pragma unroll
        for (int w = 0; w < L::kWV; ++w) m = fmaxf(m, red[w * L::BT + threadIdx.x].x);
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < L::kWV; ++w) {
            const float2 p = red[w * L::BT + threadIdx.x];
            s += p.y * __builtin_amdgcn_exp2f((p.x - ref) * kLog2e);
        }
        part[(int64_t)vt * a.tokens + t0 + threadIdx.x] = float2{m, s};
    }
}

// Joins a token's tiles: TOKENS tokens a workgroup, 256 / TOKENS threads each.
template <int TOKENS>
__global__ __launch_bounds__(256) void awq_logprobs_join_kernel(LogprobsArgs a, int v_tiles) {
    constexpr int kEach = 256 / TOKENS;
    __shared__ float2 red[256];
    const int tok = threadIdx.x % TOKENS, token = blockIdx.x * TOKENS + tok;
    const float2* part = reinterpret_cast<const float2*>(a.part);
    float m = -INFINITY, s = 0.0f;
    auto add = [&](float2 p) {
        const float top = fmaxf(m, p.x), ref = top == -INFINITY ? 0.0f : top;
        s = s * __builtin_amdgcn_exp2f((m - ref) * kLog2e) + p.y * __builtin_amdgcn_exp2f((p.x - ref) * kLog2e);
        m = top;
    };
    if (token < a.tokens) {
        for (int v = threadIdx.x / TOKENS; v < v_tiles; v += 4 * kEach) {
            float2 p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                p[i] = v + i * kEach < v_tiles ? part[(int64_t)(v + i * kEach) * a.tokens + token] : float2{-INFINITY, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) add(p[i]);
        }
    }
    red[threadIdx.x] = float2{m, s};
    for (int n = kEach / 2; n > 0; n /= 2) {
        __syncthreads();
        if ((int)threadIdx.x < n * TOKENS) {
            add(red[threadIdx.x + n * TOKENS]);
            red[threadIdx.x] = float2{m, s};
        }
    }
    if ((int)threadIdx.x >= TOKENS || token >= a.tokens) return;
    const int64_t want = a.token_bytes == 8 ? reinterpret_cast<const int64_t*>(a.targets)[token]
                                            : reinterpret_cast<const int32_t*>(a.targets)[token];
    // An infinite logit is all of the sum (its tile's sum is NaN: infinity less itself).
    const float log_s = m == INFINITY ? 0.0f : logf(s);
    a.lse[token] = m == -INFINITY && s == 0.0f ? m : m + log_s;
    // (z - m) - log s: closer than z - lse where the target is likely
    a.logprobs[token] = want < 0 ? 0.0f : want >= a.vocab ? NAN : (a.chosen[token] - m) - log_s;
}

using Wide = LpTile<4, 2, 4, 8, 2, 1>;       // 256 rows x 256 tokens
using Tall = LpTile<4, 2, 4, 5, 3, 1>;       // 256 x 160
using Middle = LpTile<4, 2, 4, 4, 3, 1>;     // 256 x 128
using Narrow = LpTile<4, 1, 2, 4, 3, 2>;     // 128 x 64
using Thin = LpTile<4, 1, 2, 1, 4, 2>;       // 128 x 16

// Many tokens: the tiles that take least, by what one of them costs where there are several (Middle 126 us for 152064 rows
// of 3584, Tall 150, Wide 218).  Wide / Tall / Middle there, in one run, us: 160 tokens 334 / 268 / 327,
// 256 345 / 389 / 350, 300 484 / 398 / 438, 384 505 / 520 / 462, 512 530 / 682 / 621, 2047 1906 / 2252 / 2185.
// The vocabulary does not enter: from 50000 rows on the choice is within 4 % of the best; with fewer the tiles leave CUs
// empty, and smaller ones would take less.  Wide / Middle / Narrow / Thin, 256 tokens: 1000 rows 85 / 54 / 32 / 21, 4000
// 88 / 56 / 34 / 32, 16000 87 / 57 / 45 / 99, 50000 116 / 135 / 175 / 362.
template <class F>
auto with_tile(int tokens, F f) {
    if (tokens <= 16) return f(Thin{});
    if (tokens <= 64) return f(Narrow{});
    auto cost = [&](int width, int64_t each) { return (int64_t)((tokens + (int64_t)width - 1) / width) * each; };
    const int64_t wide = cost(Wide::BT, 218), tall = cost(Tall::BT, 150), middle = cost(Middle::BT, 126);
    if (middle < wide && middle < tall) return f(Middle{});
    return tall < wide ? f(Tall{}) : f(Wide{});
}

}  // namespace

// The tiles' maxima and sums, then the targets' logits; 0: too many tiles for a launch.
size_t logprobs_workspace(int tokens, int vocab) {
    return with_tile(tokens, [&](auto tile) {
        using L = decltype(tile);
        const size_t v_tiles = ((size_t)vocab + L::BV - 1) / L::BV, t_tiles = ((size_t)tokens + L::BT - 1) / L::BT;
        if ((v_tiles * t_tiles + 8) * L::kThreads >= (size_t)1 << 32) return (size_t)0;
        return (v_tiles * 2 + 1) * (size_t)tokens * sizeof(float);
    });
}

hipError_t launch_logprobs(LogprobsArgs a, bool bf16, hipStream_t stream) {
    return with_tile(a.tokens, [&](auto tile) {
        using L = decltype(tile);
        LpGrid g;
        g.v_tiles = (a.vocab + L::BV - 1) / L::BV;
        g.t_tiles = (a.tokens + L::BT - 1) / L::BT;
        g.group = g.t_tiles < 8 ? g.t_tiles : 8;
        g.per_xcd = (g.v_tiles * g.t_tiles + 7) / 8;
        a.chosen = a.part + 2 * (size_t)g.v_tiles * a.tokens;
        auto kernel = bf16 ? awq_logprobs_kernel<L, true> : awq_logprobs_kernel<L, false>;
        hipLaunchKernelGGL(kernel, dim3(8 * (unsigned)g.per_xcd), dim3(L::kThreads), 0, stream, a, g);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (a.tokens <= 64)
            hipLaunchKernelGGL(awq_logprobs_join_kernel<1>, dim3((unsigned)a.tokens), dim3(256), 0, stream, a, g.v_tiles);
        else
            hipLaunchKernelGGL(awq_logprobs_join_kernel<8>, dim3((unsigned)(a.tokens + 7) / 8), dim3(256), 0, stream, a, g.v_tiles);
        return hipGetLastError();
    });
}

}  // namespace awq
