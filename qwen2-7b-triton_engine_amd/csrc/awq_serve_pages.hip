// Block tables, slots and positions of a serving step, from the requests'
// lengths (include/awq_serving.h: awq_serve_page_step, awq_serve_page_release).
//
// With len and new the lengths before the step and the tokens it adds, P tokens
// a page and c free pages F[0 .. c - 1]:
//   start[b] = new[0] + .. + new[b - 1]                           first row
//   need[b]  = ceil((len + new) / P) - ceil(len / P)              pages to take
//   taken[b] = need[0] + .. + need[b - 1],   k-th page = F[c - 1 - k]
// and token p of a request lies in slot page(p / P) * P + p % P.
//
// What bounds it: latency -- a few kilobytes pass.  One launch, no atomics in memory and
// nothing between workgroups: each has the two prefix sums of all requests to
// itself (16 requests a thread at most) and keeps them in LDS, then places one row
// a thread by binary search.  The torch form is some forty launches.  Measured: 64
// requests of a token each 2.9 us, 16384 rows of 256 requests 6.0 (9.7 with
// 64-bit wave sums), 4096 requests of a token each 16; a release of every eighth request of 64 or
// 256 3.1 us, of 4096 26 (every workgroup adds all of them up).
#include "awq_serving.h"

namespace awq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMax = AWQ_SERVE_MAX_REQUESTS;

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_log2) {
    return (tokens + (1 << page_log2) - 1) >> page_log2;
}

__global__ __launch_bounds__(kThreads) void awq_page_step_kernel(PageStepArgs a) {
    __shared__ int sums[kWaves];
    __shared__ int start[kMax + 1];    // first row, at most a.total
    __shared__ int taken[kMax];        // pages taken before it; -1: refused
    __shared__ int all_taken;
    const int B = a.requests, tid = threadIdx.x;
    const int count_in = a.state[B];
    const int64_t count = count_in < 0 ? 0 : count_in < a.capacity ? count_in : a.capacity;
    const int64_t room = (int64_t)a.width << a.page_log2;
    if (tid == 0) all_taken = 0;

    int64_t rows = 0, used = 0;        // of the requests before this stretch of kThreads
    for (int b0 = 0; b0 < B; b0 += kThreads) {
        const int b = b0 + tid;
        const int64_t len = b < B ? a.state[b] : 0;
        const int64_t add = b < B ? a.tokens[b] : 0;
        int64_t all;
        // What passes `total` or the free pages is refused however much it is: one more stands for it.
        const int add_rows = add < 0 ? 0 : add <= a.total ? (int)add : a.total + 1;
        const int64_t end = rows + block_scan<kWaves>(add_rows, sums, all);
        rows += all;
        const bool fits = add >= 0 && len >= 0 && end <= a.total && len + add <= room;
        const int64_t pages = fits ? pages_of(len + add, a.page_log2) - pages_of(len, a.page_log2) : 0;
        const int need = (int)(pages <= count ? pages : count + 1);
        const int64_t upto = used + block_scan<kWaves>(need, sums, all);
        used += all;
        const bool served = fits && (need == 0 || upto <= count);
        if (b < B) {
            const int64_t first = end - add_rows;
            start[b] = (int)(first < a.total ? first : a.total);
            const int64_t before = upto - need;   // past int only where none are needed
            taken[b] = served ? (int)(before < INT32_MAX ? before : INT32_MAX) : -1;
            // Sums grow along the requests: the last served that takes pages has the largest.
            if (served && need > 0) atomicMax(&all_taken, (int)upto);
            if (blockIdx.x == 0) {
                a.new_state[b] = (int)(served ? len + add : len);
                a.failed[b] = served ? 0 : 1;
                a.query_start[b] = start[b];
            }
        }
    }
    const int rows_in = (int)(rows < a.total ? rows : a.total);
    if (tid == 0) start[B] = rows_in;
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        a.query_start[B] = rows_in;
        a.new_state[B] = (int)(count - all_taken);
    }

    const int64_t row = (int64_t)blockIdx.x * kThreads + tid;
    if (row >= a.total) return;
    int slot = -1, pos = -1;
    if (row < rows_in) {
        int lo = 0, hi = B;            // start[lo] <= row < start[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= row) lo = mid;
            else hi = mid;
        }
        const int before = taken[lo];
        if (before >= 0) {
            const int len = a.state[lo];
            pos = len + (int)(row - start[lo]);
            const int index = pos >> a.page_log2, held = (int)pages_of(len, a.page_log2);
            const int offset = pos & ((1 << a.page_log2) - 1);
            int32_t* entry = a.tables + (int64_t)lo * a.width + index;
            int page;
            if (index >= held) {       // one of the step's: its first token writes the table
                page = a.free_pages[count - 1 - (before + index - held)];
                if (offset == 0) *entry = page;
            } else {
                page = *entry;
            }
            slot = page >= 0 && page < (1 << (31 - a.page_log2)) ? (page << a.page_log2) + offset : -1;
        }
    }
    a.slots[row] = slot;
    a.positions[row] = pos;
}

// One workgroup per request: the sums again, then its own pages.
__global__ __launch_bounds__(kThreads) void awq_page_release_kernel(PageStepArgs a) {
    __shared__ int sums[kWaves];
    __shared__ int64_t mine[2];        // this request's pages: first place, number
    const int B = a.requests, tid = threadIdx.x, me = blockIdx.x;
    const int count_in = a.state[B];
    const int64_t count = count_in < 0 ? 0 : count_in < a.capacity ? count_in : a.capacity;
    int64_t before = 0;
    for (int b0 = 0; b0 < B; b0 += kThreads) {
        const int b = b0 + tid;
        const int64_t room = (int64_t)a.width << a.page_log2;
        int64_t len = b < B ? a.state[b] : 0;
        len = len < 0 ? 0 : len < room ? len : room;
        int64_t keep = b < B ? a.tokens[b] : 0;
        keep = keep < 0 ? 0 : keep < len ? keep : len;
        const int64_t all_give = pages_of(len, a.page_log2) - pages_of(keep, a.page_log2);
        const int give = (int)(all_give <= a.capacity ? all_give : a.capacity);   // no request holds more
        int64_t all;
        const int64_t upto = before + block_scan<kWaves>(give, sums, all);
        before += all;
        if (b == me) {
            mine[0] = count + upto - give;
            mine[1] = give;
            a.new_state[b] = (int)keep;
        }
    }
    __syncthreads();
    if (me == 0 && tid == 0) a.new_state[B] = (int)(count + before < a.capacity ? count + before : a.capacity);
    const int64_t room = (int64_t)a.width << a.page_log2;
    int64_t len = a.state[me];
    len = len < 0 ? 0 : len < room ? len : room;
    const int64_t first = pages_of(len, a.page_log2) - mine[1];
    for (int64_t i = tid; i < mine[1]; i += kThreads)
        if (mine[0] + i < a.capacity) a.free_pages[mine[0] + i] = a.tables[(int64_t)me * a.width + first + i];
}

}  // namespace

hipError_t launch_page_step(const PageStepArgs& a, hipStream_t stream) {
    const int grid = a.total > 0 ? (a.total + kThreads - 1) / kThreads : 1;
    hipLaunchKernelGGL(awq_page_step_kernel, dim3(grid), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_page_release(const PageStepArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(awq_page_release_kernel, dim3(a.requests), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace awq
