// C ABI of the serving operators: checks and launches.  Declarations:
// include/awq_serving.h.
#include <limits.h>
#include <math.h>

#include "awq_serving.h"

using namespace awq;

namespace {

constexpr int64_t kIndexLimit = INT_MAX;
constexpr int64_t kMostRows = 1 << 24, kMostPages = 1 << 24;   // of a step: 32-bit sums over a wave

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int log2_page(int64_t page_size) {
    for (int l = 4; l <= 8; ++l)
        if (page_size == (int64_t)1 << l) return l;
    return -1;
}

int done(hipError_t e) { return e == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH; }

// Tables of `requests` rows: slots stay 32-bit integers, lengths below 2^30 (sums of
// a length and a stretch of tokens do not overflow).
int check_pages(int64_t requests, int64_t width, int64_t num_pages, int64_t page_size) {
    if (requests <= 0 || width <= 0 || num_pages <= 0) return AWQ_ERR_BAD_DIMS;
    if (log2_page(page_size) < 0) return AWQ_ERR_PATH;
    if (requests > AWQ_SERVE_MAX_REQUESTS || width > (1 << 30) / page_size || num_pages > kIndexLimit / page_size)
        return AWQ_ERR_TOO_LARGE;
    return AWQ_OK;
}

int check_cache(int64_t kvh, int64_t hd, int64_t num_pages, int64_t page_size, int64_t group_size, int32_t dtype,
                Kv4Shape* s) {
    if (kvh <= 0 || num_pages <= 0) return AWQ_ERR_BAD_DIMS;
    if ((hd != 64 && hd != 128) || log2_page(page_size) < 0 || (dtype != AWQ_SERVE_FP16 && dtype != AWQ_SERVE_BF16))
        return AWQ_ERR_PATH;
    if ((group_size != 32 && group_size != 64 && group_size != 128) || group_size > hd) return AWQ_ERR_GROUP_SIZE;
    if (kvh > 4096 || num_pages > kIndexLimit / page_size) return AWQ_ERR_TOO_LARGE;
    *s = Kv4Shape{(int)kvh, (int)hd, (int)(hd / group_size), log2_page(page_size), (int)num_pages};
    return AWQ_OK;
}

int check_cache16(int64_t kvh, int64_t hd, int64_t num_pages, int64_t page_size, int32_t dtype, Kv16Shape* s) {
    if (kvh <= 0 || num_pages <= 0) return AWQ_ERR_BAD_DIMS;
    if ((hd != 64 && hd != 128) || log2_page(page_size) < 0 || (dtype != AWQ_SERVE_FP16 && dtype != AWQ_SERVE_BF16))
        return AWQ_ERR_PATH;
    if (kvh > 4096 || num_pages > kIndexLimit / page_size) return AWQ_ERR_TOO_LARGE;
    *s = Kv16Shape{(int)kvh, (int)hd, log2_page(page_size), (int)num_pages};
    return AWQ_OK;
}

int check_step(const PageStepArgs& a, int64_t requests, int64_t width, int64_t capacity, int64_t page_size) {
    const int st = check_pages(requests, width, capacity, page_size);
    if (st != AWQ_OK) return st;
    if (capacity > kMostPages) return AWQ_ERR_TOO_LARGE;
    if (!a.state || !a.tokens || !a.tables || !a.free_pages || !a.new_state) return AWQ_ERR_NULL_POINTER;
    if (!aligned(a.state, 4) || !aligned(a.tokens, 4) || !aligned(a.tables, 4) || !aligned(a.free_pages, 4) ||
        !aligned(a.new_state, 4))
        return AWQ_ERR_MISALIGNED;
    return AWQ_OK;
}

}  // namespace

extern "C" {

int awq_serve_page_step(const int32_t* state, const int32_t* new_tokens, int32_t* block_tables,
                        const int32_t* free_pages, int32_t* new_state, int32_t* query_start, int32_t* slots,
                        int32_t* positions, int32_t* failed, int64_t requests, int64_t total, int64_t table_width,
                        int64_t capacity, int64_t page_size, void* stream) {
    PageStepArgs a = {};
    a.state = state;
    a.tokens = new_tokens;
    a.tables = block_tables;
    a.free_pages = const_cast<int32_t*>(free_pages);
    a.new_state = new_state;
    a.query_start = query_start;
    a.slots = slots;
    a.positions = positions;
    a.failed = failed;
    const int st = check_step(a, requests, table_width, capacity, page_size);
    if (st != AWQ_OK) return st;
    if (total < 0) return AWQ_ERR_BAD_DIMS;
    if (total > kMostRows) return AWQ_ERR_TOO_LARGE;
    if (!query_start || !failed || (total > 0 && (!slots || !positions))) return AWQ_ERR_NULL_POINTER;
    if (!aligned(query_start, 4) || !aligned(failed, 4) || !aligned(slots, 4) || !aligned(positions, 4))
        return AWQ_ERR_MISALIGNED;
    a.requests = (int)requests;
    a.total = (int)total;
    a.width = (int)table_width;
    a.capacity = (int)capacity;
    a.page_log2 = log2_page(page_size);
    return done(launch_page_step(a, static_cast<hipStream_t>(stream)));
}

int awq_serve_page_release(const int32_t* state, const int32_t* keep, const int32_t* block_tables,
                           int32_t* free_pages, int32_t* new_state, int64_t requests, int64_t table_width,
                           int64_t capacity, int64_t page_size, void* stream) {
    PageStepArgs a = {};
    a.state = state;
    a.tokens = keep;
    a.tables = const_cast<int32_t*>(block_tables);
    a.free_pages = free_pages;
    a.new_state = new_state;
    const int st = check_step(a, requests, table_width, capacity, page_size);
    if (st != AWQ_OK) return st;
    a.requests = (int)requests;
    a.width = (int)table_width;
    a.capacity = (int)capacity;
    a.page_log2 = log2_page(page_size);
    return done(launch_page_release(a, static_cast<hipStream_t>(stream)));
}

int awq_serve_kv4_append(const void* qkv, int64_t qkv_stride, void* cache, const int32_t* slots,
                         const int32_t* positions, const void* cos, const void* sin, void* q_out, int64_t tokens,
                         int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_pages,
                         int64_t page_size, int64_t group_size, int64_t max_pos, int32_t dtype, void* stream) {
    Kv4AppendArgs a;
    const int st = check_cache(num_kv_heads, head_dim, num_pages, page_size, group_size, dtype, &a.s);
    if (st != AWQ_OK) return st;
    if (tokens < 0 || num_heads <= 0 || max_pos <= 0 || qkv_stride < (num_heads + 2 * num_kv_heads) * head_dim)
        return AWQ_ERR_BAD_DIMS;
    if (num_heads > 4096 || max_pos > kIndexLimit || tokens > kIndexLimit / ((num_heads + num_kv_heads) * 16))
        return AWQ_ERR_TOO_LARGE;
    if (tokens == 0) return AWQ_OK;
    if (!qkv || !cache || !slots || !positions || !q_out || !cos != !sin) return AWQ_ERR_NULL_POINTER;
    if (!aligned(qkv, 16) || qkv_stride % 8 != 0 || !aligned(cache, 16) || !aligned(slots, 4) ||
        !aligned(positions, 4) || !aligned(cos, 16) || !aligned(sin, 16) || !aligned(q_out, 16))
        return AWQ_ERR_MISALIGNED;
    a.qkv = qkv;
    a.ld = qkv_stride;
    a.cache = static_cast<uint8_t*>(cache);
    a.slots = slots;
    a.positions = positions;
    a.cos = static_cast<const float*>(cos);
    a.sin = static_cast<const float*>(sin);
    a.q = q_out;
    a.tokens = (int)tokens;
    a.nh = (int)num_heads;
    a.max_pos = (int)max_pos;
    return done(launch_kv4_append(a, dtype == AWQ_SERVE_BF16, static_cast<hipStream_t>(stream)));
}

int awq_serve_kv4_gather(const void* cache, const int32_t* slots, void* k, void* v, int64_t tokens,
                         int64_t num_kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
                         int64_t group_size, int32_t dtype, void* stream) {
    Kv4GatherArgs a;
    const int st = check_cache(num_kv_heads, head_dim, num_pages, page_size, group_size, dtype, &a.s);
    if (st != AWQ_OK) return st;
    if (tokens < 0) return AWQ_ERR_BAD_DIMS;
    if (tokens > kIndexLimit / (num_kv_heads * 16)) return AWQ_ERR_TOO_LARGE;
    if (tokens == 0) return AWQ_OK;
    if (!cache || !slots || !k || !v) return AWQ_ERR_NULL_POINTER;
    if (!aligned(cache, 16) || !aligned(slots, 4) || !aligned(k, 16) || !aligned(v, 16)) return AWQ_ERR_MISALIGNED;
    a.cache = static_cast<const uint8_t*>(cache);
    a.slots = slots;
    a.k = k;
    a.v = v;
    a.tokens = (int)tokens;
    return done(launch_kv4_gather(a, dtype == AWQ_SERVE_BF16, static_cast<hipStream_t>(stream)));
}

// Sizes that attention's grid, workspace and checks go by.
static int check_attention(int64_t requests, int64_t total, int64_t max_query, int64_t nh, int64_t kvh, int64_t hd,
                           int64_t width, int64_t page_size) {
    const int st = check_pages(requests, width, 1, page_size);
    if (st != AWQ_OK) return st;
    if (total < 0 || max_query <= 0 || kvh <= 0 || nh <= 0 || nh % kvh != 0) return AWQ_ERR_BAD_DIMS;
    if ((hd != 64 && hd != 128) || nh / kvh > AWQ_SERVE_MAX_GROUP) return AWQ_ERR_PATH;
    if (nh > 4096 || max_query > kIndexLimit / 64 || total > kIndexLimit / 4096) return AWQ_ERR_TOO_LARGE;
    return AWQ_OK;
}

size_t awq_serve_kv4_attention_workspace(int64_t requests, int64_t total, int64_t max_query, int64_t num_heads,
                                         int64_t num_kv_heads, int64_t head_dim, int64_t table_width,
                                         int64_t page_size) {
    if (check_attention(requests, total, max_query, num_heads, num_kv_heads, head_dim, table_width, page_size) != AWQ_OK)
        return 0;
    return kv4_attn_workspace((int)requests, (int)total, (int)max_query, (int)num_heads, (int)num_kv_heads, (int)head_dim);
}

int awq_serve_kv4_attention(const void* q, int64_t q_stride, const void* cache, const int32_t* block_tables,
                            const int32_t* seq_lens, const int32_t* query_start, void* out, int64_t requests,
                            int64_t total, int64_t max_query, int64_t num_heads, int64_t num_kv_heads,
                            int64_t head_dim, int64_t table_width, int64_t num_pages, int64_t page_size,
                            int64_t group_size, float scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                            void* stream) {
    Kv4AttnArgs a = {};
    int st = check_cache(num_kv_heads, head_dim, num_pages, page_size, group_size, dtype, &a.s);
    if (st != AWQ_OK) return st;
    st = check_attention(requests, total, max_query, num_heads, num_kv_heads, head_dim, table_width, page_size);
    if (st != AWQ_OK) return st;
    if (q_stride < num_heads * head_dim || !(scale > 0.0f) || !(scale < HUGE_VALF)) return AWQ_ERR_BAD_DIMS;
    if (total == 0) return AWQ_OK;
    if (!q || !cache || !block_tables || !seq_lens || !query_start || !out) return AWQ_ERR_NULL_POINTER;
    if (!aligned(q, 16) || q_stride % 8 != 0 || !aligned(cache, 16) || !aligned(block_tables, 4) ||
        !aligned(seq_lens, 4) || !aligned(query_start, 4) || !aligned(out, 16) || !aligned(workspace, 16))
        return AWQ_ERR_MISALIGNED;
    if (!workspace || workspace_bytes < kv4_attn_workspace((int)requests, (int)total, (int)max_query, (int)num_heads,
                                                           (int)num_kv_heads, (int)head_dim))
        return AWQ_ERR_WORKSPACE;
    a.q = q;
    a.ld = q_stride;
    a.cache = static_cast<const uint8_t*>(cache);
    a.tables = block_tables;
    a.seq_lens = seq_lens;
    a.query_start = query_start;
    a.part = static_cast<float*>(workspace);
    a.out = out;
    a.requests = (int)requests;
    a.total = (int)total;
    a.max_query = (int)max_query;
    a.nh = (int)num_heads;
    a.width = (int)table_width;
    a.scale = scale;
    return done(launch_kv4_attention(a, dtype == AWQ_SERVE_BF16, static_cast<hipStream_t>(stream)));
}

int awq_serve_kv16_append(const void* qkv, int64_t qkv_stride, void* cache, const int32_t* slots,
                          const int32_t* positions, const void* cos, const void* sin, void* q_out, int64_t tokens,
                          int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_pages,
                          int64_t page_size, int64_t max_pos, int32_t dtype, void* stream) {
    Kv16AppendArgs a;
    const int st = check_cache16(num_kv_heads, head_dim, num_pages, page_size, dtype, &a.s);
    if (st != AWQ_OK) return st;
    if (tokens < 0 || num_heads <= 0 || max_pos <= 0 || qkv_stride < (num_heads + 2 * num_kv_heads) * head_dim)
        return AWQ_ERR_BAD_DIMS;
    if (num_heads > 4096 || max_pos > kIndexLimit || tokens > kIndexLimit / ((num_heads + 2 * num_kv_heads) * 16))
        return AWQ_ERR_TOO_LARGE;
    if (tokens == 0) return AWQ_OK;
    if (!qkv || !cache || !slots || !positions || !q_out || !cos != !sin) return AWQ_ERR_NULL_POINTER;
    if (!aligned(qkv, 16) || qkv_stride % 8 != 0 || !aligned(cache, 16) || !aligned(slots, 4) ||
        !aligned(positions, 4) || !aligned(cos, 16) || !aligned(sin, 16) || !aligned(q_out, 16))
        return AWQ_ERR_MISALIGNED;
    a.qkv = qkv;
    a.ld = qkv_stride;
    a.cache = static_cast<uint16_t*>(cache);
    a.slots = slots;
    a.positions = positions;
    a.cos = static_cast<const float*>(cos);
    a.sin = static_cast<const float*>(sin);
    a.q = q_out;
    a.tokens = (int)tokens;
    a.nh = (int)num_heads;
    a.max_pos = (int)max_pos;
    return done(launch_kv16_append(a, dtype == AWQ_SERVE_BF16, static_cast<hipStream_t>(stream)));
}

size_t awq_serve_kv16_attention_workspace(int64_t requests, int64_t total, int64_t max_query, int64_t num_heads,
                                          int64_t num_kv_heads, int64_t head_dim, int64_t table_width,
                                          int64_t page_size) {
    if (check_attention(requests, total, max_query, num_heads, num_kv_heads, head_dim, table_width, page_size) != AWQ_OK)
        return 0;
    if (!kv16_attn_fits((int)requests, (int)total, (int)max_query, (int)num_heads, (int)num_kv_heads)) return 0;
    return kv16_attn_workspace((int)requests, (int)total, (int)max_query, (int)num_heads, (int)num_kv_heads, (int)head_dim);
}

int awq_serve_kv16_attention(const void* q, int64_t q_stride, const void* cache, const int32_t* block_tables,
                             const int32_t* seq_lens, const int32_t* query_start, const float* slopes,
                             const int32_t* prefix, const int32_t* first, void* out, int64_t requests, int64_t total,
                             int64_t max_query, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                             int64_t table_width, int64_t num_pages, int64_t page_size, int64_t window, float scale,
                             float softcap, int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
    Kv16AttnArgs a = {};
    int st = check_cache16(num_kv_heads, head_dim, num_pages, page_size, dtype, &a.s);
    if (st != AWQ_OK) return st;
    st = check_attention(requests, total, max_query, num_heads, num_kv_heads, head_dim, table_width, page_size);
    if (st != AWQ_OK) return st;
    if (q_stride < num_heads * head_dim || !(scale > 0.0f) || !(scale < HUGE_VALF) || window < 0 ||
        !(softcap == 0.0f || (softcap >= 0x1p-100f && softcap < HUGE_VALF)))
        return AWQ_ERR_BAD_DIMS;
    if (!kv16_attn_fits((int)requests, (int)total, (int)max_query, (int)num_heads, (int)num_kv_heads)) return AWQ_ERR_TOO_LARGE;
    if (total == 0) return AWQ_OK;
    if (!q || !cache || !block_tables || !seq_lens || !query_start || !out) return AWQ_ERR_NULL_POINTER;
    if (!aligned(q, 16) || q_stride % 8 != 0 || !aligned(cache, 16) || !aligned(block_tables, 4) ||
        !aligned(seq_lens, 4) || !aligned(query_start, 4) || !aligned(slopes, 4) || !aligned(prefix, 4) ||
        !aligned(first, 4) || !aligned(out, 16) || !aligned(workspace, 16))
        return AWQ_ERR_MISALIGNED;
    if (!workspace || workspace_bytes < kv16_attn_workspace((int)requests, (int)total, (int)max_query, (int)num_heads,
                                                            (int)num_kv_heads, (int)head_dim))
        return AWQ_ERR_WORKSPACE;
    a.q = q;
    a.ld = q_stride;
    a.cache = static_cast<const uint16_t*>(cache);
    a.tables = block_tables;
    a.seq_lens = seq_lens;
    a.query_start = query_start;
    a.slopes = slopes;
    a.prefix = prefix;
    a.first = first;
    a.part = static_cast<float*>(workspace);
    a.out = out;
    a.requests = (int)requests;
    a.total = (int)total;
    a.max_query = (int)max_query;
    a.nh = (int)num_heads;
    a.width = (int)table_width;
    a.window = window < kIndexLimit ? (int)window : 0;   // more than any position: none
    a.scale = scale;
    a.softcap = softcap;
    return done(launch_kv16_attention(a, dtype == AWQ_SERVE_BF16, static_cast<hipStream_t>(stream)));
}

size_t awq_serve_logprobs_workspace(int64_t tokens, int64_t vocab) {
    if (tokens <= 0 || vocab <= 0 || tokens > kMostRows || vocab > kMostRows) return 0;
    return logprobs_workspace((int)tokens, (int)vocab);
}

int awq_serve_logprobs(const void* hidden, int64_t hidden_stride, const void* weight, const void* targets,
                       int32_t target_bytes, float* logprobs, float* lse, int64_t tokens, int64_t vocab, int64_t k,
                       int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (tokens < 0 || vocab <= 0 || k <= 0 || k % 64 != 0 || hidden_stride < k) return AWQ_ERR_BAD_DIMS;
    if ((dtype != AWQ_SERVE_FP16 && dtype != AWQ_SERVE_BF16) || (target_bytes != 4 && target_bytes != 8)) return AWQ_ERR_PATH;
    if (tokens > kMostRows || vocab > kMostRows || k > (1 << 20) || hidden_stride > (1 << 22)) return AWQ_ERR_TOO_LARGE;
    if (tokens == 0) return AWQ_OK;
    const size_t need = logprobs_workspace((int)tokens, (int)vocab);
    if (need == 0) return AWQ_ERR_TOO_LARGE;
    if (!hidden || !weight || !targets || !logprobs || !lse) return AWQ_ERR_NULL_POINTER;
    if (!aligned(hidden, 16) || hidden_stride % 8 != 0 || !aligned(weight, 16) || !aligned(targets, target_bytes) ||
        !aligned(logprobs, 4) || !aligned(lse, 4) || !aligned(workspace, 8))
        return AWQ_ERR_MISALIGNED;
    if (!workspace || workspace_bytes < need) return AWQ_ERR_WORKSPACE;
    LogprobsArgs a = {};
    a.hidden = hidden;
    a.ld = hidden_stride;
    a.weight = weight;
    a.targets = targets;
    a.token_bytes = target_bytes;
    a.logprobs = logprobs;
    a.lse = lse;
    a.part = static_cast<float*>(workspace);
    a.tokens = (int)tokens;
    a.vocab = (int)vocab;
    a.k = (int)k;
    return done(launch_logprobs(a, dtype == AWQ_SERVE_BF16, static_cast<hipStream_t>(stream)));
}

size_t awq_serve_logits_workspace(int64_t rows, int64_t vocab) {
    if (rows <= 0 || vocab <= 0 || rows > 65535 || vocab > kIndexLimit / 2) return 0;
    return logits_workspace((int)rows, (int)vocab);
}

int awq_serve_logits(const void* logits, int64_t row_stride, void* out, int64_t* next_token, int64_t rows,
                     int64_t vocab, int32_t dtype, const void* tokens, int32_t token_bytes, int64_t width,
                     const int32_t* lengths, const int32_t* prompt_lens, const float* repetition,
                     const float* presence, const float* frequency, const int32_t* bias_start,
                     const int32_t* bias_tokens, const float* bias_values, int64_t bias_count, const int32_t* mask,
                     void* workspace, size_t workspace_bytes, void* stream) {
    if (rows < 0 || vocab <= 0 || row_stride < vocab || width < 0 || bias_count < 0) return AWQ_ERR_BAD_DIMS;
    if (dtype != AWQ_SERVE_FP16 && dtype != AWQ_SERVE_BF16 && dtype != AWQ_SERVE_FP32) return AWQ_ERR_PATH;
    if (tokens && token_bytes != 4 && token_bytes != 8) return AWQ_ERR_PATH;
    if (rows > 65535 || vocab > kIndexLimit / 2 || bias_count >= kIndexLimit || width > kIndexLimit)
        return AWQ_ERR_TOO_LARGE;
    if (rows == 0) return AWQ_OK;
    if (!logits || !out || !next_token) return AWQ_ERR_NULL_POINTER;
    if (!tokens != !lengths || !tokens != !prompt_lens || !bias_start != !bias_tokens || !bias_start != !bias_values)
        return AWQ_ERR_NULL_POINTER;
    if (!tokens && (repetition || presence || frequency)) return AWQ_ERR_NULL_POINTER;
    const uintptr_t size = dtype == AWQ_SERVE_FP32 ? 4 : 2;
    if (!aligned(logits, size) || !aligned(out, size) || !aligned(next_token, 8) || !aligned(workspace, 8) ||
        (tokens && !aligned(tokens, token_bytes)) || !aligned(lengths, 4) || !aligned(prompt_lens, 4) ||
        !aligned(repetition, 4) || !aligned(presence, 4) || !aligned(frequency, 4) || !aligned(bias_start, 4) ||
        !aligned(bias_tokens, 4) || !aligned(bias_values, 4) || !aligned(mask, 4))
        return AWQ_ERR_MISALIGNED;
    if (!workspace || workspace_bytes < logits_workspace((int)rows, (int)vocab)) return AWQ_ERR_WORKSPACE;
    LogitsArgs a = {};
    a.logits = logits;
    a.ld = row_stride;
    a.out = out;
    a.next = next_token;
    a.rows = (int)rows;
    a.vocab = (int)vocab;
    a.dtype = dtype;
    a.tokens = tokens;
    a.token_bytes = token_bytes;
    a.width = width;
    a.lengths = lengths;
    a.prompt_lens = prompt_lens;
    a.repetition = repetition;
    a.presence = presence;
    a.frequency = frequency;
    a.bias_start = bias_start;
    a.bias_tokens = bias_tokens;
    a.bias_values = bias_values;
    a.bias_count = (int)bias_count;
    a.mask = reinterpret_cast<const uint32_t*>(mask);
    a.keys = static_cast<uint64_t*>(workspace);
    return done(launch_logits(a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
