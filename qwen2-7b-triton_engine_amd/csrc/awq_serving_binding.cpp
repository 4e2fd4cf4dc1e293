// Python binding of the serving operators for torch tensors (host code only;
// include/awq_serving.h): checks, outputs, workspace and the current stream in
// one call from kernels/paged.py, kv4.py and logits.py.  ValueError for a bad operand,
// AwqNativeError for a status of the library.  Their kernels take 4 to 12 us where
// a step is small, and the same call through ctypes took 15 to 25.
#include "awq_binding.h"

#include <ATen/DeviceGuard.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <limits>
#include <tuple>

#include "../../include/awq_serving.h"

namespace awq_binding {
namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
constexpr int64_t kIntMax = std::numeric_limits<int32_t>::max();

hipStream_t stream_of(const at::Device& device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

void check_on_gpu(const Tensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.device().is_cuda(), what, " must be on a ROCm device, got ", t.device());
}
void check_i32(const Tensor& t, const char* what, at::IntArrayRef shape, const at::Device& device) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.sizes() == shape && t.is_contiguous() && t.device() == device, what,
                      " must be a contiguous int32 tensor ", shape, " on ", device, ", got ", t.scalar_type(), " ",
                      t.sizes(), " on ", t.device());
}
const int32_t* i32(const Tensor& t) { return t.data_ptr<int32_t>(); }

// fp16 or bf16
int type16(const Tensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, what, " must be float16 or bfloat16, got ",
                      t.scalar_type());
    return t.scalar_type() == at::kHalf ? AWQ_SERVE_FP16 : AWQ_SERVE_BF16;
}
// `t` [rows, columns] itself where its rows are dense and start on 16 bytes, else a copy.
Tensor rows16(const Tensor& t) {
    if (t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1))) &&
        (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0)
        return t;
    return aligned16(t.contiguous());
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// None of these is differentiable: their allocations and views go straight to the backend.
using Plain = at::AutoDispatchBelowADInplaceOrView;

struct Cache {
    const Tensor& data;
    int64_t head_dim, page_size, group_size;
    int64_t pages() const { return data.size(0); }
    int64_t heads() const { return data.size(1); }
};

// Tables as kernels/paged.py holds them.  Checked where they are made and in every call: their parts
// can be set, and the kernels go by them.
void check_tables(const Tensor& block_tables, const Tensor& state, const Tensor& free_pages, int64_t page_size) {
    TORCH_CHECK_VALUE(block_tables.dim() == 2 && free_pages.dim() == 1, "block_tables must be 2-D and free_pages 1-D");
    const int64_t requests = block_tables.size(0), width = block_tables.size(1), capacity = free_pages.size(0);
    const at::Device device = block_tables.device();
    check_i32(block_tables, "block_tables", {requests, width}, device);
    check_i32(state, "state", {requests + 1}, device);
    check_i32(free_pages, "free_pages", {capacity}, device);
    TORCH_CHECK_VALUE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 || page_size == 256, "page_size ",
                      page_size, " must be 16, 32, 64, 128 or 256");
    TORCH_CHECK_VALUE(requests > 0 && requests <= AWQ_SERVE_MAX_REQUESTS && width > 0 && capacity > 0, requests, " requests of ",
                      width, " pages, ", capacity, " pages in all: need 1 to ", AWQ_SERVE_MAX_REQUESTS,
                      " requests and at least one page");
    TORCH_CHECK_VALUE(width <= (1 << 30) / page_size && capacity <= (1 << 24), "a request's tokens pass 2^30, or the free pages 2^24");
}
// A cache as kernels/kv4.py holds it, checked alike.
void check_cache(const Tensor& data, int64_t head_dim, int64_t page_size, int64_t group_size) {
    TORCH_CHECK_VALUE(head_dim == 64 || head_dim == 128, "head_dim ", head_dim, " must be 64 or 128");
    TORCH_CHECK_VALUE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 || page_size == 256, "page_size ",
                      page_size, " must be 16, 32, 64, 128 or 256");
    TORCH_CHECK_VALUE((group_size == 32 || group_size == 64 || group_size == 128) && group_size <= head_dim, "group_size ", group_size,
                      " must be 32, 64 or 128 and at most head_dim ", head_dim);
    const int64_t block = page_size * (head_dim + 8 * (head_dim / group_size));
    TORCH_CHECK_VALUE(data.scalar_type() == at::kByte && data.dim() == 3 && data.size(2) == block && data.is_contiguous(),
                      "data must be a contiguous uint8 tensor [pages, kv heads, ", block, "], got ", data.scalar_type(), " ",
                      data.sizes());
    TORCH_CHECK_VALUE(data.size(0) >= 1 && data.size(1) >= 1 && (reinterpret_cast<uintptr_t>(data.data_ptr()) & 15u) == 0,
                      "data must hold a page and a head and start on 16 bytes");
    TORCH_CHECK_VALUE(data.size(0) <= kIntMax / page_size, "slot numbers pass 32 bits");
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> paged_step(const Tensor& state, const Tensor& new_tokens,
                                                              const Tensor& block_tables, const Tensor& free_pages,
                                                              int64_t page_size, int64_t total,
                                                              const c10::optional<std::vector<Tensor>>& out) {
    const Plain plain;
    check_tables(block_tables, state, free_pages, page_size);
    const at::Device device = state.device();
    check_on_gpu(state, "the tables");
    const int64_t requests = block_tables.size(0), width = block_tables.size(1);
    check_i32(new_tokens, "new_tokens", {requests}, device);
    TORCH_CHECK_VALUE(total >= 0 && total <= (1 << 24), "total ", total, " must be in [0, 2^24]");
    Tensor o[5];
    const int64_t sizes[5] = {requests + 1, requests + 1, total, total, requests};
    if (out.has_value()) {
        static const char* names[5] = {"out.state", "out.query_start", "out.slots", "out.positions", "out.failed"};
        for (int i = 0; i < 5; ++i) check_i32(o[i] = (*out)[i], names[i], {sizes[i]}, device);
        TORCH_CHECK_VALUE(o[0].data_ptr() != state.data_ptr(),
                          "out.state is the tables' own state: the step reads it while it writes");
    } else {
        // one allocation, one call for its parts
        const std::vector<Tensor> parts =
            at::empty({3 * requests + 2 + 2 * total}, state.options()).unsafe_split_with_sizes(sizes, 0);
        for (int i = 0; i < 5; ++i) o[i] = parts[i];
    }
    const at::DeviceGuard guard(device);
    check_status(awq_serve_page_step(i32(state), i32(new_tokens), block_tables.data_ptr<int32_t>(), i32(free_pages),
                                     o[0].data_ptr<int32_t>(), o[1].data_ptr<int32_t>(), o[2].data_ptr<int32_t>(),
                                     o[3].data_ptr<int32_t>(), o[4].data_ptr<int32_t>(), requests, total, width,
                                     free_pages.size(0), page_size, stream_of(device)),
                 "awq_serve_page_step");
    return {o[0], o[1], o[2], o[3], o[4]};
}

Tensor paged_release(const Tensor& state, const Tensor& keep, const Tensor& block_tables, const Tensor& free_pages,
                     int64_t page_size) {
    check_tables(block_tables, state, free_pages, page_size);
    const at::Device device = state.device();
    check_on_gpu(state, "the tables");
    const int64_t requests = block_tables.size(0);
    check_i32(keep, "keep", {requests}, device);
    Tensor out = at::empty_like(state);
    const at::DeviceGuard guard(device);
    check_status(awq_serve_page_release(i32(state), i32(keep), i32(block_tables), free_pages.data_ptr<int32_t>(),
                                        out.data_ptr<int32_t>(), requests, block_tables.size(1), free_pages.size(0),
                                        page_size, stream_of(device)),
                 "awq_serve_page_release");
    return out;
}

// RoPE's tables, both or neither, aligned; their positions (no table: any).
int64_t check_rope(const OptTensor& cos_in, const OptTensor& sin_in, int64_t head_dim, const at::Device& device, Tensor& cos,
                   Tensor& sin) {
    TORCH_CHECK_VALUE(cos_in.has_value() == sin_in.has_value(), "cos and sin come together");
    if (!cos_in.has_value()) return kIntMax;
    const int64_t max_pos = cos_in->dim() == 2 ? cos_in->size(0) : 0;
    for (const Tensor* t : {&*cos_in, &*sin_in})
        TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == max_pos && max_pos > 0 &&
                              t->size(1) == head_dim && t->is_contiguous() && t->device() == device,
                          "cos and sin must be contiguous float32 tensors [max_pos, ", head_dim, "] on ", device);
    cos = aligned16(*cos_in);
    sin = aligned16(*sin_in);
    return max_pos;
}

Tensor kv4_append(const Tensor& qkv_in, const Tensor& data, int64_t head_dim, int64_t page_size, int64_t group_size,
                  const Tensor& slots, const Tensor& positions, const OptTensor& cos_in, const OptTensor& sin_in,
                  int64_t num_heads) {
    const Plain plain;
    check_cache(data, head_dim, page_size, group_size);
    const Cache cache{data, head_dim, page_size, group_size};
    const at::Device device = qkv_in.device();
    const int64_t columns = (num_heads + 2 * cache.heads()) * head_dim;
    const int dtype = type16(qkv_in, "qkv");
    TORCH_CHECK_VALUE(qkv_in.dim() == 2 && qkv_in.size(1) == columns && num_heads >= 1, "qkv must be a tensor [T, ", columns,
                      "], got ", qkv_in.sizes());
    check_on_gpu(qkv_in, "qkv");
    TORCH_CHECK_VALUE(data.device() == device, "qkv and the cache must be on one device, got ", device, " and ", data.device());
    const int64_t T = qkv_in.size(0);
    check_i32(slots, "slots", {T}, device);
    check_i32(positions, "positions", {T}, device);
    const at::DeviceGuard guard(device);
    Tensor cos, sin;
    const int64_t max_pos = check_rope(cos_in, sin_in, head_dim, device, cos, sin);
    const Tensor qkv = rows16(qkv_in);
    Tensor q = at::empty({T, num_heads * head_dim}, qkv.options());
    check_status(awq_serve_kv4_append(qkv.data_ptr(), row_stride(qkv), data.data_ptr(), i32(slots), i32(positions),
                                      cos.defined() ? cos.data_ptr() : nullptr, sin.defined() ? sin.data_ptr() : nullptr,
                                      q.data_ptr(), T, num_heads, cache.heads(), head_dim, cache.pages(), page_size,
                                      group_size, max_pos, dtype, stream_of(device)),
                 "awq_serve_kv4_append");
    return q;
}

std::tuple<Tensor, Tensor> kv4_gather(const Tensor& data, int64_t head_dim, int64_t page_size, int64_t group_size,
                                      const Tensor& slots, at::ScalarType dtype) {
    const Plain plain;
    check_cache(data, head_dim, page_size, group_size);
    const Cache cache{data, head_dim, page_size, group_size};
    TORCH_CHECK_VALUE(dtype == at::kHalf || dtype == at::kBFloat16, "dtype must be float16 or bfloat16, got ", dtype);
    check_on_gpu(data, "the cache");
    TORCH_CHECK_VALUE(slots.dim() == 1, "slots must be 1-D");
    const int64_t T = slots.size(0);
    check_i32(slots, "slots", {T}, data.device());
    const at::DeviceGuard guard(data.device());
    Tensor k = at::empty({T, cache.heads(), head_dim}, data.options().dtype(dtype)), v = at::empty_like(k);
    check_status(awq_serve_kv4_gather(data.data_ptr(), i32(slots), k.data_ptr(), v.data_ptr(), T, cache.heads(), head_dim,
                                      cache.pages(), page_size, group_size,
                                      dtype == at::kHalf ? AWQ_SERVE_FP16 : AWQ_SERVE_BF16, stream_of(data.device())),
                 "awq_serve_kv4_gather");
    return {k, v};
}

// What the attention calls have in common: sizes, checked.
struct AttentionCall {
    at::Device device;
    int64_t heads, requests, width, rows, most;
    float scale;
};
AttentionCall check_attention(const Tensor& q_in, const Tensor& data, int64_t kvh, int64_t head_dim, int64_t page_size,
                              const Tensor& block_tables, const Tensor& seq_lens, const Tensor& query_start, int64_t max_query,
                              c10::optional<double> scale_in) {
    const at::Device device = q_in.device();
    TORCH_CHECK_VALUE(q_in.dim() == 2 && q_in.size(1) > 0 && q_in.size(1) % (head_dim * kvh) == 0, "q must be a tensor [T, heads * ",
                      head_dim, "] with heads a multiple of ", kvh, ", got ", q_in.sizes());
    const int64_t heads = q_in.size(1) / head_dim;
    TORCH_CHECK_VALUE(heads / kvh <= AWQ_SERVE_MAX_GROUP, heads / kvh, " heads share a kv head: at most ", AWQ_SERVE_MAX_GROUP,
                      " are served");
    check_on_gpu(q_in, "q");
    TORCH_CHECK_VALUE(data.device() == device, "q and the cache must be on one device, got ", device, " and ", data.device());
    TORCH_CHECK_VALUE(block_tables.dim() == 2 && block_tables.scalar_type() == at::kInt && block_tables.is_contiguous() &&
                          block_tables.device() == device,
                      "block_tables must be a contiguous int32 tensor [requests, width] on ", device);
    const int64_t requests = block_tables.size(0), width = block_tables.size(1);
    TORCH_CHECK_VALUE(requests > 0 && requests <= AWQ_SERVE_MAX_REQUESTS && width >= 1, "block_tables ", block_tables.sizes(),
                      ": need 1 to ", AWQ_SERVE_MAX_REQUESTS, " requests");
    TORCH_CHECK_VALUE(width <= (1 << 30) / page_size, "a request's tokens pass 2^30");
    check_i32(seq_lens, "seq_lens", {requests}, device);
    check_i32(query_start, "query_start", {requests + 1}, device);
    TORCH_CHECK_VALUE(max_query >= 1, "max_query ", max_query, " must be positive");
    const double scale = scale_in.has_value() ? *scale_in : 1.0 / std::sqrt((double)head_dim);
    TORCH_CHECK_VALUE(scale > 0.0 && std::isfinite(scale) && (float)scale > 0.0f && std::isfinite((float)scale), "scale ", scale,
                      " must be positive and finite");
    const int64_t T = q_in.size(0);
    const int64_t most = std::min(max_query, std::max<int64_t>(T, 1));
    return {device, heads, requests, width, T, most, (float)scale};
}

Tensor kv4_attention(const Tensor& q_in, const Tensor& data, int64_t head_dim, int64_t page_size, int64_t group_size,
                     const Tensor& block_tables, const Tensor& seq_lens, const Tensor& query_start, int64_t max_query,
                     c10::optional<double> scale_in) {
    const Plain plain;
    check_cache(data, head_dim, page_size, group_size);
    const Cache cache{data, head_dim, page_size, group_size};
    const at::Device device = q_in.device();
    const int64_t kvh = cache.heads();
    const int dtype = type16(q_in, "q");
    const AttentionCall c =
        check_attention(q_in, data, kvh, head_dim, page_size, block_tables, seq_lens, query_start, max_query, scale_in);
    const int64_t heads = c.heads, requests = c.requests, width = c.width, T = c.rows, most = c.most;
    const at::DeviceGuard guard(device);
    const Tensor q = rows16(q_in);
    Tensor out = at::empty({T, heads * head_dim}, q.options());
    if (T == 0) return out;
    const size_t bytes = awq_serve_kv4_attention_workspace(requests, T, most, heads, kvh, head_dim, width, page_size);
    const Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check_status(awq_serve_kv4_attention(q.data_ptr(), row_stride(q), data.data_ptr(), i32(block_tables), i32(seq_lens),
                                         i32(query_start), out.data_ptr(), requests, T, most, heads, kvh, head_dim, width,
                                         cache.pages(), page_size, group_size, c.scale, dtype, ws.data_ptr(), bytes,
                                         stream_of(device)),
                 "awq_serve_kv4_attention");
    return out;
}

// A 16-bit cache as kernels/kv16.py holds it.
void check_cache16(const Tensor& data) {
    TORCH_CHECK_VALUE((data.scalar_type() == at::kHalf || data.scalar_type() == at::kBFloat16) && data.dim() == 5 && data.size(2) == 2 &&
                          data.is_contiguous(),
                      "data must be a contiguous fp16 or bf16 tensor [pages, kv heads, 2, page_size, head_dim], got ",
                      data.scalar_type(), " ", data.sizes());
    const int64_t page_size = data.size(3), head_dim = data.size(4);
    TORCH_CHECK_VALUE(head_dim == 64 || head_dim == 128, "head_dim ", head_dim, " must be 64 or 128");
    TORCH_CHECK_VALUE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 || page_size == 256, "page_size ",
                      page_size, " must be 16, 32, 64, 128 or 256");
    TORCH_CHECK_VALUE(data.size(0) >= 1 && data.size(1) >= 1 && (reinterpret_cast<uintptr_t>(data.data_ptr()) & 15u) == 0,
                      "data must hold a page and a head and start on 16 bytes");
    TORCH_CHECK_VALUE(data.size(0) <= kIntMax / page_size, "slot numbers pass 32 bits");
}

Tensor kv16_append(const Tensor& qkv_in, const Tensor& data, const Tensor& slots, const Tensor& positions,
                   const OptTensor& cos_in, const OptTensor& sin_in, int64_t num_heads) {
    const Plain plain;
    check_cache16(data);
    const at::Device device = qkv_in.device();
    const int64_t kvh = data.size(1), head_dim = data.size(4), columns = (num_heads + 2 * kvh) * head_dim;
    const int dtype = type16(qkv_in, "qkv");
    TORCH_CHECK_VALUE(qkv_in.scalar_type() == data.scalar_type(), "qkv and the cache must be of one type, got ",
                      qkv_in.scalar_type(), " and ", data.scalar_type());
    TORCH_CHECK_VALUE(qkv_in.dim() == 2 && qkv_in.size(1) == columns && num_heads >= 1, "qkv must be a tensor [T, ", columns,
                      "], got ", qkv_in.sizes());
    check_on_gpu(qkv_in, "qkv");
    TORCH_CHECK_VALUE(data.device() == device, "qkv and the cache must be on one device, got ", device, " and ", data.device());
    const int64_t T = qkv_in.size(0);
    check_i32(slots, "slots", {T}, device);
    check_i32(positions, "positions", {T}, device);
    const at::DeviceGuard guard(device);
    Tensor cos, sin;
    const int64_t max_pos = check_rope(cos_in, sin_in, head_dim, device, cos, sin);
    const Tensor qkv = rows16(qkv_in);
    Tensor q = at::empty({T, num_heads * head_dim}, qkv.options());
    check_status(awq_serve_kv16_append(qkv.data_ptr(), row_stride(qkv), data.data_ptr(), i32(slots), i32(positions),
                                       cos.defined() ? cos.data_ptr() : nullptr, sin.defined() ? sin.data_ptr() : nullptr,
                                       q.data_ptr(), T, num_heads, kvh, head_dim, data.size(0), data.size(3), max_pos, dtype,
                                       stream_of(device)),
                 "awq_serve_kv16_append");
    return q;
}

Tensor kv16_attention(const Tensor& q_in, const Tensor& data, const Tensor& block_tables, const Tensor& seq_lens,
                      const Tensor& query_start, int64_t max_query, c10::optional<double> scale_in,
                      c10::optional<double> softcap_in, const OptTensor& slopes, c10::optional<int64_t> window_in,
                      const OptTensor& prefix, const OptTensor& first) {
    const Plain plain;
    check_cache16(data);
    const int64_t head_dim = data.size(4), page_size = data.size(3);
    TORCH_CHECK_VALUE(q_in.scalar_type() == data.scalar_type(), "q and the cache must be of one type, got ", q_in.scalar_type(),
                      " and ", data.scalar_type());
    const AttentionCall c = check_attention(q_in, data, data.size(1), head_dim, page_size, block_tables, seq_lens, query_start,
                                            max_query, scale_in);
    double softcap = 0.0;
    if (softcap_in.has_value()) {
        softcap = *softcap_in;
        TORCH_CHECK_VALUE(softcap >= 0x1p-100 && std::isfinite((float)softcap), "softcap ", softcap, " must be positive and finite");
    }
    int64_t window = 0;
    if (window_in.has_value()) {
        window = *window_in;
        TORCH_CHECK_VALUE(window >= 1, "window ", window, " must be positive");
    }
    const float* slope = nullptr;
    if (slopes.has_value()) {
        TORCH_CHECK_VALUE(slopes->scalar_type() == at::kFloat && slopes->sizes() == at::IntArrayRef({c.heads}) &&
                              slopes->is_contiguous() && slopes->device() == c.device,
                          "slopes must be a contiguous float32 tensor [", c.heads, "] on ", c.device);
        slope = slopes->data_ptr<float>();
    }
    if (prefix.has_value()) check_i32(*prefix, "prefix", {c.requests}, c.device);
    if (first.has_value()) check_i32(*first, "first", {c.rows}, c.device);
    const at::DeviceGuard guard(c.device);
    const Tensor q = rows16(q_in);
    Tensor out = at::empty({c.rows, c.heads * head_dim}, q.options());
    if (c.rows == 0) return out;
    const size_t bytes =
        awq_serve_kv16_attention_workspace(c.requests, c.rows, c.most, c.heads, data.size(1), head_dim, c.width, page_size);
    const Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check_status(awq_serve_kv16_attention(q.data_ptr(), row_stride(q), data.data_ptr(), i32(block_tables), i32(seq_lens),
                                          i32(query_start), slope, prefix.has_value() ? i32(*prefix) : nullptr,
                                          first.has_value() ? i32(*first) : nullptr, out.data_ptr(), c.requests, c.rows, c.most,
                                          c.heads, data.size(1), head_dim, c.width, data.size(0), page_size, window, c.scale,
                                          (float)softcap, q.scalar_type() == at::kHalf ? AWQ_SERVE_FP16 : AWQ_SERVE_BF16,
                                          ws.data_ptr(), bytes, stream_of(c.device)),
                 "awq_serve_kv16_attention");
    return out;
}

std::tuple<Tensor, Tensor> token_logprobs(const Tensor& hidden_in, const Tensor& weight_in, const Tensor& targets) {
    const Plain plain;
    const int dtype = type16(hidden_in, "hidden");
    TORCH_CHECK_VALUE(weight_in.scalar_type() == hidden_in.scalar_type(), "hidden and weight must be of one type, got ",
                      hidden_in.scalar_type(), " and ", weight_in.scalar_type());
    TORCH_CHECK_VALUE(hidden_in.dim() == 2 && weight_in.dim() == 2 && hidden_in.size(1) == weight_in.size(1) && weight_in.size(0) > 0,
                      "hidden must be [T, K] and weight [V, K], got ", hidden_in.sizes(), " and ", weight_in.sizes());
    const int64_t T = hidden_in.size(0), K = hidden_in.size(1), V = weight_in.size(0);
    TORCH_CHECK_VALUE(K > 0 && K % 64 == 0, "K = ", K, " must be a multiple of 64");
    TORCH_CHECK_VALUE(K <= (1 << 20) && V <= (1 << 24) && T <= (1 << 24), "hidden ", hidden_in.sizes(), " and weight ",
                      weight_in.sizes(), ": at most 2^24 tokens, as many vocabulary rows and K = 2^20 are served");
    check_on_gpu(hidden_in, "hidden");
    const at::Device device = hidden_in.device();
    TORCH_CHECK_VALUE(weight_in.device() == device, "hidden and weight must be on one device, got ", device, " and ",
                      weight_in.device());
    TORCH_CHECK_VALUE((targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt) && targets.dim() == 1 &&
                          targets.size(0) == T && targets.is_contiguous() && targets.device() == device,
                      "targets must be a contiguous int64 or int32 tensor [", T, "] on ", device);
    const at::DeviceGuard guard(device);
    Tensor hidden = rows16(hidden_in);
    if (row_stride(hidden) > (1 << 22)) hidden = hidden.contiguous();
    const Tensor weight = aligned16(weight_in.contiguous());
    Tensor out = at::empty({2, T}, hidden.options().dtype(at::kFloat));
    const std::vector<Tensor> parts = out.unbind(0);
    if (T == 0) return {parts[0], parts[1]};
    const size_t bytes = awq_serve_logprobs_workspace(T, V);
    TORCH_CHECK_VALUE(bytes > 0, T, " tokens of ", V, " are more than one launch serves: give fewer at a time");
    const Tensor ws = at::empty({(int64_t)bytes}, hidden.options().dtype(at::kByte));
    check_status(awq_serve_logprobs(hidden.data_ptr(), row_stride(hidden), weight.data_ptr(), targets.data_ptr(),
                                    (int32_t)targets.element_size(), parts[0].data_ptr<float>(), parts[1].data_ptr<float>(), T, V,
                                    K, dtype, ws.data_ptr(), bytes, stream_of(device)),
                 "awq_serve_logprobs");
    return {parts[0], parts[1]};
}

std::tuple<Tensor, Tensor> process_logits(const Tensor& logits_in, const OptTensor& tokens, const OptTensor& lengths,
                                          const OptTensor& prompt_lens, const OptTensor& repetition,
                                          const OptTensor& presence, const OptTensor& frequency,
                                          const c10::optional<std::tuple<Tensor, Tensor, Tensor>>& bias,
                                          const OptTensor& mask, const OptTensor& out_in) {
    const Plain plain;
    const at::ScalarType type = logits_in.scalar_type();
    TORCH_CHECK_VALUE((type == at::kHalf || type == at::kBFloat16 || type == at::kFloat) && logits_in.dim() == 2 &&
                          logits_in.size(1) > 0,
                      "logits must be an fp16, bf16 or fp32 tensor [B, V], got ", type, " ", logits_in.sizes());
    check_on_gpu(logits_in, "logits");
    const at::Device device = logits_in.device();
    const int64_t B = logits_in.size(0), V = logits_in.size(1);
    TORCH_CHECK_VALUE(B <= 65535 && V <= kIntMax / 2, "logits ", logits_in.sizes(),
                      ": at most 65535 rows and 2^30 - 1 tokens are served");
    auto vector = [&](const OptTensor& t, const char* what, at::ScalarType dtype, int64_t n) -> const void* {
        if (!t.has_value()) return nullptr;
        TORCH_CHECK_VALUE(t->scalar_type() == dtype && t->dim() == 1 && t->size(0) == n && t->is_contiguous() &&
                              t->device() == device,
                          what, " must be a contiguous ", dtype, " tensor [", n, "] on ", device);
        return t->data_ptr();
    };
    const void *lens = vector(lengths, "lengths", at::kInt, B), *prompts = vector(prompt_lens, "prompt_lens", at::kInt, B);
    const void *rep = vector(repetition, "repetition", at::kFloat, B), *pres = vector(presence, "presence", at::kFloat, B),
               *freq = vector(frequency, "frequency", at::kFloat, B);
    const void* text = nullptr;
    int64_t width = 0;
    int32_t token_bytes = 8;
    if (tokens.has_value()) {
        TORCH_CHECK_VALUE((tokens->scalar_type() == at::kLong || tokens->scalar_type() == at::kInt) && tokens->dim() == 2 &&
                              tokens->size(0) == B && tokens->is_contiguous() && tokens->device() == device,
                          "tokens must be a contiguous int64 or int32 tensor [", B, ", L] on ", device);
        TORCH_CHECK_VALUE(lengths.has_value() && prompt_lens.has_value(), "tokens, lengths and prompt_lens come together");
        width = tokens->size(1);
        token_bytes = (int32_t)tokens->element_size();
        text = tokens->data_ptr();
        if (width == 0) text = lens = prompts = rep = pres = freq = nullptr;   // no history: no penalties
    } else {
        TORCH_CHECK_VALUE(!lengths.has_value() && !prompt_lens.has_value() && !rep && !pres && !freq && !repetition.has_value() &&
                              !presence.has_value() && !frequency.has_value(),
                          "penalties need the history: tokens, lengths and prompt_lens");
    }
    const void *start = nullptr, *ids = nullptr, *values = nullptr;
    int64_t count = 0;
    if (bias.has_value()) {
        const auto& [s, i, v] = *bias;
        TORCH_CHECK_VALUE(i.dim() == 1, "bias must be (start, tokens, values)");
        count = i.size(0);
        start = vector(s, "bias start", at::kInt, B + 1);
        ids = vector(i, "bias tokens", at::kInt, count);
        values = vector(v, "bias values", at::kFloat, count);
        if (count == 0) start = ids = values = nullptr;
    }
    const void* bits = nullptr;
    if (mask.has_value()) {
        check_i32(*mask, "mask", {B, (V + 31) / 32}, device);
        bits = mask->data_ptr();
    }
    const at::DeviceGuard guard(device);
    const Tensor logits =
        logits_in.stride(1) != 1 || (B > 1 && logits_in.stride(0) < V) ? logits_in.contiguous() : logits_in;
    Tensor out;
    if (out_in.has_value()) {
        out = *out_in;
        TORCH_CHECK_VALUE(out.scalar_type() == type && out.sizes() == at::IntArrayRef({B, V}) && out.is_contiguous() &&
                              out.device() == device,
                          "out must be a contiguous ", type, " tensor [", B, ", ", V, "] on ", device);
    } else {
        out = at::empty({B, V}, logits.options());
    }
    Tensor token = at::empty({B}, logits.options().dtype(at::kLong));
    if (B == 0) return {out, token};
    const size_t bytes = awq_serve_logits_workspace(B, V);
    const Tensor ws = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte));
    check_status(awq_serve_logits(logits.data_ptr(), row_stride(logits), out.data_ptr(), token.data_ptr<int64_t>(), B, V,
                                  type == at::kHalf ? AWQ_SERVE_FP16 : type == at::kBFloat16 ? AWQ_SERVE_BF16 : AWQ_SERVE_FP32,
                                  text, token_bytes, width, static_cast<const int32_t*>(lens),
                                  static_cast<const int32_t*>(prompts), static_cast<const float*>(rep),
                                  static_cast<const float*>(pres), static_cast<const float*>(freq),
                                  static_cast<const int32_t*>(start), static_cast<const int32_t*>(ids),
                                  static_cast<const float*>(values), count, static_cast<const int32_t*>(bits), ws.data_ptr(),
                                  bytes, stream_of(device)),
                 "awq_serve_logits");
    return {out, token};
}

}  // namespace

void define_serving(py::module_& m) {
    m.def("check_tables", &check_tables);
    m.def("check_cache", &check_cache);
    m.def("paged_step", &paged_step);
    m.def("paged_release", &paged_release);
    m.def("kv4_append", &kv4_append);
    m.def("kv4_gather", &kv4_gather);
    m.def("kv4_attention", &kv4_attention);
    m.def("check_cache16", &check_cache16);
    m.def("kv16_append", &kv16_append);
    m.def("kv16_attention", &kv16_attention);
    m.def("token_logprobs", &token_logprobs);
    m.def("process_logits", &process_logits);
}

}  // namespace awq_binding
