// Bindings of a KV cache in 8 bits: kv8_append, kv8_read and kv8_fwd_kvcache over fa_kv8_append, fa_kv8_read and
// fa_kv8_attention.
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <optional>
#include <tuple>
#include <utility>
#include <vector>

#include "api_common.h"

namespace {

int32_t dtype_of(const at::Tensor &t) {
    TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16,
                "attention over a cache in 8 bits needs float16 or bfloat16 tensors");
    return t.scalar_type() == at::kBFloat16 ? FA_BF16 : FA_FP16;
}

const int32_t *int32s(const std::optional<at::Tensor> &t, const at::Device &device, int64_t dim, int64_t size, const char *name) {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == device, name, " must be on the device of the cache");
    TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == dim && t->size(0) == size &&
                    (t->numel() == 0 || t->stride(-1) == 1 || t->size(-1) == 1),
                name, " must be an int32 tensor of rank ", dim, " with ", size, " rows");
    return t->data_ptr<int32_t>();
}

// Whether two elements share a place: of the sizes over 1, in the order of their strides, each stride has to pass what
// those before it span.
bool overlaps(const at::Tensor &c) {
    std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
    for (int64_t i = 0; i < c.dim(); ++i)
        if (c.size(i) > 1) dims.emplace_back(c.stride(i), c.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t span = 1;
    for (const auto &[stride, size] : dims) {
        if (stride < span) return true;
        span += (size - 1) * stride;
    }
    return false;
}

// The descriptor of a rank-3 (packed) or rank-4 tensor; a size of 1 has no stride (torch leaves any number there).
fa_tensor desc(const at::Tensor &t) {
    fa_tensor d = t.dim() == 3 ? desc3(t) : desc4(t);
    const int64_t i = t.dim() - 3;
    if (i == 0 || t.size(0) == 1) d.batch_stride = 0;
    if (t.size(i) == 1) d.row_stride = 0;
    if (t.size(i + 1) == 1) d.head_stride = 0;
    return d;
}

fa_kv8_scales scales(const at::Tensor &s, const at::Tensor &c, const char *name) {
    TORCH_CHECK(s.device() == c.device() && s.scalar_type() == at::kFloat, name, " must be a float32 tensor on the device of the cache");
    TORCH_CHECK(s.dim() == 3 && s.size(0) == c.size(0) && s.size(2) == c.size(2), name,
                " must have shape [num_blocks or rows, tokens / block, nheads_k]");
    return fa_kv8_scales{s.data_ptr<float>(), s.size(0) == 1 ? 0 : s.stride(0), s.size(1) == 1 ? 0 : s.stride(1),
                         s.size(2) == 1 ? 0 : s.stride(2)};
}

// batch: sequences of the call; write: the call appends.
fa_kv8_cache cache_of(const at::Tensor &k, const at::Tensor &v, const at::Tensor &k_scale, const at::Tensor &v_scale,
                      const std::optional<at::Tensor> &index, const std::optional<at::Tensor> &table, int64_t batch, bool write,
                      const std::optional<at::Tensor> &status) {
    fa_kv8_cache c{};
    for (const auto &[t, name] : {std::pair<const at::Tensor &, const char *>(k, "k_cache"), {v, "v_cache"}}) {
        TORCH_CHECK(t.is_cuda() && t.device() == k.device(), name, " must be a CUDA (HIP) tensor on the device of k_cache");
        TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kChar, name,
                    " must be a float8_e4m3fn or int8 tensor");
        TORCH_CHECK(t.dim() == 4, name, " must be a rank-4 tensor");
        bool ok = (t.stride(3) == 1 || t.size(3) == 1) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
        for (int64_t i = 0; i < 3; ++i) ok = ok && (t.stride(i) % 16 == 0 || t.size(i) == 1);
        TORCH_CHECK(ok, name, " must have a contiguous last dimension and 16-byte aligned rows");
        TORCH_CHECK(t.size(1) <= 1 || t.stride(1) <= int64_t(1) << 23, name, " must have tokens at most 2^23 elements apart");
        TORCH_CHECK(!write || !overlaps(t), name, " must not overlap itself");
    }
    TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), "k_cache and v_cache must match");
    check_supported_head_dim(k.size(3));
    TORCH_CHECK(k.size(2) > 0, "the cache must have heads");
    c.k = desc(k);
    c.v = desc(v);
    c.k_scale = scales(k_scale, k, "k_scale");
    c.v_scale = scales(v_scale, v, "v_scale");
    TORCH_CHECK(!write || (!overlaps(k_scale) && !overlaps(v_scale)), "k_scale and v_scale must not overlap themselves");
    const int64_t tokens = k.size(1), blocks = k_scale.size(1);
    TORCH_CHECK(v_scale.size(1) == blocks, "k_scale and v_scale must match");
    c.scale_block = 32;  // of a cache without tokens
    if (tokens > 0) {
        TORCH_CHECK(blocks > 0 && tokens % blocks == 0, "the tokens of a page or row must be a multiple of its scales");
        const int64_t block = tokens / blocks;
        TORCH_CHECK(block == 32 || block == 64 || block == 128 || block == 256, "blocks of a scale must have 32, 64, 128 or 256 tokens");
        c.scale_block = int32_t(block);
    }
    c.batch = i32(batch, "batch_size");
    c.nheads_k = i32(k.size(2), "num_heads_k");
    c.head_dim = int32_t(k.size(3));
    c.kind = k.scalar_type() == at::kChar ? FA_KV8_INT8 : FA_KV8_E4M3;
    c.cache_batch_idx = int32s(index, k.device(), 1, batch, "cache_batch_idx");
    c.block_table = int32s(table, k.device(), 2, batch, "block_table");
    if (table.has_value()) {
        TORCH_CHECK(!index.has_value(), "Paged KV cache does not support cache_batch_idx");
        TORCH_CHECK(tokens > 0, "Paged KV cache block size must be divisible by the scales' blocks");
        c.block_table_stride = table->stride(0);
        c.page_block_size = i32(tokens, "page_block_size");
        c.num_pages = i32(k.size(0), "num_blocks");
        c.cache_capacity = i32(table->size(1) * tokens, "cache capacity");
    } else {
        TORCH_CHECK(index.has_value() || k.size(0) == batch, "k_cache batch size must match the call's");
        c.cache_capacity = i32(tokens, "cache capacity");
        c.cache_batch = i32(k.size(0), "cache batch");
    }
    if (status.has_value()) c.status = const_cast<int32_t *>(int32s(status, k.device(), 1, 1, "status"));
    return c;
}

void check_new(const at::Tensor &k, const at::Tensor &v, const at::Tensor &cache, int64_t batch) {
    for (const auto *t : {&k, &v})
        TORCH_CHECK(t->device() == cache.device() && t->scalar_type() == k.scalar_type(),
                    "k and v must have one dtype and be on the device of the cache");
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == batch && k.size(2) == cache.size(2) &&
                    k.size(3) == cache.size(3),
                "k and v must have shape [batch_size, seqlen_new, nheads_k, head_dim]");
}

void kv8_append(at::Tensor k, at::Tensor v, at::Tensor k_cache, at::Tensor v_cache, at::Tensor k_scale, at::Tensor v_scale,
                at::Tensor cache_seqlens, std::optional<at::Tensor> cache_batch_idx, std::optional<at::Tensor> block_table,
                std::optional<at::Tensor> seqlens_new, std::optional<at::Tensor> status) {
    TORCH_CHECK(k.is_cuda(), "k must be a CUDA (HIP) tensor");
    TORCH_CHECK(k.dim() == 4, "k and v must be rank-4 tensors");
    const int64_t batch = k.size(0);
    fa_kv8_args a{};
    a.cache = cache_of(k_cache, v_cache, k_scale, v_scale, cache_batch_idx, block_table, batch, true, status);
    check_new(k, v, k_cache, batch);
    a.dtype = dtype_of(k);
    a.cache_seqlens = int32s(cache_seqlens, k_cache.device(), 1, batch, "cache_seqlens");
    a.seqlens_new = int32s(seqlens_new, k_cache.device(), 1, batch, "seqlens_new");
    a.seqlen_new = i32(k.size(1), "seqlen_new");
    if (batch == 0 || a.seqlen_new == 0) return;
    TORCH_CHECK(k_cache.numel() > 0, "cache capacity is insufficient for the requested append length");
    c10::DeviceGuard guard(k_cache.device());
    k = aligned(k);
    v = aligned(v);
    a.k_new = desc(k);
    a.v_new = desc(v);
    check_rc(fa_kv8_append(&a, current_stream()), "fa_kv8_append");
}

std::tuple<at::Tensor, at::Tensor> kv8_read(at::Tensor k_cache, at::Tensor v_cache, at::Tensor k_scale, at::Tensor v_scale,
                                            at::Tensor cu_seqlens, int64_t total, std::optional<at::Tensor> cache_batch_idx,
                                            std::optional<at::Tensor> block_table, bool bf16, std::optional<at::Tensor> status) {
    TORCH_CHECK(cu_seqlens.dim() == 1 && cu_seqlens.numel() >= 1, "cu_seqlens_k must have batch_size + 1 elements");
    const int64_t batch = cu_seqlens.numel() - 1;
    fa_kv8_read_args a{};
    a.cache = cache_of(k_cache, v_cache, k_scale, v_scale, cache_batch_idx, block_table, batch, false, status);
    a.cu_seqlens = int32s(cu_seqlens, k_cache.device(), 1, batch + 1, "cu_seqlens_k");
    a.total = i32(total, "total_k");
    a.dtype = bf16 ? FA_BF16 : FA_FP16;
    c10::DeviceGuard guard(k_cache.device());
    const auto options = k_cache.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
    at::Tensor k = at::empty({total, k_cache.size(2), k_cache.size(3)}, options), v = at::empty(k.sizes(), options);
    if (total == 0) return {k, v};
    if (k_cache.numel() == 0) {
        k.zero_();
        v.zero_();
        return {k, v};
    }
    a.k_out = desc(k);
    a.v_out = desc(v);
    check_rc(fa_kv8_read(&a, current_stream()), "fa_kv8_read");
    return {k, v};
}

std::tuple<at::Tensor, at::Tensor> kv8_fwd_kvcache(at::Tensor q, at::Tensor k_cache, at::Tensor v_cache, at::Tensor k_scale,
                                                   at::Tensor v_scale, std::optional<at::Tensor> k_, std::optional<at::Tensor> v_,
                                                   at::Tensor cache_seqlens, std::optional<at::Tensor> cache_batch_idx,
                                                   std::optional<at::Tensor> block_table, double softmax_scale, bool causal,
                                                   int64_t window_left, int64_t window_right, int64_t num_splits,
                                                   std::optional<at::Tensor> status) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA (HIP) tensor");
    TORCH_CHECK(q.dim() == 4, "q must be a rank-4 tensor");
    TORCH_CHECK(k_.has_value() == v_.has_value(), "k and v must either both be provided or both be None");
    const int64_t batch = q.size(0);
    fa_kv8_args a{};
    a.cache = cache_of(k_cache, v_cache, k_scale, v_scale, cache_batch_idx, block_table, batch, k_.has_value(), status);
    TORCH_CHECK(q.device() == k_cache.device(), "q must be on the device of the cache");
    TORCH_CHECK(q.size(3) == k_cache.size(3), "q/k/v head_dim must match");
    TORCH_CHECK(q.size(2) > 0 && q.size(2) % k_cache.size(2) == 0, "num_heads_q must be divisible by num_heads_k for GQA/MQA");
    a.dtype = dtype_of(q);
    a.cache_seqlens = int32s(cache_seqlens, q.device(), 1, batch, "cache_seqlens");
    c10::DeviceGuard guard(q.device());
    q = aligned(q);
    at::Tensor k, v;
    if (k_.has_value()) {
        check_new(*k_, *v_, k_cache, batch);
        TORCH_CHECK(k_->scalar_type() == q.scalar_type(), "k must have the dtype of q");
        k = aligned(*k_);
        v = aligned(*v_);
        a.seqlen_new = i32(k.size(1), "seqlen_new");
        if (a.seqlen_new > 0) {
            a.k_new = desc(k);
            a.v_new = desc(v);
        }
    }
    at::Tensor out = at::empty(q.sizes(), q.options());
    at::Tensor lse = at::empty({batch, q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    if (batch == 0 || (q.numel() == 0 && a.seqlen_new == 0)) return {out, lse};
    if (k_cache.numel() == 0) {
        TORCH_CHECK(a.seqlen_new == 0, "cache capacity is insufficient for the requested append length");
        out.zero_();
        lse.zero_();
        return {out, lse};
    }
    a.q = desc(q);
    a.o = desc(out);
    a.lse = lse.data_ptr<float>();
    a.seqlen_q = i32(q.size(1), "seqlen_q");
    a.nheads = i32(q.size(2), "num_heads");
    a.causal = causal;
    a.window_left = int32_t(std::min<int64_t>(window_left, INT32_MAX / 2));
    a.window_right = int32_t(std::min<int64_t>(window_right, INT32_MAX / 2));
    a.num_splits = i32(num_splits, "num_splits");
    a.softmax_scale = float(softmax_scale);
    at::Tensor ws;
    a.ws_bytes = int64_t(fa_kv8_ws_bytes(&a));
    if (a.ws_bytes > 0) {
        ws = at::empty({a.ws_bytes}, q.options().dtype(at::kByte));
        a.ws = ws.data_ptr();
    }
    check_rc(fa_kv8_attention(&a, current_stream()), "fa_kv8_attention");
    return {out, lse};
}

}  // namespace

void bind_kv8(py::module_ &m) {
    m.def("kv8_append", &kv8_append, "Append to a KV cache in 8 bits");
    m.def("kv8_read", &kv8_read, "Read a KV cache in 8 bits back");
    m.def("kv8_fwd_kvcache", &kv8_fwd_kvcache, "Attention over a KV cache in 8 bits");
}
