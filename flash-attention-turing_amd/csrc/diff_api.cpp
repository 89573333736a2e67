// Bindings of differential attention: diff_fwd, diff_bwd, their varlen forms and
// diff_fwd_kvcache over fa_diff_fwd, fa_diff_bwd and fa_diff_kvcache.  Checks,
// streams and workspaces as in flash_api.cpp; fp16 and bf16.
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <optional>
#include <vector>

#include "api_common.h"

namespace {

int32_t dtype_of(const at::Tensor &q) {
    TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
                "differential attention needs float16 or bfloat16 tensors");
    return q.scalar_type() == at::kBFloat16 ? FA_BF16 : FA_FP16;
}

void check_like(const at::Tensor &t, const at::Tensor &q, const char *name) {
    TORCH_CHECK(t.is_cuda() && t.device() == q.device(), name, " must be on the device of q");
    TORCH_CHECK(t.scalar_type() == q.scalar_type(), name, " must have the dtype of q");
}

void check_int32(const at::Tensor &t, const at::Tensor &q, const char *name) {
    TORCH_CHECK(t.device() == q.device(), name, " must be on the device of q");
    TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be an int32 tensor");
}

// Sizes of q against k and v, whose leading sizes (batch and rows, or rows) are theirs.
void check_heads(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA (HIP) tensor");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
    TORCH_CHECK(q.size(-1) == k.size(-1), "q/k/v head_dim must match");
    TORCH_CHECK(k.size(-2) > 0 && q.size(-2) > 0 && q.size(-2) % k.size(-2) == 0,
                "num_heads_q must be divisible by num_heads_k for GQA/MQA");
    check_supported_head_dim(q.size(-1));
    check_like(k, q, "k");
    check_like(v, q, "v");
}

// lam as the kernels read it: one value, one a head, or one for each row and head (the leading sizes of q).
fa_diff_lam lam_of(const at::Tensor &lam, const at::Tensor &q) {
    TORCH_CHECK(lam.device() == q.device(), "lam must be on the device of q");
    TORCH_CHECK(lam.scalar_type() == at::kFloat, "lam must be a float32 tensor");
    fa_diff_lam l{lam.data_ptr<float>(), 0, 0, 0};
    if (lam.dim() == 0) return l;
    const bool rows = lam.dim() == q.dim() - 1 && lam.sizes() == q.sizes().slice(0, q.dim() - 1);
    TORCH_CHECK(rows || (lam.dim() == 1 && lam.size(0) == q.size(-2)),
                "lam must be a scalar tensor, [nheads], or have the shape of q without head_dim");
    l.head_stride = lam.stride(-1);
    if (rows) {
        l.row_stride = lam.stride(-2);
        if (lam.dim() == 3) l.batch_stride = lam.stride(0);
    }
    return l;
}

// A gradient of lam (new and contiguous) as the kernels write it; its strides tell the kernels what they sum.
fa_diff_dlam dlam_of(const at::Tensor &dlam) {
    fa_diff_dlam l{dlam.data_ptr<float>(), 0, 0, 0};
    if (dlam.dim() >= 1) l.head_stride = 1;
    if (dlam.dim() >= 2) l.row_stride = std::max<int64_t>(dlam.size(-1), 1);
    if (dlam.dim() == 3) l.batch_stride = dlam.size(1) * dlam.size(2);
    return l;
}

// Rows further apart than the kernels' 32-bit tile offsets reach (8 M elements) are copied, as misaligned ones are.
constexpr int64_t kMostRowStride = int64_t(1) << 23;
bool rows_near(const at::Tensor &t) { return t.size(-3) <= 1 || t.stride(-3) <= kMostRowStride; }
at::Tensor usable(const at::Tensor &t) { return rows_near(t) ? aligned(t) : t.clone(at::MemoryFormat::Contiguous); }

struct Varlen {
    const at::Tensor *cu_q, *cu_k;
    int max_q, max_k;
};

void check_varlen(const Varlen &x, const at::Tensor &q) {
    check_int32(*x.cu_q, q, "cu_seqlens_q");
    check_int32(*x.cu_k, q, "cu_seqlens_k");
    TORCH_CHECK(x.cu_q->dim() == 1 && x.cu_k->dim() == 1 && x.cu_q->is_contiguous() && x.cu_k->is_contiguous(),
                "cu_seqlens_q/cu_seqlens_k must be contiguous rank-1 tensors");
    TORCH_CHECK(x.cu_q->numel() >= 2 && x.cu_k->numel() == x.cu_q->numel(),
                "cu_seqlens_q/cu_seqlens_k must have batch_size + 1 elements");
    TORCH_CHECK(x.max_q >= 0 && x.max_k >= 0, "max_seqlen_q/max_seqlen_k must be non-negative");
}

// Sizes of a dense (varlen NULL) or packed call.
template <class Args>
void set_sizes(Args &a, const at::Tensor &q, const at::Tensor &k, const Varlen *x) {
    if (x) {
        a.cu_seqlens_q = x->cu_q->data_ptr<int32_t>();
        a.cu_seqlens_k = x->cu_k->data_ptr<int32_t>();
        a.batch = i32(x->cu_q->numel() - 1, "batch_size");
        a.seqlen_q = x->max_q;
        a.seqlen_k = x->max_k;
    } else {
        a.batch = i32(q.size(0), "batch_size");
        a.seqlen_q = i32(q.size(1), "seqlen_q");
        a.seqlen_k = i32(k.size(1), "seqlen_k");
    }
    a.lse_seqlen = a.seqlen_q;
    a.nheads = i32(q.size(-2), "num_heads");
    a.nheads_k = i32(k.size(-2), "num_heads_k");
    a.head_dim = int32_t(q.size(-1));
    a.dtype = dtype_of(q);
}

// Whether no row sees a key: empty tensors, or maxima of 0, to which packed sequences are cut.
template <class Args>
bool no_pairs(const Args &a, const at::Tensor &q, const at::Tensor &k) {
    return q.numel() == 0 || k.numel() == 0 || a.seqlen_q == 0 || a.seqlen_k == 0;
}

// The descriptor of a rank-3 or rank-4 tensor; a size of 1 has no stride (torch leaves any number there).
fa_tensor desc(const at::Tensor &t) {
    fa_tensor d = t.dim() == 3 ? desc3(t) : desc4(t);
    const int64_t i = t.dim() - 3;
    if (i == 0 || t.size(0) == 1) d.batch_stride = 0;
    if (t.size(i) == 1) d.row_stride = 0;
    if (t.size(i + 1) == 1) d.head_stride = 0;
    return d;
}

std::vector<std::optional<at::Tensor>> run_fwd(at::Tensor q, at::Tensor k, at::Tensor v, const at::Tensor &lam,
                                               double softmax_scale, bool causal, bool save, const Varlen *x) {
    c10::DeviceGuard guard(q.device());
    fa_diff_fwd_args a{};
    set_sizes(a, q, k, x);
    a.lam = lam_of(lam, q);
    q = usable(q);
    k = usable(k);
    v = usable(v);
    at::Tensor out = at::empty(q.sizes(), q.options()), o2;
    if (save) o2 = at::empty(q.sizes(), q.options());
    at::Tensor lse = at::empty({2, a.batch, a.nheads, a.lse_seqlen}, q.options().dtype(at::kFloat));
    auto got = [&]() {
        return std::vector<std::optional<at::Tensor>>{out, save ? std::optional<at::Tensor>(o2) : std::nullopt, lse};
    };
    if (no_pairs(a, q, k)) {
        out.zero_();
        if (save) o2.zero_();
        lse.zero_();
        return got();
    }
    a.q = desc(q);
    a.k = desc(k);
    a.v = desc(v);
    a.o = desc(out);
    if (save) a.o2 = desc(o2);
    a.lse = lse.data_ptr<float>();
    a.softmax_scale = float(softmax_scale);
    a.causal = causal;
    at::Tensor order;
    if (x) {
        a.o_rows = i32(q.size(0), "total_q");
        a.k_rows = i32(k.size(0), "total_k");
        order = at::empty({int64_t(std::max<size_t>(fa_diff_fwd_order_len(&a), 1))}, x->cu_q->options());
        a.work_order = order.data_ptr<int32_t>();
    }
    check_rc(fa_diff_fwd(&a, current_stream()), "fa_diff_fwd");
    return got();
}

std::vector<std::optional<at::Tensor>> run_bwd(at::Tensor q, at::Tensor k, at::Tensor v, const at::Tensor &lam,
                                               at::Tensor out, at::Tensor o2, const at::Tensor &lse, at::Tensor dout,
                                               double softmax_scale, bool causal, bool need_dlam, const Varlen *x) {
    c10::DeviceGuard guard(q.device());
    for (auto *t : {&out, &o2, &dout}) {
        TORCH_CHECK(t->sizes() == q.sizes(), "out, o2 and dout must match q shape");
        check_like(*t, q, "out, o2 and dout");
    }
    fa_diff_bwd_args a{};
    set_sizes(a, q, k, x);
    a.lam = lam_of(lam, q);
    TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.dim() == 4 &&
                    lse.size(0) == 2 && lse.size(1) == a.batch && lse.size(2) == a.nheads && lse.size(3) == a.lse_seqlen,
                "lse must be a contiguous float32 tensor of shape [2, batch_size, nheads, seqlen_q]");
    q = usable(q);
    k = usable(k);
    v = usable(v);
    out = aligned(out);
    o2 = aligned(o2);
    dout = usable(dout);
    at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
               dv = at::empty(v.sizes(), v.options()), dlam;
    const bool none = no_pairs(a, q, k);
    if (need_dlam)  // packed rows of no sequence read 0
        dlam = none || (x && lam.dim() == 2) ? at::zeros(lam.sizes(), lam.options().memory_format(at::MemoryFormat::Contiguous))
                                             : at::empty(lam.sizes(), lam.options().memory_format(at::MemoryFormat::Contiguous));
    std::vector<std::optional<at::Tensor>> got{dq, dk, dv, need_dlam ? std::optional<at::Tensor>(dlam) : std::nullopt};
    if (none) {
        dq.zero_();
        dk.zero_();
        dv.zero_();
        return got;
    }
    a.q = desc(q);
    a.k = desc(k);
    a.v = desc(v);
    a.o = desc(out);
    a.o2 = desc(o2);
    a.dout = desc(dout);
    a.dq = desc(dq);
    a.dk = desc(dk);
    a.dv = desc(dv);
    if (need_dlam) a.dlam = dlam_of(dlam);
    a.lse = lse.data_ptr<float>();
    a.softmax_scale = float(softmax_scale);
    a.causal = causal;
    at::Tensor order;
    if (x) {
        a.dq_rows = i32(q.size(0), "total_q");
        a.dkv_rows = i32(k.size(0), "total_k");
        order = at::empty({int64_t(std::max<size_t>(fa_diff_bwd_order_len(&a), 1))}, x->cu_q->options());
        a.work_order = order.data_ptr<int32_t>();
    }
    // One allocation: the row planes and, where there is memory for it, the workspace of shared dK/dV items.
    a.dsum_bytes = int64_t(fa_diff_bwd_ws_bytes(&a));
    const int64_t split = int64_t(fa_diff_bwd_split_bytes(&a)), at_split = (a.dsum_bytes + 255) / 256 * 256;
    at::Tensor ws = split > 0 ? optional_workspace(at_split + split, q.options().dtype(at::kByte)) : at::Tensor();
    if (ws.defined()) {
        a.split_ws = static_cast<char *>(ws.data_ptr()) + at_split;
        a.split_ws_bytes = split;
    } else {
        ws = at::empty({a.dsum_bytes}, q.options().dtype(at::kByte));
    }
    a.dsum = static_cast<float *>(ws.data_ptr());
    check_rc(fa_diff_bwd(&a, current_stream()), "fa_diff_bwd");
    return got;
}

void check_dense(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v) {
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be rank-4 tensors");
    TORCH_CHECK(k.size(0) == q.size(0), "k/v batch size must match q");
    check_heads(q, k, v);
}

void check_packed(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const Varlen &x) {
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k, v must be rank-3 packed tensors");
    check_heads(q, k, v);
    check_varlen(x, q);
}

std::vector<std::optional<at::Tensor>> diff_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor lam,
                                                double softmax_scale, bool causal, bool save) {
    check_dense(q, k, v);
    return run_fwd(q, k, v, lam, softmax_scale, causal, save, nullptr);
}

std::vector<std::optional<at::Tensor>> diff_bwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor lam, at::Tensor out,
                                                at::Tensor o2, at::Tensor lse, at::Tensor dout, double softmax_scale,
                                                bool causal, bool need_dlam) {
    check_dense(q, k, v);
    return run_bwd(q, k, v, lam, out, o2, lse, dout, softmax_scale, causal, need_dlam, nullptr);
}

std::vector<std::optional<at::Tensor>> diff_varlen_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor lam,
                                                       at::Tensor cu_q, at::Tensor cu_k, int max_q, int max_k,
                                                       double softmax_scale, bool causal, bool save) {
    const Varlen x{&cu_q, &cu_k, max_q, max_k};
    check_packed(q, k, v, x);
    return run_fwd(q, k, v, lam, softmax_scale, causal, save, &x);
}

std::vector<std::optional<at::Tensor>> diff_varlen_bwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor lam,
                                                       at::Tensor out, at::Tensor o2, at::Tensor lse, at::Tensor dout,
                                                       at::Tensor cu_q, at::Tensor cu_k, int max_q, int max_k,
                                                       double softmax_scale, bool causal, bool need_dlam) {
    const Varlen x{&cu_q, &cu_k, max_q, max_k};
    check_packed(q, k, v, x);
    return run_bwd(q, k, v, lam, out, o2, lse, dout, softmax_scale, causal, need_dlam, &x);
}

// A cache is written in place, so it is never copied: its layout has to suit the kernels.
void check_cache(const at::Tensor &c, const at::Tensor &q, const char *name) {
    check_like(c, q, name);
    TORCH_CHECK(c.dim() == 4, name, " must be a rank-4 tensor");
    TORCH_CHECK(is_aligned(c), name, " must have a contiguous last dimension and 16-byte aligned rows");
    TORCH_CHECK(rows_near(c), name, " must have tokens at most 2^23 elements apart");
}

std::vector<at::Tensor> diff_fwd_kvcache(at::Tensor q, at::Tensor k_cache, at::Tensor v_cache, at::Tensor lam,
                                         std::optional<at::Tensor> k_, std::optional<at::Tensor> v_,
                                         at::Tensor cache_seqlens, std::optional<at::Tensor> cache_batch_idx,
                                         std::optional<at::Tensor> block_table, double softmax_scale, bool causal,
                                         int num_splits, std::optional<at::Tensor> status) {
    TORCH_CHECK(q.dim() == 4, "q must be a rank-4 tensor");
    check_cache(k_cache, q, "k_cache");
    check_cache(v_cache, q, "v_cache");
    check_heads(q, k_cache, v_cache);
    const int64_t batch = q.size(0), seqlen_q = q.size(1);
    check_int32(cache_seqlens, q, "cache_seqlens");
    TORCH_CHECK(cache_seqlens.dim() == 1 && cache_seqlens.size(0) == batch && cache_seqlens.is_contiguous(),
                "cache_seqlens must be contiguous of shape [batch_size]");
    TORCH_CHECK(num_splits >= 0, "num_splits must be non-negative");
    TORCH_CHECK(k_.has_value() == v_.has_value(), "k and v must either both be provided or both be None");
    c10::DeviceGuard guard(q.device());
    fa_diff_kvcache_args a{};
    a.dtype = dtype_of(q);
    a.lam = lam_of(lam, q);
    q = aligned(q);
    at::Tensor k, v;
    if (k_.has_value()) {
        k = aligned(*k_);
        v = aligned(*v_);
        TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == batch && k.size(2) == k_cache.size(2) &&
                        k.size(3) == k_cache.size(3),
                    "k and v must have shape [batch_size, seqlen_new, nheads_k, head_dim]");
        check_like(k, q, "k");
        check_like(v, q, "v");
        a.seqlen_new = i32(k.size(1), "seqlen_new");
        if (a.seqlen_new > 0) {
            a.k_new = desc(k);
            a.v_new = desc(v);
        }
    }
    if (cache_batch_idx.has_value()) {
        check_int32(*cache_batch_idx, q, "cache_batch_idx");
        TORCH_CHECK(!block_table.has_value(), "Paged KV cache does not support cache_batch_idx");
        TORCH_CHECK(cache_batch_idx->dim() == 1 && cache_batch_idx->size(0) == batch && cache_batch_idx->is_contiguous(),
                    "cache_batch_idx must be contiguous of shape [batch_size]");
        a.cache_batch_idx = cache_batch_idx->data_ptr<int32_t>();
    }
    if (block_table.has_value()) {
        check_int32(*block_table, q, "block_table");
        TORCH_CHECK(block_table->dim() == 2 && block_table->size(0) == batch &&
                        (block_table->stride(1) == 1 || block_table->size(1) <= 1),
                    "block_table must have shape [batch_size, max_num_blocks_per_seq]");
        TORCH_CHECK(k_cache.size(1) > 0 && k_cache.size(1) % 64 == 0, "Paged KV cache block size must be divisible by 64");
        a.block_table = block_table->data_ptr<int32_t>();
        a.block_table_stride = block_table->stride(0);
        a.page_block_size = i32(k_cache.size(1), "page_block_size");
        a.num_pages = i32(k_cache.size(0), "num_blocks");
        a.cache_capacity = i32(block_table->size(1) * k_cache.size(1), "cache capacity");
    } else {
        TORCH_CHECK(cache_batch_idx.has_value() || k_cache.size(0) == batch, "k_cache batch size must match q");
        a.cache_capacity = i32(k_cache.size(1), "cache capacity");
        a.cache_batch = i32(k_cache.size(0), "cache batch");
    }
    if (status.has_value()) {
        check_int32(*status, q, "status");
        a.status = status->data_ptr<int32_t>();
    }
    at::Tensor out = at::empty(q.sizes(), q.options());
    at::Tensor lse = at::empty({2, batch, q.size(2), seqlen_q}, q.options().dtype(at::kFloat));
    if (batch == 0 || (q.numel() == 0 && a.seqlen_new == 0)) return {out, lse};
    if (k_cache.numel() == 0) {
        TORCH_CHECK(a.seqlen_new == 0, "cache capacity is insufficient for the requested append length");
        out.zero_();
        lse.zero_();
        return {out, lse};
    }
    a.q = desc(q);
    a.o = desc(out);
    a.k_cache = desc(k_cache);
    a.v_cache = desc(v_cache);
    a.lse = lse.data_ptr<float>();
    a.cache_seqlens = cache_seqlens.data_ptr<int32_t>();
    a.batch = i32(batch, "batch_size");
    a.seqlen_q = i32(seqlen_q, "seqlen_q");
    a.nheads = i32(q.size(2), "num_heads");
    a.nheads_k = i32(k_cache.size(2), "num_heads_k");
    a.head_dim = int32_t(q.size(3));
    a.num_splits = num_splits;
    a.softmax_scale = float(softmax_scale);
    a.causal = causal;
    at::Tensor ws;
    a.ws_bytes = int64_t(fa_diff_kvcache_ws_bytes(&a));
    if (a.ws_bytes > 0) {
        ws = at::empty({a.ws_bytes}, q.options().dtype(at::kByte));
        a.ws = ws.data_ptr();
    }
    check_rc(fa_diff_kvcache(&a, current_stream()), "fa_diff_kvcache");
    return {out, lse};
}

}  // namespace

void bind_diff(py::module_ &m) {
    m.def("diff_fwd", &diff_fwd, "Differential attention forward pass");
    m.def("diff_bwd", &diff_bwd, "Differential attention backward pass");
    m.def("diff_varlen_fwd", &diff_varlen_fwd, "Differential attention varlen forward pass");
    m.def("diff_varlen_bwd", &diff_varlen_bwd, "Differential attention varlen backward pass");
    m.def("diff_fwd_kvcache", &diff_fwd_kvcache, "Differential attention with a KV cache");
}
