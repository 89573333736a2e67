// Bindings of the calls on the pages of a KV cache (fa_kvpages_*).
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <optional>
#include <tuple>
#include <utility>
#include <vector>

#include "api_common.h"

namespace {

void check_ints(const at::Tensor &t, const at::Device &device, int64_t dim, const char *name) {
    TORCH_CHECK(t.is_cuda() && t.device() == device, name, " must be on the device of the cache");
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim && (t.numel() == 0 || dim == 0 || t.stride(-1) == 1 || t.size(-1) == 1),
                name, " must be an int32 tensor of rank ", dim, " with a contiguous last dimension");
}

// Whether two of a cache's elements may share a place: of the sizes over 1, in the order of their strides, each
// stride has to pass what those before it span, as in any slice and order of a dense tensor.  Tokens or heads that a
// stride of 0 repeats within a page are one place.
bool may_overlap(const at::Tensor &c) {
    std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
    for (int64_t i = 0; i < c.dim(); ++i)
        if (c.size(i) > 1 && (i == 0 || c.stride(i) != 0)) dims.emplace_back(c.stride(i), c.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t span = 1;
    for (const auto &[stride, size] : dims) {
        if (stride < span) return true;
        span += (size - 1) * stride;
    }
    return false;
}

int32_t *ints(const std::optional<at::Tensor> &t) { return t.has_value() ? t->data_ptr<int32_t>() : nullptr; }

struct Call {
    fa_kvpages_args a{};
    at::Tensor ws;
    at::Device device;
    explicit Call(const at::Device &d, const std::optional<at::Tensor> &status) : device(d) {
        if (status.has_value()) {
            check_ints(*status, device, 1, "status");
            a.status = status->data_ptr<int32_t>();
        }
    }
    fa_tensor pages(const at::Tensor &c, const at::Tensor &like, const char *name) const {
        TORCH_CHECK(c.is_cuda() && c.device() == device && c.dim() == 4, name,
                    " must be a rank-4 CUDA (HIP) tensor [num_blocks, page_block_size, nheads_k, head_dim]");
        TORCH_CHECK(c.sizes() == like.sizes() && c.scalar_type() == like.scalar_type(), "k_cache and v_cache must match");
        const int64_t e = c.element_size();
        TORCH_CHECK(c.numel() > 0 && c.size(3) * e % 16 == 0 && (c.stride(3) == 1 || c.size(3) == 1) &&
                        c.stride(0) * e % 16 == 0 && c.stride(1) * e % 16 == 0 && c.stride(2) * e % 16 == 0 &&
                        (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0,
                    name, " must have a contiguous last dimension and 16-byte aligned rows");
        TORCH_CHECK(!may_overlap(c), "pages of ", name, " must not overlap");
        return fa_tensor{c.data_ptr(), c.stride(0) * e, c.stride(1) * e, c.stride(2) * e};
    }
    void cache(const at::Tensor &k, const at::Tensor &v) {
        a.k_cache = pages(k, k, "k_cache");
        a.v_cache = pages(v, k, "v_cache");
        a.num_pages = i32(k.size(0), "num_blocks");
        a.page_block_size = i32(k.size(1), "page_block_size");
        a.nheads_k = i32(k.size(2), "nheads_k");
        a.head_bytes = i32(k.size(3) * k.element_size(), "head_dim");
    }
    void table(const at::Tensor &t, const std::optional<at::Tensor> &lens, const at::Tensor &refs) {
        check_ints(t, device, 2, "block_table");
        check_ints(refs, device, 1, "page_refs");
        TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), "rows of block_table must not overlap");
        TORCH_CHECK(a.num_pages == 0 || refs.size(0) == a.num_pages, "page_refs must have one entry a page");
        a.num_pages = i32(refs.size(0), "num_blocks");
        a.block_table = t.data_ptr<int32_t>();
        a.block_table_stride = t.stride(0);
        a.rows = i32(t.size(0), "rows");
        a.max_pages = i32(t.size(1), "max_num_blocks_per_seq");
        a.page_refs = refs.data_ptr<int32_t>();
        if (lens.has_value()) {
            check_ints(*lens, device, 1, "cache_seqlens");
            TORCH_CHECK(lens->size(0) == t.size(0), "cache_seqlens must have one entry a row of block_table");
            a.cache_seqlens = lens->data_ptr<int32_t>();
        }
    }
    void list(const at::Tensor &from, const std::optional<at::Tensor> &to, const char *from_name, const char *to_name) {
        check_ints(from, device, 1, from_name);
        a.from = from.data_ptr<int32_t>();
        a.n = i32(from.size(0), from_name);
        if (to.has_value()) {
            check_ints(*to, device, 1, to_name);
            TORCH_CHECK(to->size(0) == from.size(0), from_name, " and ", to_name, " must have the same length");
            a.to = to->data_ptr<int32_t>();
        }
    }
    void workspace() {
        a.ws_bytes = int64_t(fa_kvpages_ws_bytes(&a));
        ws = at::empty({a.ws_bytes / 4}, at::TensorOptions().device(device).dtype(at::kInt));
        a.ws = ws.data_ptr();
    }
};

void pages_copy(at::Tensor k_cache, at::Tensor v_cache, at::Tensor src, at::Tensor dst, std::optional<at::Tensor> status) {
    Call c(k_cache.device(), status);
    c.cache(k_cache, v_cache);
    c.list(src, dst, "src", "dst");
    c10::DeviceGuard guard(c.device);
    check_rc(fa_kvpages_copy(&c.a, current_stream()), "fa_kvpages_copy");
}

void pages_alloc(at::Tensor block_table, at::Tensor cache_seqlens, at::Tensor page_refs, int64_t seqlen_new,
                 std::optional<at::Tensor> seqlens_new, int64_t page_block_size, std::optional<at::Tensor> status) {
    Call c(block_table.device(), status);
    c.table(block_table, cache_seqlens, page_refs);
    c.a.page_block_size = i32(page_block_size, "page_block_size");
    c.a.seqlen_new = i32(seqlen_new, "seqlen_new");
    if (seqlens_new.has_value()) {
        check_ints(*seqlens_new, c.device, 1, "seqlen_new");
        TORCH_CHECK(seqlens_new->size(0) == block_table.size(0), "seqlen_new must have one entry a row of block_table");
        c.a.seqlens_new = ints(seqlens_new);
    }
    if (block_table.size(0) == 0) return;
    c10::DeviceGuard guard(c.device);
    c.workspace();
    check_rc(fa_kvpages_alloc(&c.a, current_stream()), "fa_kvpages_alloc");
}

void pages_fork(at::Tensor k_cache, at::Tensor v_cache, at::Tensor block_table, at::Tensor cache_seqlens,
                at::Tensor page_refs, at::Tensor parents, at::Tensor children, std::optional<at::Tensor> status) {
    Call c(k_cache.device(), status);
    c.cache(k_cache, v_cache);
    c.table(block_table, cache_seqlens, page_refs);
    c.list(parents, children, "parents", "children");
    if (c.a.n == 0) return;
    c10::DeviceGuard guard(c.device);
    c.workspace();
    check_rc(fa_kvpages_fork(&c.a, current_stream()), "fa_kvpages_fork");
}

void pages_free(at::Tensor block_table, at::Tensor cache_seqlens, at::Tensor page_refs, at::Tensor rows,
                std::optional<at::Tensor> status) {
    Call c(block_table.device(), status);
    c.table(block_table, cache_seqlens, page_refs);
    c.a.page_block_size = 1;  // not looked at
    c.list(rows, std::nullopt, "rows", "");
    if (c.a.n == 0) return;
    c10::DeviceGuard guard(c.device);
    check_rc(fa_kvpages_free(&c.a, current_stream()), "fa_kvpages_free");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> pages_compact(at::Tensor k_cache, at::Tensor v_cache, at::Tensor block_table,
                                                             at::Tensor page_refs) {
    Call c(k_cache.device(), std::nullopt);
    c.cache(k_cache, v_cache);
    c.table(block_table, std::nullopt, page_refs);
    c10::DeviceGuard guard(c.device);
    at::Tensor table = at::empty(block_table.sizes(), block_table.options()),
               refs = at::empty(page_refs.sizes(), page_refs.options()), used = at::empty({1}, page_refs.options());
    c.a.out_table = table.data_ptr<int32_t>();
    c.a.out_table_stride = table.stride(0);
    c.a.out_refs = refs.data_ptr<int32_t>();
    c.a.out_used = used.data_ptr<int32_t>();
    c.workspace();
    check_rc(fa_kvpages_compact(&c.a, current_stream()), "fa_kvpages_compact");
    return {table, refs, used};
}

}  // namespace

void bind_kvpages(py::module_ &m) {
    m.def("kvpages_copy", &pages_copy, "Copy pages of a KV cache");
    m.def("kvpages_alloc", &pages_alloc, "Give rows of a paged KV cache pages for new tokens");
    m.def("kvpages_fork", &pages_fork, "Fork rows of a paged KV cache");
    m.def("kvpages_free", &pages_free, "Give back the pages of rows of a paged KV cache");
    m.def("kvpages_compact", &pages_compact, "Move the used pages of a KV cache to its front");
}
