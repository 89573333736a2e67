// Bindings of rotary positions: rotary_tables and rotary over fa_rotary_tables and fa_rotary.
#include <c10/core/DeviceGuard.h>

#include <optional>
#include <vector>

#include "api_common.h"

namespace {

int32_t rotary_dtype(const at::ScalarType t) { return t == at::kHalf ? FA_FP16 : t == at::kBFloat16 ? FA_BF16 : FA_FP32; }

void check_int32(const std::optional<at::Tensor> &t, const at::Tensor &q, const char *name) {
    if (!t.has_value()) return;
    TORCH_CHECK(t->device() == q.device(), name, " must be on the device of q");
    TORCH_CHECK(t->scalar_type() == at::kInt, name, " must be an int32 tensor");
}

// A size of 1 has no stride (torch leaves any number there).
fa_tensor desc(const at::Tensor &t) {
    fa_tensor d = t.dim() == 3 ? desc3(t) : desc4(t);
    const int64_t i = t.dim() - 3;
    if (i == 0 || t.size(0) == 1) d.batch_stride = 0;
    if (t.size(i) == 1) d.row_stride = 0;
    if (t.size(i + 1) == 1) d.head_stride = 0;
    return d;
}

std::vector<std::optional<at::Tensor>> rotary(at::Tensor q, std::optional<at::Tensor> k_, at::Tensor cos, at::Tensor sin,
                                              bool interleaved, std::optional<at::Tensor> positions,
                                              std::optional<at::Tensor> offsets, int64_t offset,
                                              std::optional<at::Tensor> cu, bool inverse) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA (HIP) tensor");
    TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
                "rotary positions need float16 or bfloat16 tensors");
    const bool packed = cu.has_value();
    const int64_t rank = packed ? 3 : 4;
    TORCH_CHECK(q.dim() == rank && (!k_.has_value() || k_->dim() == rank), "q and k must be rank-", rank, " tensors");
    check_supported_head_dim(q.size(-1));
    c10::DeviceGuard guard(q.device());
    fa_rotary_args a{};
    if (k_.has_value()) {
        TORCH_CHECK(k_->device() == q.device() && k_->scalar_type() == q.scalar_type(), "k must have the device and dtype of q");
        TORCH_CHECK(k_->sizes().slice(0, rank - 2) == q.sizes().slice(0, rank - 2) && k_->size(-1) == q.size(-1),
                    "k must have the shape of q, its number of heads apart");
    }
    for (const auto *t : {&cos, &sin}) {
        TORCH_CHECK(t->device() == q.device() && t->dim() == 2, "rotary_cos and rotary_sin must be rank-2 tensors on the device of q");
        TORCH_CHECK(t->scalar_type() == cos.scalar_type() && t->sizes() == cos.sizes(), "rotary_cos and rotary_sin must match");
    }
    TORCH_CHECK(cos.scalar_type() == at::kFloat || cos.scalar_type() == at::kHalf || cos.scalar_type() == at::kBFloat16,
                "rotary_cos and rotary_sin must be float32, float16 or bfloat16 tensors");
    const int64_t rotary_dim = 2 * cos.size(1);
    TORCH_CHECK(rotary_dim > 0 && rotary_dim % 16 == 0 && rotary_dim <= q.size(-1),
                "rotary_dim must be a multiple of 16 up to head_dim");
    TORCH_CHECK(cos.size(0) > 0, "rotary_cos and rotary_sin must have a row");
    check_int32(positions, q, "positions");
    check_int32(offsets, q, "seqlen_offsets");
    check_int32(cu, q, "cu_seqlens");
    TORCH_CHECK(offset >= INT32_MIN && offset <= INT32_MAX, "seqlen_offsets must fit in 32 bits");
    if (packed) {
        TORCH_CHECK(cu->dim() == 1 && cu->numel() >= 2 && cu->is_contiguous(), "cu_seqlens must be contiguous with batch_size + 1 elements");
        a.cu_seqlens = cu->data_ptr<int32_t>();
        a.batch = i32(cu->numel() - 1, "batch_size");
        a.seqlen = i32(q.size(0), "total");
    } else {
        a.batch = i32(q.size(0), "batch_size");
        a.seqlen = i32(q.size(1), "seqlen");
    }
    at::Tensor pos;
    if (positions.has_value()) {
        TORCH_CHECK(!offsets.has_value() && offset == 0, "positions and seqlen_offsets exclude each other");
        TORCH_CHECK(positions->sizes() == q.sizes().slice(0, rank - 2), "positions must have the leading shape of q");
        pos = *positions;
        if (pos.stride(-1) != 1) pos = pos.contiguous();
        a.positions = pos.data_ptr<int32_t>();
        a.positions_stride = packed ? 0 : pos.stride(0);
    }
    if (offsets.has_value()) {
        TORCH_CHECK(offsets->dim() == 1 && offsets->size(0) == a.batch && offsets->is_contiguous(),
                    "seqlen_offsets must be an int or contiguous of shape [batch_size]");
        a.seqlen_offsets = offsets->data_ptr<int32_t>();
    }
    q = aligned(q);
    at::Tensor k, q_out = at::empty(q.sizes(), q.options()), k_out;
    if (k_.has_value()) {
        k = aligned(*k_);
        k_out = at::empty(k.sizes(), k.options());
    }
    std::vector<std::optional<at::Tensor>> got{q_out, k_.has_value() ? std::optional<at::Tensor>(k_out) : std::nullopt};
    if (q.numel() == 0 && (!k_.has_value() || k.numel() == 0)) return got;
    cos = aligned(cos);
    sin = aligned(sin);
    if (q.numel() > 0) {
        a.q = desc(q);
        a.q_out = desc(q_out);
        a.nheads = i32(q.size(-2), "num_heads");
    }
    if (k_.has_value() && k.numel() > 0) {
        a.k = desc(k);
        a.k_out = desc(k_out);
        a.nheads_k = i32(k.size(-2), "num_heads_k");
    }
    a.cos = cos.data_ptr();
    a.sin = sin.data_ptr();
    a.cos_stride = cos.size(0) == 1 ? 0 : cos.stride(0);
    a.sin_stride = sin.size(0) == 1 ? 0 : sin.stride(0);
    a.head_dim = int32_t(q.size(-1));
    a.rotary_dim = int32_t(rotary_dim);
    a.table_rows = i32(cos.size(0), "rows of rotary_cos");
    a.offset = int32_t(offset);
    a.interleaved = interleaved;
    a.inverse = inverse;
    a.dtype = rotary_dtype(q.scalar_type());
    a.table_dtype = rotary_dtype(cos.scalar_type());
    check_rc(fa_rotary(&a, current_stream()), "fa_rotary");
    return got;
}

// cos and sin: contiguous tensors that the caller made.
void rotary_tables(at::Tensor cos, at::Tensor sin, int64_t offset, double base, double factor, double original_seqlen,
                   double low_turns, double high_turns, double attention_factor) {
    TORCH_CHECK(cos.is_cuda(), "rotary tables are made on a CUDA (HIP) device");
    TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.device() == sin.device() &&
                    cos.scalar_type() == sin.scalar_type() && cos.is_contiguous() && sin.is_contiguous(),
                "cos and sin must be contiguous and match");
    TORCH_CHECK(cos.scalar_type() == at::kFloat || cos.scalar_type() == at::kHalf || cos.scalar_type() == at::kBFloat16,
                "rotary tables must be float32, float16 or bfloat16");
    c10::DeviceGuard guard(cos.device());
    fa_rotary_tables_args a{};
    a.cos = cos.data_ptr();
    a.sin = sin.data_ptr();
    a.seqlen = i32(cos.size(0), "seqlen");
    a.rotary_dim = i32(2 * cos.size(1), "rotary_dim");
    a.dtype = rotary_dtype(cos.scalar_type());
    a.offset = offset;
    a.base = base;
    a.factor = factor;
    a.original_seqlen = original_seqlen;
    a.low_turns = low_turns;
    a.high_turns = high_turns;
    a.attention_factor = attention_factor;
    check_rc(fa_rotary_tables(&a, current_stream()), "fa_rotary_tables");
}

}  // namespace

void bind_rotary(py::module_ &m) {
    m.def("rotary", &rotary, "Rotary positions of q and k");
    m.def("rotary_tables", &rotary_tables, "Cosines and sines of rotary angles");
}
