// Shared by the extension's sources: checks and descriptors of tensors for the C ABI.
#pragma once

#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <cstdint>

#include "fa_mi355x.h"

inline void check_supported_head_dim(const int64_t head_size) {
    TORCH_CHECK(head_size == 64 || head_size == 128, "Turing FlashAttention supports head_dim 64 or 128");
}

inline void check_fp16_cuda(const at::Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA (HIP) tensor");
    TORCH_CHECK(t.scalar_type() == at::kHalf, name, " must be a float16 tensor");
}

// 16-byte aligned base and strides (in elements, multiple of 8), last dim contiguous.
inline bool is_aligned(const at::Tensor &t) {
    bool ok = t.stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
    for (int64_t i = 0; ok && i + 1 < t.dim(); ++i) ok = (t.stride(i) % 8) == 0 || t.size(i) == 1;
    return ok;
}
// A fresh contiguous copy when not (contiguous() alone would keep a misaligned base).
inline at::Tensor aligned(const at::Tensor &t) { return is_aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

inline fa_tensor desc4(const at::Tensor &t) {  // [batch][row][head][d]
    return fa_tensor{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
inline fa_tensor desc3(const at::Tensor &t) {  // packed [total][head][d]
    return fa_tensor{t.data_ptr(), 0, t.stride(0), t.stride(1)};
}

// Sizes go to the kernels as int32 (their index math is 64-bit where products can overflow).
inline int32_t i32(int64_t v, const char *what) {
    TORCH_CHECK(v >= 0 && v <= INT32_MAX, what, " must be below 2^31");
    return int32_t(v);
}

inline hipStream_t current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

inline void check_rc(int rc, const char *what) {
    TORCH_CHECK(rc == FA_OK, what, " failed: ", fa_error_string(rc));
}

// A workspace that a call is faster with but can do without: undefined where the
// device has no memory left for it.
inline at::Tensor optional_workspace(int64_t numel, const at::TensorOptions &options) {
    try {
        return at::empty({numel}, options);
    } catch (const c10::OutOfMemoryError &) {
        return at::Tensor();
    }
}

// Bindings of the extension's other sources.
void bind_diff(py::module_ &m);     // diff_api.cpp
void bind_kvpages(py::module_ &m);  // kvpages_api.cpp
void bind_rotary(py::module_ &m);   // rotary_api.cpp
void bind_kv8(py::module_ &m);      // kv8_api.cpp
