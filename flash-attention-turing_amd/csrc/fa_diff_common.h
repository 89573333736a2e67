// Shared by the differential attention kernels: 16-bit types and the work of a call.
//
// One head of differential attention holds two maps in the two halves of q's
// and k's channels (q = [q1 | q2], k = [k1 | k2], head_dim / 2 each) and one
// value head of head_dim channels:
//   o = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v.
// q, k, v and o so have the shapes and the LDS tiles of ordinary attention of
// that head_dim; an MFMA K step of the first half of the channels belongs to
// map 1, of the second half to map 2.
#pragma once

#include "fa_common.h"

namespace fa {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// fp16 or bf16 (BF) data travels as f16x8 bits; only the products and the
// conversions know the type.
template <bool BF>
__device__ __forceinline__ f32x16 mfma16(const f16x8 a, const f16x8 b, const f32x16 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f16x8 pack16(const f32x16 &acc, int base) {
    if constexpr (BF) {
        bf16x8 r;
#pragma unroll
        for (int t = 0; t < 8; ++t) r[t] = (__bf16)acc[base + t];
        return __builtin_bit_cast(f16x8, r);
    } else {
        return pack8(acc, base);
    }
}
template <bool BF>
__device__ __forceinline__ f16x4 pack4(float a, float b, float c, float d) {
    if constexpr (BF)
        return __builtin_bit_cast(f16x4, bf16x4{(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d});
    else
        return f16x4{(f16)a, (f16)b, (f16)c, (f16)d};
}
template <bool BF>
__device__ __forceinline__ float elem(const f16x8 v, int i) {
    if constexpr (BF)
        return float(__builtin_bit_cast(bf16x8, v)[i]);
    else
        return float(v[i]);
}

// lam of (batch, row of the tensor, head); strides in elements, 0 where it is shared.
__device__ __forceinline__ float diff_lam(const fa_diff_lam &l, int b, int64_t row, int h) {
    return l.ptr[int64_t(b) * l.batch_stride + row * l.row_stride + int64_t(h) * l.head_stride];
}

// A wave-uniform int32 of memory that no kernel in flight writes, through the
// scalar cache: a vector load would wait for the tile copies that are in flight.
__device__ __forceinline__ int scalar_load(const int32_t *p) {
    const uint64_t u = reinterpret_cast<uint64_t>(p);
    // (The builtin returns an int: widened as it is, a low half from 2^31 on would set all of the high half.)
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(u)), hi = __builtin_amdgcn_readfirstlane(uint32_t(u >> 32));
    const uint64_t s = uint64_t(hi) << 32 | lo;
    int v;
    asm volatile("s_load_dword %0, %1, 0x0\n\ts_waitcnt lgkmcnt(0)" : "=s"(v) : "s"(s) : "memory");
    return v;
}

// Page at table entry pg of sequence b, checked: one outside the cache becomes
// page 0 and is reported, so that no access leaves the cache.
__device__ __forceinline__ int checked_page(const int32_t *table, int64_t stride, int b, int pg, int num_pages,
                                            int32_t *status) {
    const int blk = scalar_load(table + int64_t(b) * stride + pg);
    if (blk >= 0 && blk < num_pages) return blk;
    if (status && (threadIdx.x & 63) == 0) atomicOr(status, FA_KV_BAD_PAGE);
    return 0;
}

}  // namespace fa
