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

// max(a, b, c) in one instruction and without the canonicalisation of each
// operand that fmaxf adds.  A NaN among them is passed over, as by fmaxf.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// max_xor32 (fa_common.h) without the canonicalisations.
__device__ __forceinline__ float max2_xor32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    return max3(a, b, b);
}
// A wave-uniform float in a scalar register.
__device__ __forceinline__ float uniform(float x) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}

// Rows of sequence b of a dense or packed call.  A packed sequence is cut to the
// call's maximum length, on which the LSE's rows, the grids and the work orders
// go, and to the rows that its tensor has (rows; 0: not known), so that no access
// leaves a tensor whatever cu holds.
struct DiffRows {
    int start, n;
};
__device__ __forceinline__ DiffRows diff_rows(const int32_t *cu, int b, int seqlen, int rows) {
    DiffRows r{0, seqlen};
    if (cu) {
        const int most = rows > 0 ? rows : INT_MAX;
        r.start = min(max(cu[b], 0), most);
        r.n = min(max(min(cu[b + 1], most) - r.start, 0), seqlen);
    }
    return r;
}

// lam of (batch, row of the tensor, head); strides in elements, 0 where it is shared.
__device__ __forceinline__ float diff_lam(const fa_diff_lam &l, int b, int64_t row, int h) {
    return l.ptr[int64_t(b) * l.batch_stride + row * l.row_stride + int64_t(h) * l.head_stride];
}

// A wave-uniform address as scalar registers.  (The builtin returns an int:
// widened as it is, a low half from 2^31 on would set all of the high half.)
template <class T>
__device__ __forceinline__ const T *uniform(const T *p) {
    const uint64_t u = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(u)), hi = __builtin_amdgcn_readfirstlane(uint32_t(u >> 32));
    return reinterpret_cast<const T *>(uint64_t(hi) << 32 | lo);
}

// A wave-uniform int32 of memory that no kernel in flight writes, through the
// scalar cache: a vector load would wait for the tile copies that are in flight.
__device__ __forceinline__ int scalar_load(const int32_t *p) {
    int v;
    asm volatile("s_load_dword %0, %1, 0x0\n\ts_waitcnt lgkmcnt(0)" : "=s"(v) : "s"(uniform(p)) : "memory");
    return v;
}

// The same through the compiler, which waits where the value is used; for memory
// that nothing writes while the kernel runs.
__device__ __forceinline__ int scalar_load_ahead(const int32_t *p) {
    return *(const __attribute__((address_space(4))) int32_t *)uniform(p);
}

// g2l16 (fa_common.h) with the address as a wave-uniform base and a 32-bit byte
// offset per lane: no 64-bit address is formed or held per lane and copy.  Same
// waiting rules.
__device__ __forceinline__ void g2l16_at(const f16 *base, uint32_t off, uint32_t l) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(off), "s"(base), "s"(l)
        : "memory");
}
// Row strides (elements) with which a tile's lane offsets, below 128 rows, stay
// under 2^32 bytes.
constexpr int64_t kDiffMaxRowStride = int64_t(1) << 23;

// Copies of a [ROWS][HD] tile by NT threads into the swizzled layout of
// TileCopier (fa_common.h), from a wave-uniform first row.  rows: how many there
// are; the rows past them re-read the last one.
template <int HD, int ROWS, int NT>
struct DiffCopier {
    static constexpr int KCH = HD / 8, CPT = ROWS * KCH / NT, WAVES = NT / 64, RSTEP = NT / KCH;
    static_assert(RSTEP % 16 == 0, "row step must keep the swizzle");
    uint32_t rc;  // the lane's row, and 16 times its swizzled chunk in the high half
    uint32_t lds0;
    __device__ __forceinline__ void init(int wave, int lane) {
        const int p = wave * 64 + lane, row = p / KCH;
        rc = row | ((p % KCH) ^ swz<KCH>(row)) << 20;
        lds0 = wave * 1024;
    }
    __device__ __forceinline__ void copy(uint32_t tile_l, const f16 *row0, int64_t rs, int rows) const {
        const uint32_t l0 = __builtin_amdgcn_readfirstlane(tile_l + lds0), rsb = uint32_t(rs) * 2;
        uint32_t x = rc;
        asm volatile("" : "+v"(x));  // the offsets are formed here, not held between copies
        row0 = uniform(row0);
        const uint32_t row = x & 0xffff, c = x >> 16;
        if (rows >= ROWS) {
            const uint32_t off = row * rsb + c;
#pragma unroll
            for (int i = 0; i < CPT; ++i) g2l16_at(row0 + i * RSTEP * rs, off, l0 + i * WAVES * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < CPT; ++i)
                g2l16_at(row0, min(int(row) + i * RSTEP, rows - 1) * rsb + c, l0 + i * WAVES * 1024);
        }
    }
};

// A table's entry, checked: a page outside the cache becomes page 0 and is
// reported, so that no access leaves the cache.
__device__ __forceinline__ int checked_page(int blk, int num_pages, int32_t *status) {
    const bool ok = blk >= 0 && blk < num_pages;
    if (!ok && status && (threadIdx.x & 63) == 0) atomicOr(status, FA_KV_BAD_PAGE);
    return __builtin_amdgcn_readfirstlane(ok ? blk : 0);
}

}  // namespace fa
