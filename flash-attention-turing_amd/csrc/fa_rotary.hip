// Rotary positions: tables of cosines and sines, and the rotation of q and k with its gradient.
//
// Pair (x1, x2) of a row at position p becomes (x1 c - x2 s, x2 c + x1 s) with c, s = cos, sin(p f_j): a rotation, so
// the gradient is the rotation by the opposite angle, and forward and backward are one kernel.  Six operations a pair
// against 8 bytes moved: memory bounds it.  16 packed texts of up to 4096 tokens, 32/8 heads of 128, bf16, half of the channels:
// forward and backward 200 us, 5.4 TB/s (a large copy 5.2); one text of 77 tokens 3.3 us a launch.
//
// A wave takes one row of q and k, all heads: the row's cosines and sines go to registers once (16 a lane) and serve
// every head, and each load or store of the wave covers whole 128-byte lines.
#include <algorithm>
#include <cmath>

#include "fa_diff_common.h"

namespace fa {

constexpr int kRtThreads = 256, kRtHeads = 4;  // heads a lane has in flight

template <bool BF>
__device__ __forceinline__ void rt_unpack(const u32x4 v, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = elem<BF>(as_h8(v), i);
}
template <bool BF>
__device__ __forceinline__ u32x4 rt_pack(const float (&x)[8]) {
    const f16x4 lo = pack4<BF>(x[0], x[1], x[2], x[3]), hi = pack4<BF>(x[4], x[5], x[6], x[7]);
    return __builtin_bit_cast(u32x4, f16x8(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)));
}

// N table entries from element i on, in fp32.
template <int N>
__device__ __forceinline__ void rt_table(const void *t, int64_t i, int dtype, float *x) {
    if (dtype == FA_FP32) {
        const float *p = static_cast<const float *>(t) + i;
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(p + k);
#pragma unroll
            for (int u = 0; u < 4; ++u) x[k + u] = v[u];
        }
        return;
    }
    const f16 *p = static_cast<const f16 *>(t) + i;
#pragma unroll
    for (int k = 0; k < N; k += 4) {
        const u32x2 v = *reinterpret_cast<const u32x2 *>(p + k);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t w = v[u / 2] >> (u % 2 * 16) & 0xffffu;
            x[k + u] = dtype == FA_BF16 ? __uint_as_float(w << 16) : float(__builtin_bit_cast(f16, uint16_t(w)));
        }
    }
}

// Lane (unit u of HD / 16, head) holds two 16-byte chunks of a head: in the half layout the two halves of 8 pairs,
// else chunks u and u + HD / 16, 4 pairs each; units past the rotated channels copy the chunks that are left.
template <int HD, bool BF, bool INTER>
__global__ __launch_bounds__(kRtThreads) void rotary_kernel(const fa_rotary_args a) {
    constexpr int U = HD / 16, HP = 64 / U;  // units of a head, heads of a wave at a time
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t rows = a.cu_seqlens ? a.seqlen : int64_t(a.batch) * a.seqlen;
    const int64_t r = int64_t(blockIdx.x) * (kRtThreads / 64) + wave;
    if (r >= rows) return;
    int b = 0, i = int(r), seq = 0;
    bool covered = true;
    if (a.cu_seqlens) {
        seq = packed_sequence(a.cu_seqlens, a.batch, i);
        covered = seq >= 0 && seq < a.batch;
    } else {
        b = seq = int(r / a.seqlen);
        i = int(r - int64_t(b) * a.seqlen);
    }
    int64_t pos;
    if (a.positions)
        pos = a.positions[int64_t(b) * a.positions_stride + i];
    else
        pos = int64_t(a.offset) + (a.seqlen_offsets && covered ? a.seqlen_offsets[seq] : 0) + i -
              (a.cu_seqlens && covered ? a.cu_seqlens[seq] : 0);
    const bool in_table = pos >= 0 && pos < a.table_rows;
    if (!in_table) pos = 0;

    const int u = lane % U, sub = lane / U, turned = a.rotary_dim / 16;
    int ca, cb;  // the chunks
    float c[8], s[8];
    if constexpr (INTER) {
        ca = u;
        cb = u + U;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int ch = k ? cb : ca;
            if (8 * ch < a.rotary_dim) {
                rt_table<4>(a.cos, pos * a.cos_stride + 4 * ch, a.table_dtype, c + 4 * k);
                rt_table<4>(a.sin, pos * a.sin_stride + 4 * ch, a.table_dtype, s + 4 * k);
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t) c[4 * k + t] = 1.f, s[4 * k + t] = 0.f;
            }
        }
    } else {
        ca = u < turned ? u : 2 * u;
        cb = u < turned ? turned + u : 2 * u + 1;
        if (u < turned) {
            rt_table<8>(a.cos, pos * a.cos_stride + 8 * u, a.table_dtype, c);
            rt_table<8>(a.sin, pos * a.sin_stride + 8 * u, a.table_dtype, s);
        }
    }
    // Chunks that are copied keep their bits; of a chunk pair in the interleaved layout each may be.
    const bool turn_a = INTER ? 8 * ca < a.rotary_dim : u < turned, turn_b = INTER ? 8 * cb < a.rotary_dim : u < turned;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        if (!in_table) c[t] = s[t] = __builtin_nanf("");
        if (a.inverse) s[t] = -s[t];
    }
    const int heads = a.nheads + a.nheads_k;
    auto place = [&](const fa_tensor &q, const fa_tensor &k, int h) FA_INLINE {
        const bool is_k = h >= a.nheads;
        const fa_tensor &t = is_k ? k : q;
        return (f16 *)t.ptr + int64_t(b) * t.batch_stride + int64_t(i) * t.row_stride +
               int64_t(is_k ? h - a.nheads : h) * t.head_stride;
    };
    for (int h0 = sub; h0 < heads; h0 += HP * kRtHeads) {
        u32x4 va[kRtHeads], vb[kRtHeads];
#pragma unroll
        for (int n = 0; n < kRtHeads; ++n)
            if (h0 + n * HP < heads) {
                const f16 *p = place(a.q, a.k, h0 + n * HP);
                va[n] = ldg16(p + 8 * ca);
                vb[n] = ldg16(p + 8 * cb);
            }
#pragma unroll
        for (int n = 0; n < kRtHeads; ++n) {
            if (h0 + n * HP >= heads) continue;
            float x[8], y[8], ox[8], oy[8];
            rt_unpack<BF>(va[n], x);
            rt_unpack<BF>(vb[n], y);
            if constexpr (INTER) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    ox[2 * t] = x[2 * t] * c[t] - x[2 * t + 1] * s[t];
                    ox[2 * t + 1] = x[2 * t + 1] * c[t] + x[2 * t] * s[t];
                    oy[2 * t] = y[2 * t] * c[4 + t] - y[2 * t + 1] * s[4 + t];
                    oy[2 * t + 1] = y[2 * t + 1] * c[4 + t] + y[2 * t] * s[4 + t];
                }
            } else {
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    ox[t] = x[t] * c[t] - y[t] * s[t];
                    oy[t] = y[t] * c[t] + x[t] * s[t];
                }
            }
            u32x4 ra = turn_a ? rt_pack<BF>(ox) : va[n], rb = turn_b ? rt_pack<BF>(oy) : vb[n];
            if (!covered) ra = rb = zero_u4();
            f16 *p = place(a.q_out, a.k_out, h0 + n * HP);
            *reinterpret_cast<u32x4 *>(p + 8 * ca) = ra;
            *reinterpret_cast<u32x4 *>(p + 8 * cb) = rb;
        }
    }
}

// ---------------------------------------------------------------------------
// Tables.

struct RotaryTurns {
    double f[FA_ROTARY_MAX_DIM / 2];  // turns a token
};

// cos and sin of 2 pi t.  A turn count has four roundings of 2^-53: the angle is off by 2^-51 of itself, 2^-25 at the last position
// that the tables may have (FA_ROTARY_MAX_POSITION), half a step of fp32.  t less its nearest quarter turn leaves an angle y of at most pi / 4; the Taylor sums of sine
// and cosine to y^11 and y^12 are off by less than 1e-11 there, far under half a step of fp32.
__device__ __forceinline__ void rt_cos_sin(double t, double &c, double &s) {
    t -= rint(t);
    const double n = rint(4 * t), y = (t - n * 0.25) * 6.283185307179586476925, z = y * y;
    double p = -1.0 / 39916800, q = 1.0 / 479001600;
    p = fma(p, z, 1.0 / 362880);
    q = fma(q, z, -1.0 / 3628800);
    p = fma(p, z, -1.0 / 5040);
    q = fma(q, z, 1.0 / 40320);
    p = fma(p, z, 1.0 / 120);
    q = fma(q, z, -1.0 / 720);
    p = fma(p, z, -1.0 / 6);
    q = fma(q, z, 1.0 / 24);
    q = fma(q, z, -0.5);
    const double sy = fma(p * z, y, y), cy = fma(q, z, 1.0);
    const int k = int(n) & 3;
    s = k & 1 ? cy : sy;
    c = k & 1 ? sy : cy;
    if (k & 2) s = -s;
    if (k == 1 || k == 2) c = -c;
}

// Four neighbouring entries of a row a thread (rotary_dim / 2 is a multiple of 8).
__global__ __launch_bounds__(kRtThreads) void rotary_tables_kernel(const fa_rotary_tables_args a, const RotaryTurns turns) {
    const int half = a.rotary_dim / 2;
    const int64_t n = int64_t(a.seqlen) * (half / 4);
    for (int64_t e = int64_t(blockIdx.x) * kRtThreads + threadIdx.x; e < n; e += int64_t(gridDim.x) * kRtThreads) {
        const int row = int(e / (half / 4)), j = int(e - int64_t(row) * (half / 4)) * 4;
        const double p = double(a.offset + row);
        float c[4], s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            double x, y;
            rt_cos_sin(p * turns.f[j + u], x, y);
            c[u] = float(x * a.attention_factor);
            s[u] = float(y * a.attention_factor);
        }
        if (a.dtype == FA_FP32) {
            static_cast<f32x4 *>(a.cos)[e] = f32x4{c[0], c[1], c[2], c[3]};
            static_cast<f32x4 *>(a.sin)[e] = f32x4{s[0], s[1], s[2], s[3]};
        } else if (a.dtype == FA_BF16) {
            static_cast<f16x4 *>(a.cos)[e] = pack4<true>(c[0], c[1], c[2], c[3]);
            static_cast<f16x4 *>(a.sin)[e] = pack4<true>(s[0], s[1], s[2], s[3]);
        } else {
            static_cast<f16x4 *>(a.cos)[e] = pack4<false>(c[0], c[1], c[2], c[3]);
            static_cast<f16x4 *>(a.sin)[e] = pack4<false>(s[0], s[1], s[2], s[3]);
        }
    }
}

static bool rt_table_ok(const void *p, int64_t stride) { return p && !(reinterpret_cast<uintptr_t>(p) & 15u) && stride % 8 == 0; }

}  // namespace fa

extern "C" int fa_rotary_tables(const fa_rotary_tables_args *args, void *stream) {
    using namespace fa;
    if (!args) return FA_ERR_INVALID_ARG;
    const fa_rotary_tables_args &a = *args;
    if (a.rotary_dim <= 0 || a.rotary_dim % 16 || a.rotary_dim > FA_ROTARY_MAX_DIM || a.seqlen < 0) return FA_ERR_INVALID_ARG;
    if (a.dtype != FA_FP16 && a.dtype != FA_BF16 && a.dtype != FA_FP32) return FA_ERR_UNSUPPORTED;
    if (!(a.base > 0) || !(a.factor > 0) || !(a.original_seqlen >= 0) || !std::isfinite(a.attention_factor) ||
        a.offset < -FA_ROTARY_MAX_POSITION || a.offset > FA_ROTARY_MAX_POSITION ||
        a.offset + std::max(a.seqlen, 1) - 1 > FA_ROTARY_MAX_POSITION ||
        (a.original_seqlen > 0 && !(a.high_turns > a.low_turns)))
        return FA_ERR_INVALID_ARG;
    if (a.seqlen == 0) return FA_OK;
    if (!rt_table_ok(a.cos, 0) || !rt_table_ok(a.sin, 0)) return FA_ERR_INVALID_ARG;
    RotaryTurns turns{};
    constexpr double two_pi = 6.283185307179586476925;
    for (int j = 0; j < a.rotary_dim / 2; ++j) {
        double f = std::pow(a.base, -2.0 * j / a.rotary_dim);
        double keep = 0;
        if (a.original_seqlen > 0)
            keep = std::min(std::max((a.original_seqlen * f / two_pi - a.low_turns) / (a.high_turns - a.low_turns), 0.0), 1.0);
        turns.f[j] = f * (keep + (1 - keep) / a.factor) / two_pi;
    }
    const int64_t units = int64_t(a.seqlen) * (a.rotary_dim / 8);
    const int64_t wgs = std::min<int64_t>((units + kRtThreads - 1) / kRtThreads, 8 * device_cus());
    hipLaunchKernelGGL(rotary_tables_kernel, dim3(unsigned(wgs)), dim3(kRtThreads), 0, reinterpret_cast<hipStream_t>(stream),
                       a, turns);
    return int(hipGetLastError());
}

extern "C" int fa_rotary(const fa_rotary_args *args, void *stream) {
    using namespace fa;
    if (!args) return FA_ERR_INVALID_ARG;
    fa_rotary_args a = *args;
    if (a.head_dim != 64 && a.head_dim != 128) return FA_ERR_UNSUPPORTED;
    if (a.dtype != FA_FP16 && a.dtype != FA_BF16) return FA_ERR_UNSUPPORTED;
    if (a.table_dtype != FA_FP16 && a.table_dtype != FA_BF16 && a.table_dtype != FA_FP32) return FA_ERR_UNSUPPORTED;
    if (!a.k.ptr) a.nheads_k = 0;
    if (a.batch < 0 || a.seqlen < 0 || a.nheads < 0 || a.nheads_k < 0 || a.rotary_dim <= 0 || a.rotary_dim % 16 ||
        a.rotary_dim > a.head_dim || a.table_rows < 0)
        return FA_ERR_INVALID_ARG;
    const int64_t rows = a.cu_seqlens ? a.seqlen : int64_t(a.batch) * a.seqlen;
    if (rows == 0 || a.nheads + a.nheads_k == 0) return FA_OK;
    // A table without rows is not read (its entries would be at position 0).
    if (a.table_rows == 0 || !rt_table_ok(a.cos, a.cos_stride) || !rt_table_ok(a.sin, a.sin_stride)) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.q, &a.q_out})
        if (check_tensor(*t, a.nheads > 0)) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.k, &a.k_out})
        if (check_tensor(*t, a.nheads_k > 0)) return FA_ERR_INVALID_ARG;
    const int64_t grid = (rows + kRtThreads / 64 - 1) / (kRtThreads / 64);
    if (grid > 0xffffffffu / kRtThreads) return FA_ERR_INVALID_ARG;  // a launch has less than 2^32 threads
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    auto go = [&](auto hd, auto bf, auto inter) {
        hipLaunchKernelGGL((rotary_kernel<decltype(hd)::value, decltype(bf)::value, decltype(inter)::value>),
                           dim3(unsigned(grid)), dim3(kRtThreads), 0, s, a);
    };
    auto by_layout = [&](auto hd, auto bf) {
        if (a.interleaved)
            go(hd, bf, std::true_type{});
        else
            go(hd, bf, std::false_type{});
    };
    auto by_type = [&](auto hd) {
        if (a.dtype == FA_BF16)
            by_layout(hd, std::true_type{});
        else
            by_layout(hd, std::false_type{});
    };
    if (a.head_dim == 128)
        by_type(std::integral_constant<int, 128>{});
    else
        by_type(std::integral_constant<int, 64>{});
    return int(hipGetLastError());
}
