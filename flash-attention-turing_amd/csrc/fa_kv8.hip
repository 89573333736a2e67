// A key-value cache in 8 bits: quantising as it is written, reading back, and attention of few query rows
// (decode steps, drafted tokens) split over the cache's length.
#include <algorithm>

#include "fa_kv8_common.h"

namespace fa {

// ---------------------------------------------------------------------------
// Append.
//
// A workgroup takes one block of tokens of one head of K or V: it reads the new rows into registers, finds their largest
// magnitude as an integer (the bits of |x|, in which infinities and NaN come out on top), settles the block's scale, and
// writes codes.  Only where the scale grows are the block's earlier codes read and written again.  Scales are powers of
// two: the quotients are exact, codes that stay in e4m3's normal range keep their bits when a scale grows, and a block is
// raised at most a few times however many appends fill it.
//
// One token for each of 64 sequences takes 5 us, a chain of four latencies (length, page, rows, scale), and where it raises the
// scale of a full block 3 us more (64 tokens) to 10 (256); 4 prompts of up to 4096 tokens 15 us at 4.8 TB/s, a copy's rate
// at that size.

constexpr int kKv8Threads = 256;
constexpr int64_t kKv8MaxGrid = 0xffffffffu / kKv8Threads;  // a launch has less than 2^32 threads

// The smallest power of two s >= 2^-126 with x <= most * s, from the bits of |x| in the tensors' type; NaN if x is not finite.
template <bool BF, bool INT8>
__device__ __forceinline__ float kv8_scale_for(uint32_t bits) {
    if (bits >= (BF ? 0x7f80u : 0x7c00u)) return __builtin_nanf("");
    const float x = BF ? __uint_as_float(bits << 16) : float(__builtin_bit_cast(f16, uint16_t(bits)));
    const uint32_t u = __float_as_uint(x);
    // x = (1 + f) 2^e; 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.
    const int e = int(u >> 23) - 127 - (INT8 ? 6 : 8) + ((u & 0x7fffffu) > (INT8 ? 0x7e0000u : 0x600000u) ? 1 : 0);
    return e <= -126 ? kKv8MinScale : __uint_as_float(uint32_t(e + 127) << 23);
}

// x / s for eight values, as codes.  A power of two divides by its reciprocal, exactly.
template <bool INT8>
__device__ __forceinline__ u32x2 kv8_encode(const float (&x)[8], float s) {
    f32x4 v[2];
    if ((__float_as_uint(s) & 0x7fffffu) == 0) {
        const float inv = 1.f / s;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = x[i] * inv;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = __fdiv_rn(x[i], s);
    }
    return u32x2{kv8_codes<INT8>(v[0]), kv8_codes<INT8>(v[1])};
}

template <int HD, bool BF, bool INT8, int U>
__global__ __launch_bounds__(kKv8Threads) void kv8_append_kernel(const fa_kv8_args a, const Kv8Plan plan, const int plan_wgs,
                                                                 const int clear_wgs, const int blocks) {
    if (int(blockIdx.x) < plan_wgs) return kv8_make_plan(a, plan);
    if (int(blockIdx.x) < plan_wgs + clear_wgs) {
        const int64_t i = int64_t(blockIdx.x - plan_wgs) * kKv8Threads + threadIdx.x;
        if (i < plan.counters) static_cast<int32_t *>(a.ws)[i] = 0;
        return;
    }
    constexpr int KCH = HD / 8;  // units of a row: 8 elements
    __shared__ uint32_t part[kKv8Threads / 64];
    const fa_kv8_cache &c = a.cache;
    int rest = int(blockIdx.x) - plan_wgs - clear_wgs;
    const bool is_v = rest & 1;
    rest >>= 1;
    const int hk = rest % c.nheads_k;
    rest /= c.nheads_k;
    const int j = rest % blocks, b = rest / blocks;
    const int L0 = a.cache_seqlens[b], n = a.seqlens_new ? a.seqlens_new[b] : a.seqlen_new;
    int row;
    const int err = kv8_err(c, b, L0, n, a.seqlen_new, row);
    if (err) {
        if (c.status && rest % blocks == 0 && hk == 0 && !is_v && threadIdx.x == 0) atomicOr(c.status, err);
        return;
    }
    const int p0 = (L0 / c.scale_block + j) * c.scale_block;  // the block's first token; a capacity's blocks are whole
    const int end = min(L0 + n, p0 + c.scale_block), first = max(L0, p0);
    if (first >= end) return;
    int64_t line = row;
    int at = p0;
    if (c.block_table) {
        const int pg = p0 / c.page_block_size;
        line = c.block_table[int64_t(b) * c.block_table_stride + pg];
        at = p0 - pg * c.page_block_size;
        if (line < 0 || line >= c.num_pages) {
            if (c.status && hk == 0 && !is_v && threadIdx.x == 0) atomicOr(c.status, FA_KV_BAD_PAGE);
            return;
        }
    }
    const fa_tensor &src_t = is_v ? a.v_new : a.k_new, &dst_t = is_v ? c.v : c.k;
    const fa_kv8_scales &sc = is_v ? c.v_scale : c.k_scale;
    const f16 *src = (const f16 *)src_t.ptr + int64_t(b) * src_t.batch_stride + int64_t(hk) * src_t.head_stride;
    char *dst = (char *)dst_t.ptr + line * dst_t.batch_stride + int64_t(at) * dst_t.row_stride + int64_t(hk) * dst_t.head_stride;
    float *scale = sc.ptr + line * sc.batch_stride + int64_t(at / c.scale_block) * sc.row_stride + int64_t(hk) * sc.head_stride;

    const int units = (end - first) * KCH;
    u32x4 v[U];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int e = i * kKv8Threads + threadIdx.x;
        v[i] = e < units ? ldg16(src + int64_t(first - L0 + e / KCH) * src_t.row_stride + 8 * (e % KCH)) : zero_u4();
    }
    const bool held = p0 < L0;
    const float old = held ? *scale : kKv8MinScale;
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) top = max(top, max(v[i][w] & 0x7fffu, v[i][w] >> 16 & 0x7fffu));
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = max(top, uint32_t(__shfl_xor(int(top), d)));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();  // every thread has read the old scale, too
#pragma unroll
    for (int w = 0; w < kKv8Threads / 64; ++w) top = max(top, part[w]);
    float s = kv8_scale_for<BF, INT8>(top);
    const bool bad = !(s == s) || !(old == old);  // such a block reads as NaN; its codes are finite, so that no masked
    if (bad)                                      // key's turns up in a product
        s = __builtin_nanf("");
    else
        s = fmaxf(s, old);
    if (threadIdx.x == 0) *scale = s;
    if (held && !bad && s != old) {
        const int olds = (L0 - p0) * KCH;
#pragma unroll 4
        for (int e = threadIdx.x; e < olds; e += kKv8Threads) {
            u32x2 *p = reinterpret_cast<u32x2 *>(dst + int64_t(e / KCH) * dst_t.row_stride + 8 * (e % KCH));
            const u32x2 q = *p;
            const f32x4 lo = kv8_values<INT8>(q[0]), hi = kv8_values<INT8>(q[1]);
            const float x[8] = {lo[0] * old, lo[1] * old, lo[2] * old, lo[3] * old,
                                hi[0] * old, hi[1] * old, hi[2] * old, hi[3] * old};
            *p = kv8_encode<INT8>(x, s);
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int e = i * kKv8Threads + threadIdx.x;
        if (e >= units) continue;
        float x[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) x[t] = elem<BF>(as_h8(v[i]), t);
        u32x2 q = {0u, 0u};
        if (!bad) q = kv8_encode<INT8>(x, s);
        *reinterpret_cast<u32x2 *>(dst + int64_t(first - p0 + e / KCH) * dst_t.row_stride + 8 * (e % KCH)) = q;
    }
}

// ---------------------------------------------------------------------------
// Read back: a workgroup takes some packed rows, all heads of K and of V.  Its first threads find the rows' places, one each;
// then every thread has kKv8Reads loads of eight codes under way before the first is used.  Memory bounds it: prefixes of 16
// sequences (330 MB moved) take 73 us, 4.5 TB/s; a wave that took four rows one after the other, its places from the
// first lane to the last, took 85 us.

constexpr int kKv8Reads = 8, kKv8ReadRows = 64;

// Rows of a workgroup: one batch of loads.
static inline int kv8_read_rows(int units) { return std::min(std::max(kKv8Reads * kKv8Threads / units, 1), kKv8ReadRows); }

template <int HD, bool BF, bool INT8>
__global__ __launch_bounds__(kKv8Threads) void kv8_read_kernel(const fa_kv8_read_args a, const int rows) {
    constexpr int CH = HD / 8;
    const fa_kv8_cache &c = a.cache;
    __shared__ int64_t line_of[kKv8ReadRows];
    __shared__ int at_of[kKv8ReadRows];  // -1: zeros
    const int tid = threadIdx.x;
    const int64_t r0 = int64_t(blockIdx.x) * rows;
    const int n_rows = int(min(int64_t(rows), a.total - r0));
    const int b0 = tid < 64 ? packed_sequence(a.cu_seqlens, c.batch, int(r0)) : 0;
    if (tid < n_rows) {
        // The row's sequence is the first row's or a later one: the last that starts at or before the row.
        const int r = int(r0) + tid;
        int b = b0;
        if (b < c.batch && a.cu_seqlens[b + 1] <= r) {
            int out = c.batch + 1;  // starts behind the row, or the end
            for (++b; out - b > 1;) {
                const int mid = b + (out - b) / 2;
                if (a.cu_seqlens[mid] <= r)
                    b = mid;
                else
                    out = mid;
            }
        }
        int64_t line = 0;
        int at = -1;
        if (b >= 0 && b < c.batch) {
            const int start = a.cu_seqlens[b];
            int row;
            const int n = a.cu_seqlens[b + 1] - start, err = kv8_err(c, b, 0, n, INT_MAX, row);
            if (err && c.status) atomicOr(c.status, err);
            if (!err && r - start < n) {
                at = r - start;
                line = row;
                if (c.block_table) {
                    const int pg = at / c.page_block_size;
                    line = c.block_table[int64_t(b) * c.block_table_stride + pg];
                    at -= pg * c.page_block_size;
                    if (line < 0 || line >= c.num_pages) {
                        if (c.status) atomicOr(c.status, FA_KV_BAD_PAGE);
                        line = 0;
                    }
                }
            }
        }
        line_of[tid] = line;
        at_of[tid] = at;
    }
    __syncthreads();
    const uint32_t half = c.nheads_k * CH, units = 2 * half, n = n_rows * units;
    for (uint32_t e0 = tid; e0 < n; e0 += kKv8Reads * kKv8Threads) {
        u32x2 q[kKv8Reads];
        float s[kKv8Reads];
#pragma unroll
        for (int i = 0; i < kKv8Reads; ++i) {
            q[i] = u32x2{0u, 0u};
            s[i] = 0.f;
            const uint32_t e = e0 + i * kKv8Threads, r = e / units, x = e - r * units;
            if (e >= n || at_of[r] < 0) continue;
            const bool is_v = x >= half;
            const uint32_t y = is_v ? x - half : x, h = y / CH, ch = y % CH;
            const fa_tensor &t = is_v ? c.v : c.k;
            const fa_kv8_scales &sc = is_v ? c.v_scale : c.k_scale;
            const int64_t line = line_of[r];
            const int at = at_of[r];
            q[i] = *reinterpret_cast<const u32x2 *>((const char *)t.ptr + line * t.batch_stride + int64_t(at) * t.row_stride +
                                                    int64_t(h) * t.head_stride + 8 * ch);
            s[i] = sc.ptr[line * sc.batch_stride + int64_t(uint32_t(at) / uint32_t(c.scale_block)) * sc.row_stride +
                          int64_t(h) * sc.head_stride];
        }
#pragma unroll
        for (int i = 0; i < kKv8Reads; ++i) {
            const uint32_t e = e0 + i * kKv8Threads, r = e / units, x = e - r * units;
            if (e >= n) continue;
            const bool is_v = x >= half;
            const uint32_t y = is_v ? x - half : x, h = y / CH, ch = y % CH;
            const fa_tensor &o = is_v ? a.v_out : a.k_out;
            const f32x4 lo = kv8_values<INT8>(q[i][0]), hi = kv8_values<INT8>(q[i][1]);
            const f16x4 y0 = pack4<BF>(lo[0] * s[i], lo[1] * s[i], lo[2] * s[i], lo[3] * s[i]);
            const f16x4 y1 = pack4<BF>(hi[0] * s[i], hi[1] * s[i], hi[2] * s[i], hi[3] * s[i]);
            f16 *p = (f16 *)o.ptr + (r0 + r) * o.row_stride + int64_t(h) * o.head_stride + 8 * ch;
            *reinterpret_cast<f16x8 *>(p) = __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
}

// ---------------------------------------------------------------------------
// Attention of few rows.
//
// S^T = K Q^T in 16 x 16 x 32 MFMAs: 16 keys by 16 rows, the rows of a KV head being its query heads times the query
// positions.  A lane's 16-byte LDS read holds the codes of two K steps (which channels a step takes is free, as long as Q's
// operand takes the same), and keys are dealt to the two MFMAs of a tile so that a lane ends up with the eight consecutive
// keys that it supplies to the product with V, whose codes come transposed from LDS, eight keys of a channel a lane.
//
// A workgroup's four waves walk the 32-key tiles of its piece (tile t to wave t % 4), each through LDS slots of its own with
// no barrier in the loop; codes go from memory to LDS without passing registers.
//
// What bounds it: memory for large batches (64 sequences of 1k to 16k tokens, 8 heads of 128: 165 us of a call's 172, 5.0 TB/s),
// and a chain of latencies for short ones (1500 tokens: 11 us; length and plan, tiles' places, codes, partial results, counter,
// join).  Codes and P stay out of the vector units' way: products take codes as they are and P times V's scale as bf16 hi + lo.

constexpr int kKdTile = 32;

// g2l16_at (fa_diff_common.h); once: for bytes that no other workgroup reads, which the caches are asked not to keep.
__device__ __forceinline__ void kd_copy(const char *base, uint32_t off, uint32_t l, bool once) {
    if (!once) return g2l16_at((const f16 *)base, off, l);
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2 nt\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(off), "s"(base), "s"(l)
        : "memory");
}

template <bool BF>
__device__ __forceinline__ f32x4 kd_mfma(const f16x8 a, const f16x8 b, const f32x4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Maximum / sum over the four lanes l % 16 + 16 i.
__device__ __forceinline__ float kd_max4(float x) { return fmaxf(fmaxf(x, __shfl_xor(x, 16)), fmaxf(__shfl_xor(x, 32), __shfl_xor(x, 48))); }
__device__ __forceinline__ float kd_sum4(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <int HD, bool BF, bool INT8, int NH>
__global__ __launch_bounds__(kKv8Threads, 2) void kv8_decode_kernel(const Kv8Call call) {
    kv8_early();
    const fa_kv8_args &a = call.a;
    const Kv8Plan &plan = call.plan;
    constexpr int CH = HD / 16, TILE = kKdTile * HD, STAGE = 2 * NH * TILE, NST = NH * HD == 256 ? 1 : 2;
    constexpr int CPW = TILE / 1024;  // copies a lane for a head's K or V of a tile
    constexpr int MERGE = 17;         // row stride of the waves' O^T at the merge
    constexpr int WAVE_LDS = NST * STAGE > HD * MERGE * 4 ? NST * STAGE : HD * MERGE * 4;
    constexpr int STEPS = HD / 32, ROWS = NH * kKdRows;
    __shared__ __attribute__((aligned(1024))) char smem[4 * WAVE_LDS];
    __shared__ f32x2 ml[4][16];
    __shared__ int ticket;
    static_assert(4 * WAVE_LDS >= ROWS * (kKv8Join + 2) * 4, "the join's scratch");

    const fa_kv8_cache &c = a.cache;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int HI = c.nheads_k / NH * plan.row_tiles;
    int slot_i, hg, rt;
    if (!kv8_item(plan, c.nheads_k / NH, blockIdx.x, slot_i, hg, rt)) return;
    const int hi_i = hg * plan.row_tiles + rt, hk0 = hg * NH;
    const Kv8Slot sl = kv8_slot(a, plan, slot_i);
    if (sl.b < 0) return;
    const int G = a.nheads / c.nheads_k, R = G * a.seqlen_q, L = sl.keys;
    const int row = rt * kKdRows + col;
    const bool row_ok = row < R;
    const int qpos = row_ok ? row / G : 0, gq = row_ok ? row - qpos * G : 0;
    const int shift = L - a.seqlen_q;  // position of query 0
    const int first = kv8_first(a, qpos + shift), last = kv8_last(a, qpos + shift, L);
    // Keys that every row of the tile sees, and that any does.
    const int q_lo = rt * kKdRows / G, q_hi = min(rt * kKdRows + kKdRows - 1, R - 1) / G;
    const int all_first = kv8_first(a, q_hi + shift), all_last = kv8_last(a, q_lo + shift, L);
    const int s0 = max(sl.begin, kv8_first(a, q_lo + shift)) / kKdTile * kKdTile, s1 = min(sl.end, kv8_last(a, q_hi + shift, L) + 1);
    const int t_first = s0 / kKdTile, t_end = (s1 + kKdTile - 1) / kKdTile;
    const int my_first = t_first + wave;
    const int n_my = my_first < t_end ? (t_end - my_first + 3) / 4 : 0;

    char *const slot = smem + wave * WAVE_LDS;
    constexpr int RPC = 1024 / HD;  // rows of a copy
    const int64_t krs = c.k.row_stride, vrs = c.v.row_stride;  // (at most 2^23)
    const int row0 = lane / CH;
    uint32_t ch[CPW];
#pragma unroll
    for (int i = 0; i < CPW; ++i) ch[i] = 16 * (lane % CH ^ kv8_swz<HD>(row0 + i * RPC));
    const uint32_t k_off = uint32_t(row0) * uint32_t(krs), v_off = uint32_t(row0) * uint32_t(vrs);
    const uint32_t lds0 = lds_addr(slot);
    const float cscale = a.softmax_scale * kLog2e;
    const bool once = plan.row_tiles == 1;
    // Q^T as B operands: step st takes channels 64 (st / 2) + 16 g + 8 (st % 2) + 0..7.
    f16x8 qB[NH][STEPS];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        const f16 *qp = (const f16 *)a.q.ptr + int64_t(sl.b) * a.q.batch_stride + int64_t(qpos) * a.q.row_stride +
                        int64_t((hk0 + h) * G + gq) * a.q.head_stride + 16 * g;
#pragma unroll
        for (int st = 0; st < STEPS; ++st) qB[h][st] = as_h8(row_ok ? ldg16(qp + 64 * (st / 2) + 8 * (st % 2)) : zero_u4());
    }
    f32x4 o[NH][CH];
    float m[NH], l[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) o[h][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // LDS addresses: K rows of the tile's two MFMAs, and the transposed V reads.
    const int k_row0 = 8 * (col >> 2) + (col & 3), v_row = 8 * g + (col >> 1), v_half = 8 * (col & 1);

    // 64 tiles of the wave at a time: lane i looks up where tile i's codes begin, and its scales.
    for (int k_base = 0; k_base < n_my; k_base += 64) {
        const int n = min(n_my - k_base, 64), t_base = my_first + 4 * k_base;
        uint64_t ka, va;
        float ks[NH], vs[NH];
        {
            const int p0 = (t_base + 4 * min(lane, n - 1)) * kKdTile;
            int64_t line = sl.row;
            int at = p0;
            if (c.block_table) {
                const int pg = p0 / c.page_block_size;
                at = p0 - pg * c.page_block_size;
                line = c.block_table[int64_t(sl.b) * c.block_table_stride + pg];
                if (line < 0 || line >= c.num_pages) {
                    if (c.status) atomicOr(c.status, FA_KV_BAD_PAGE);
                    line = 0;
                }
            }
            const int blk = at >> __builtin_ctz(c.scale_block);
            ka = reinterpret_cast<uint64_t>(c.k.ptr) + line * c.k.batch_stride + int64_t(at) * krs + int64_t(hk0) * c.k.head_stride;
            va = reinterpret_cast<uint64_t>(c.v.ptr) + line * c.v.batch_stride + int64_t(at) * vrs + int64_t(hk0) * c.v.head_stride;
            const float *kp = c.k_scale.ptr + line * c.k_scale.batch_stride + int64_t(blk) * c.k_scale.row_stride;
            const float *vp = c.v_scale.ptr + line * c.v_scale.batch_stride + int64_t(blk) * c.v_scale.row_stride;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                ks[h] = kp[int64_t(hk0 + h) * c.k_scale.head_stride];
                vs[h] = vp[int64_t(hk0 + h) * c.v_scale.head_stride];
            }
        }
        auto of_lane = [](uint64_t x, int i) FA_INLINE {
            return reinterpret_cast<const char *>(uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(x), i))) |
                                                  uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(x >> 32), i))) << 32);
        };
        auto issue = [&](int k, int st) FA_INLINE {
            const char *kb = of_lane(ka, k), *vb = of_lane(va, k);
            const uint32_t to = lds0 + st * STAGE;
            const int most = L - 1 - (t_base + 4 * k) * kKdTile;
            if (most >= kKdTile - 1) {
#pragma unroll
                for (int i = 0; i < CPW; ++i)
#pragma unroll
                    for (int h = 0; h < NH; ++h) {  // (neighbouring heads are neighbouring bytes)
                        kd_copy(kb + i * RPC * krs + h * c.k.head_stride, k_off + ch[i], to + h * TILE + i * 1024, once);
                        kd_copy(vb + i * RPC * vrs + h * c.v.head_stride, v_off + ch[i], to + (NH + h) * TILE + i * 1024, once);
                    }
            } else {
                // Rows past the sequence re-read its last one, so that no stale code reaches a product.
#pragma unroll
                for (int i = 0; i < CPW; ++i) {
                    const uint32_t r = min(row0 + i * RPC, most);
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        kd_copy(kb + h * c.k.head_stride, r * uint32_t(krs) + ch[i], to + h * TILE + i * 1024, once);
                        kd_copy(vb + h * c.v.head_stride, r * uint32_t(vrs) + ch[i], to + (NH + h) * TILE + i * 1024, once);
                    }
                }
            }
        };
#pragma unroll
        for (int st = 0; st < NST; ++st)
            if (st < n) issue(st, st);
        wait_vmem();  // only tile copies are in flight inside the loop
#pragma unroll
        for (int h = 0; h < NH; ++h) asm volatile("" : "+v"(ks[h]), "+v"(vs[h]));
        for (int k0 = 0; k0 < n; k0 += NST) {
#pragma unroll
            for (int st = 0; st < NST; ++st) {
                const int k = k0 + st;
                if (k >= n) break;
                const int p0 = (t_base + 4 * k) * kKdTile;
                if (k + 1 < n)
                    wait_vmem_n<(NST - 1) * 2 * NH * CPW>();
                else
                    wait_vmem();
                u32x4 kc[NH][2][HD / 64];
                u32x2 vc[NH][CH];
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const char *kt = slot + st * STAGE + h * TILE, *vt = kt + NH * TILE;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int j = 0; j < HD / 64; ++j) {
                            const int r = k_row0 + 4 * t;
                            kc[h][t][j] = *reinterpret_cast<const u32x4 *>(kt + r * HD + 16 * ((4 * j + g) ^ kv8_swz<HD>(r)));
                        }
#pragma unroll
                    for (int d = 0; d < CH; ++d) vc[h][d] = lds_tr8(vt, v_row * HD + 16 * (d ^ kv8_swz<HD>(v_row)) + v_half);
                }
                wait_lds();
                if (k + NST < n) issue(k + NST, st);
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    // Scales reach the scores of their keys as 0, or as NaN where one is not finite (of infinity times a score of
                    // either sign, softmax would pass over half), and V's then has done its part.
                    const float ksk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks[h]), k));
                    const float vsk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs[h]), k));
                    const float sk = ksk * cscale, sv0 = fmaf(vsk, 0.f, ksk * 0.f), sv = sv0 == 0.f ? vsk : 0.f;
                    f32x4 s[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < STEPS; ++i) {
                            const u32x4 q = kc[h][t][i / 2];
                            s[t] = kd_mfma<BF>(kv8_decode<INT8, BF>(i % 2 ? u32x2{q[2], q[3]} : u32x2{q[0], q[1]}), qB[h][i], s[t]);
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][r] = fmaf(s[t][r], sk, sv0);
                    }
                    if (p0 < all_first || p0 + kKdTile - 1 > all_last) {
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int key = p0 + 8 * g + 4 * t + r;
                                if (key < first || key > last) s[t][r] = -INFINITY;
                            }
                    }
                    // The maximum is raised only when a score passes it by 2^8: sums and products keep 32 bits.
                    const float top = max3(max3(max3(s[0][0], s[0][1], s[0][2]), s[0][3], s[1][0]), max3(s[1][1], s[1][2], s[1][3]), -INFINITY);
                    if (__builtin_amdgcn_ballot_w64(top > m[h] + 8.f) != 0) {
                        const float m_new = fmaxf(m[h], kd_max4(top));
                        const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m[h] - m_new);
                        l[h] *= alpha;
#pragma unroll
                        for (int d = 0; d < CH; ++d)
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[h][d][r] *= alpha;
                        m[h] = m_new;
                    }
                    const float m_use = m[h] == -INFINITY ? 0.f : m[h];
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        e[i] = exp2_fast(s[i / 4][i % 4] - m_use);
                        l[h] += e[i];
                    }
                    // P times V's scale in bf16, which has fp32's range, as hi + lo: 16 bits.
                    bf16x8 hi, lo;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float w = e[i] * sv;
                        hi[i] = (__bf16)w;
                        lo[i] = (__bf16)(w - float(hi[i]));
                    }
#pragma unroll
                    for (int d = 0; d < CH; ++d) {
                        const f16x8 v = kv8_decode<INT8, true>(vc[h][d]);
                        o[h][d] = kd_mfma<true>(v, __builtin_bit_cast(f16x8, hi), o[h][d]);
                        o[h][d] = kd_mfma<true>(v, __builtin_bit_cast(f16x8, lo), o[h][d]);
                    }
                }
            }
        }
    }

    // Merge the four waves, a head after the other: O^T to LDS, then every thread sums pairs of channels of a row.
    const Kv8Call &late = kv8_late();
    const int rows = min(kKdRows, R - rt * kKdRows);
    const int64_t part = int64_t(sl.part) * HI + hi_i;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        if (h > 0) __syncthreads();
        const float lh = kd_sum4(l[h]);
        float *ow = reinterpret_cast<float *>(slot);
#pragma unroll
        for (int d = 0; d < CH; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) ow[(16 * d + 4 * g + r) * MERGE + col] = o[h][d][r];
        if (g == 0) ml[wave][col] = f32x2{m[h], lh};
        __syncthreads();
        for (int e = tid; e < rows * (HD / 2); e += kKv8Threads) {
            const int r = e / (HD / 2), d = 2 * (e % (HD / 2));
            const float mm = fmaxf(fmaxf(ml[0][r][0], ml[1][r][0]), fmaxf(ml[2][r][0], ml[3][r][0]));
            float ll = 0.f;
            f32x2 x = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = ml[w][r][0] == -INFINITY ? 0.f : exp2_fast(ml[w][r][0] - mm);
                const float *q = reinterpret_cast<const float *>(smem + w * WAVE_LDS);
                ll = fmaf(ml[w][r][1], f, ll);
                x[0] = fmaf(q[d * MERGE + r], f, x[0]);
                x[1] = fmaf(q[(d + 1) * MERGE + r], f, x[1]);
            }
            if (sl.n_pieces == 1) {
                kv8_store<HD, BF>(late.a, sl.b, hk0 + h, rt * kKdRows + r, d, x, mm, ll);
            } else {
                kv8_put(kv8_o<HD>(late.a, late.plan, part) + h * rows * (HD / 2) + e, x);
                if (d == 0) kv8_put(kv8_ml(late.a, late.plan, part) + h * rows + r, f32x2{mm, ll});
            }
        }
    }
    if (sl.n_pieces == 1) return;
    const int F = kv8_group(sl.n_pieces, rows * HD * 4), g0 = sl.ch / F * F, in_group = min(F, sl.n_pieces - g0), groups = (sl.n_pieces + F - 1) / F;
    const int64_t part0 = part - int64_t(sl.ch) * HI, group_part = part0 + int64_t(g0) * HI;
    float *scratch = reinterpret_cast<float *>(smem);
    if (!kv8_count(kv8_counter(late.a, late.plan.items + group_part), in_group, &ticket)) return;
    // (One copy of the join for both steps: a workgroup comes here with its instructions still in memory.)
    const auto join = [&](auto units) FA_INLINE {
        bool last = groups == 1;
        int64_t from = group_part, step = HI;
        int n = in_group;
        for (;;) {
            kv8_join<HD, ROWS, decltype(units)::value>(
                late.a, late.plan, NH * rows, n, scratch, [&](int i) { return from + i * step; },
                [&](int r, int d, f32x2 x, float mm, float ll) {
                    if (last) {
                        const int h = r / rows;
                        kv8_store<HD, BF>(late.a, sl.b, hk0 + h, rt * kKdRows + r - h * rows, d, x, mm, ll);
                    } else {
                        kv8_put(kv8_o<HD>(late.a, late.plan, group_part) + r * (HD / 2) + d / 2, x);
                        if (d == 0) kv8_put(kv8_ml(late.a, late.plan, group_part) + r, f32x2{mm, ll});
                    }
                });
            if (last || !kv8_count(kv8_counter(late.a, int64_t(sl.b) * HI + hi_i), groups, &ticket)) return;
            last = true;
            from = part0;
            step = int64_t(F) * HI;
            n = groups;
        }
    };
    if (NH * rows * (HD / 2) <= kKv8Threads)
        join(std::integral_constant<int, 1>{});
    else
        join(std::integral_constant<int, ROWS * (HD / 2) / kKv8Threads>{});
}

// ---------------------------------------------------------------------------
// Host.

int kv8_chunk(const fa_kv8_args &a, const Kv8Plan &plan, hipStream_t s);  // fa_kv8_fwd.hip

// KV heads that a workgroup of few rows takes together, one or two: their codes of a token are neighbours in memory, which reads
// longer runs faster, but there are fewer items to share a short call.  Measured (us, one and two), 8 heads of 128 channels:
// 64 x 8192 tokens 193 and 173, 8 x 32000 102 and 98, 2 x 131072 106 and 106, 1 x 131072 60 and 76; heads of 64, whose codes are
// half a line: 8 heads 64 x 8192 173 and 116, 1 x 131072 56 and 45, 4 heads 4 x 48000 43 and 35.
static int kv8_heads(const fa_kv8_args &a) {
    const int64_t bytes = int64_t(a.cache.batch) * a.cache.cache_capacity * a.cache.nheads_k * a.cache.head_dim * 2;
    const bool two = a.cache.head_dim == 64 ? bytes >= 32 << 20 : bytes >= 256 << 20 && a.cache.batch >= 4;
    return two && a.cache.nheads_k % 2 == 0 ? 2 : 1;
}

static Kv8Plan kv8_plan(const fa_kv8_args &a) {
    Kv8Plan p{};
    const int64_t rows = int64_t(a.nheads / a.cache.nheads_k) * a.seqlen_q, cap = std::max(a.cache.cache_capacity, 1);
    // The kernel of many rows reads and converts the codes once for 128 rows, the other one for 16, but it starts later and its
    // pieces' results are large.  Measured, by the 16-row tiles' keys (us, few and many): 32 rows of 8 heads x 8192 keys 25 and 37,
    // 512 rows x 8192 57 and 50, 1024 x 32768 323 and 164; batch of 32 x 20 rows x 6144 101 and 110, 16 x 32 x 8192 80 and 74.
    const int64_t few_keys = (rows + kKdRows - 1) / kKdRows * a.cache.nheads_k * a.cache.batch * cap;
    // A given number of pieces asks for sums that do not depend on the batch.
    p.many = a.num_splits > 0 ? rows >= 4 * kKdRows : rows >= 2 * kKdRows && few_keys >= int64_t(6144) * device_cus();
    const int tile = p.many ? kKcRows : kKdRows;
    p.row_tiles = int((rows + tile - 1) / tile);
    p.heads = p.many ? 1 : kv8_heads(a);
    p.rows_max = p.many ? tile : p.heads * int(std::min<int64_t>(rows, tile));
    const int64_t heads = int64_t(a.cache.nheads_k / p.heads) * p.row_tiles;
    p.items = a.cache.batch * heads;
    p.least = p.many ? 512 : 256;  // fewer and longer: 8 heads x 512 rows x 2048 keys took 36 us at 256 and 31 us at 512
    // Two workgroups run on a CU.  One reads memory as fast, but more rows compute, too (us, one a CU and two): 24 rows x 9000 keys
    // 24 and 27, 64 rows x 2000 keys of 8 sequences 29 and 30, but 256 rows x 8192 keys 49 and 39.
    p.most = int(std::max<int64_t>(2 * device_cus() / heads, 1));
    p.want = p.many || p.row_tiles > 2 ? p.most : int(std::max<int64_t>(device_cus() / heads, 1));
    int64_t slots, parts;
    if (a.num_splits > 0) {
        p.fixed = int(((cap + a.num_splits - 1) / a.num_splits + kKv8Round - 1) / kKv8Round * kKv8Round);
        slots = a.cache.batch * ((cap + p.fixed - 1) / p.fixed);
        parts = cap > p.fixed ? slots : 0;
    } else {
        // Pieces of more than total / most keys (many rows) or half of that: a sequence has at most one short piece, and a
        // sequence with several is longer than a piece.  So fewer than most (2 most) sequences have several, of fewer than
        // most (2 most) pieces and as many again as there are such sequences: none where most is 1.
        parts = p.many ? 2 * int64_t(p.most) - 2 : 4 * int64_t(p.most) - 2;
        slots = std::min<int64_t>(2 * int64_t(p.most) + a.cache.batch, a.cache.batch * ((cap + p.least - 1) / p.least));
    }
    p.slots = int(std::min<int64_t>(slots, INT32_MAX));
    if (slots == a.cache.batch) parts = 0;
    parts = std::min(parts, slots);
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    p.counters = parts ? p.items + parts * heads : 0;
    p.at_slots = up(p.counters * 4);
    p.at_ml = p.at_slots + up(slots * int64_t(sizeof(Kv8Slot)));
    p.at_o = p.at_ml + up(parts * heads * p.rows_max * 8);
    p.bytes = p.at_o + parts * heads * p.rows_max * a.cache.head_dim * 4;
    return p;
}

// Descriptors of a cache; tokens: of a page or row.
static int check_kv8_cache(const fa_kv8_cache &c) {
    if (c.head_dim != 64 && c.head_dim != 128) return FA_ERR_UNSUPPORTED;
    if (c.kind != FA_KV8_E4M3 && c.kind != FA_KV8_INT8) return FA_ERR_UNSUPPORTED;
    // (2^30 tokens: a position and a table of places behind it stay in 32 bits.)
    if (c.batch < 0 || c.nheads_k <= 0 || c.cache_capacity < 0 || c.cache_capacity > 1 << 30) return FA_ERR_INVALID_ARG;
    if (c.scale_block != 32 && c.scale_block != 64 && c.scale_block != 128 && c.scale_block != 256) return FA_ERR_INVALID_ARG;
    if (c.block_table ? c.cache_batch_idx || c.page_block_size <= 0 || c.page_block_size % c.scale_block || c.num_pages <= 0
                      : c.cache_capacity % c.scale_block != 0)
        return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&c.k, &c.v}) {
        if (!t->ptr || ((reinterpret_cast<uintptr_t>(t->ptr) | uint64_t(t->batch_stride) | uint64_t(t->row_stride) |
                         uint64_t(t->head_stride)) & 15u))
            return FA_ERR_INVALID_ARG;
        if (t->row_stride < 0 || t->row_stride > kDiffMaxRowStride) return FA_ERR_INVALID_ARG;
    }
    for (const fa_kv8_scales *s : {&c.k_scale, &c.v_scale})
        if (!s->ptr || (reinterpret_cast<uintptr_t>(s->ptr) & 3u)) return FA_ERR_INVALID_ARG;
    return FA_OK;
}

static int check_kv8_new(const fa_kv8_args &a) {
    if (a.dtype != FA_FP16 && a.dtype != FA_BF16) return FA_ERR_UNSUPPORTED;
    if (a.seqlen_new < 0 || !a.cache_seqlens) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.k_new, &a.v_new})
        if (check_tensor(*t, a.seqlen_new > 0)) return FA_ERR_INVALID_ARG;
    return FA_OK;
}

// Workgroups that plan and clear (plan NULL: none) and those that append, in one launch.
static int launch_kv8_append(const fa_kv8_args &a, const Kv8Plan *plan, hipStream_t s) {
    const fa_kv8_cache &c = a.cache;
    const int blocks = a.seqlen_new > 0 ? int((int64_t(a.seqlen_new) + 2 * c.scale_block - 2) / c.scale_block) : 0;
    const int64_t clear = plan ? (plan->counters + kKv8Threads - 1) / kKv8Threads : 0;
    const int64_t grid = (plan ? 1 : 0) + clear + int64_t(c.batch) * blocks * c.nheads_k * 2;
    if (grid > kKv8MaxGrid) return FA_ERR_INVALID_ARG;
    if (grid == 0) return FA_OK;
    const int most = std::min(c.scale_block, std::max(a.seqlen_new, 1)) * (c.head_dim / 8);  // units of a workgroup
    return kv8_by_type(c.head_dim, a.dtype, c.kind, [&](auto hd, auto bf, auto int8) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool BF = decltype(bf)::value, INT8 = decltype(int8)::value;
        auto go = [&](auto u) {
            hipLaunchKernelGGL((kv8_append_kernel<HD, BF, INT8, decltype(u)::value>), dim3(unsigned(grid)), dim3(kKv8Threads), 0,
                               s, a, plan ? *plan : Kv8Plan{}, plan ? 1 : 0, int(clear), std::max(blocks, 1));
            return int(hipGetLastError());
        };
        // As many units a thread as a block or the call has at most: registers for more cost waves.  4 x 2048 tokens, 8 heads (us,
        // so many and the most): blocks of 32, 64 channels, 12.8 and 15.2 (1 and 8); of 64, 128 channels, 11.2 and 15.5 (4 and 16);
        // 4 prompts of up to 4096 tokens, blocks of 128, 15.3 and 16.9 (8 and 16).
        if (most <= kKv8Threads) return go(std::integral_constant<int, 1>{});
        if (most <= 4 * kKv8Threads) return go(std::integral_constant<int, 4>{});
        if constexpr (HD == 128)
            if (most <= 8 * kKv8Threads) return go(std::integral_constant<int, 8>{});
        return go(std::integral_constant<int, 256 * HD / 8 / kKv8Threads>{});
    });
}

static int check_kv8(const fa_kv8_args *p) {
    if (!p) return FA_ERR_INVALID_ARG;
    const fa_kv8_args &a = *p;
    if (a.cache.batch == 0) return FA_OK;  // tensors of no sequences have no address
    int rc = check_kv8_cache(a.cache);
    if (rc == FA_OK) rc = check_kv8_new(a);
    if (rc) return rc;
    if (a.seqlen_q < 0 || a.nheads <= 0 || a.nheads % a.cache.nheads_k || a.num_splits < 0 || a.window_left < -1 ||
        a.window_right < -1 || a.seqlens_new)
        return FA_ERR_INVALID_ARG;
    if (a.seqlen_q == 0) return FA_OK;
    if (!a.lse || check_tensor(a.q, true) || check_tensor(a.o, true)) return FA_ERR_INVALID_ARG;
    const int64_t rows = int64_t(a.nheads / a.cache.nheads_k) * a.seqlen_q;
    if (rows > INT32_MAX / 2) return FA_ERR_INVALID_ARG;
    if (!a.ws || a.ws_bytes < int64_t(fa_kv8_ws_bytes(&a)) || (reinterpret_cast<uintptr_t>(a.ws) & 255u)) return FA_ERR_WORKSPACE;
    return FA_OK;
}

}  // namespace fa

extern "C" int fa_kv8_append(const fa_kv8_args *args, void *stream) {
    using namespace fa;
    if (!args) return FA_ERR_INVALID_ARG;
    if (args->cache.batch == 0) return FA_OK;
    int rc = check_kv8_cache(args->cache);
    if (rc == FA_OK) rc = check_kv8_new(*args);
    if (rc) return rc;
    return launch_kv8_append(*args, nullptr, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t fa_kv8_ws_bytes(const fa_kv8_args *a) {
    if (!a || a->cache.batch <= 0 || a->seqlen_q <= 0 || a->nheads <= 0 || a->cache.nheads_k <= 0) return 0;
    if ((a->cache.head_dim != 64 && a->cache.head_dim != 128) || a->nheads % a->cache.nheads_k) return 0;
    return size_t(fa::kv8_plan(*a).bytes);
}

extern "C" int fa_kv8_attention(const fa_kv8_args *args, void *stream) {
    using namespace fa;
    int rc = check_kv8(args);
    if (rc) return rc;
    fa_kv8_args a = *args;
    if (a.cache.batch == 0) return FA_OK;
    a.window_left = std::min(a.window_left, INT32_MAX / 2);  // positions less a window stay in 32 bits
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (a.seqlen_q == 0) return launch_kv8_append(a, nullptr, s);
    const Kv8Plan plan = kv8_plan(a);
    const int64_t grid = kv8_grid(plan, a.cache.nheads_k / plan.heads);
    if (grid > kKv8MaxGrid) return FA_ERR_INVALID_ARG;
    if ((rc = launch_kv8_append(a, &plan, s))) return rc;
    if (plan.many) return kv8_chunk(a, plan, s);
    return kv8_by_type(a.cache.head_dim, a.dtype, a.cache.kind, [&](auto hd, auto bf, auto int8) {
        constexpr int HD = decltype(hd)::value;
        auto go = [&](auto nh) {
            hipLaunchKernelGGL((kv8_decode_kernel<HD, decltype(bf)::value, decltype(int8)::value, decltype(nh)::value>),
                               dim3(unsigned(grid)), dim3(kKv8Threads), 0, s, Kv8Call{a, plan});
            return int(hipGetLastError());
        };
        if (plan.heads == 2) return go(std::integral_constant<int, 2>{});
        return go(std::integral_constant<int, 1>{});
    });
}

extern "C" int fa_kv8_read(const fa_kv8_read_args *args, void *stream) {
    using namespace fa;
    if (!args) return FA_ERR_INVALID_ARG;
    const fa_kv8_read_args &a = *args;
    if (a.total < 0 || a.cache.batch < 0) return FA_ERR_INVALID_ARG;
    if (a.total == 0) return FA_OK;
    const int rc = check_kv8_cache(a.cache);
    if (rc) return rc;
    if (a.dtype != FA_FP16 && a.dtype != FA_BF16) return FA_ERR_UNSUPPORTED;
    if (!a.cu_seqlens || check_tensor(a.k_out, true) || check_tensor(a.v_out, true)) return FA_ERR_INVALID_ARG;
    const int per = kv8_read_rows(2 * a.cache.nheads_k * (a.cache.head_dim / 8));
    const int64_t grid = (int64_t(a.total) + per - 1) / per;
    if (grid > kKv8MaxGrid) return FA_ERR_INVALID_ARG;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return kv8_by_type(a.cache.head_dim, a.dtype, a.cache.kind, [&](auto hd, auto bf, auto int8) {
        hipLaunchKernelGGL((kv8_read_kernel<decltype(hd)::value, decltype(bf)::value, decltype(int8)::value>),
                           dim3(unsigned(grid)), dim3(kKv8Threads), 0, s, a, per);
        return int(hipGetLastError());
    });
}
