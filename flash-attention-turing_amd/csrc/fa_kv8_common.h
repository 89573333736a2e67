// Shared by the kernels of a key-value cache in 8 bits: codes, places in the cache, and the plan of an attention call.
//
// A value is code * scale, one scale for each block of tokens of a head.  A tile of 32 keys lies in one block, so
// its scales are two numbers of the wave: k's multiplies scores, v's probabilities, and no element is
// ever scaled.  Codes of both types are exact in fp16 and in bf16.
#pragma once

#include <type_traits>

#include "fa_diff_common.h"

namespace fa {

constexpr float kKv8MinScale = 1.17549435e-38f;  // 2^-126

// Eight codes as MFMA operand elements: fp16 (BF: bf16).
template <bool INT8, bool BF>
__device__ __forceinline__ f16x8 kv8_decode(const u32x2 c) {
    u32x4 r;
    if constexpr (!INT8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (BF) {
                r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, false));
                r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, true));
            } else {
                r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, false));
                r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, true));
            }
        }
    } else if constexpr (BF) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float lo = float(int8_t(c[i] >> 16 * h)), hi = float(int8_t(c[i] >> (16 * h + 8)));
                // At most 7 bits: the upper halves of the fp32 words are the bf16 values.
                r[2 * i + h] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
            }
    } else {
        // 0x6400 | u is 1024 + u in fp16, u = code + 128.
        const _Float16 off = _Float16(-1152.f);
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t u = c[i] ^ 0x80808080u;
            const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(u, 0x64646464u, 0x00050004u)) + h2{off, off};
            const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(u, 0x64646464u, 0x00070006u)) + h2{off, off};
            r[2 * i] = __builtin_bit_cast(uint32_t, a);
            r[2 * i + 1] = __builtin_bit_cast(uint32_t, b);
        }
    }
    return as_h8(r);
}

// Chunk c (16 bytes) of row r of 32 rows of codes in LDS sits at chunk c ^ kv8_swz(r).  Every operand read then takes each
// bank once: 16 bytes of one chunk from 16 rows that differ in bits 0 to 3 or in bits 0, 1, 3 and 4, and transposed reads of one
// chunk from 16 rows (bits 0 to 3) or of a pair of chunks from 8 (bits 0 to 2).
template <int HD>
__device__ __forceinline__ int kv8_swz(int r) {
    if constexpr (HD == 128)
        return (r >> 3 & 1) | (r >> 1 & 1) << 1 | ((r >> 4 ^ r >> 2) & 1) << 2;
    else
        return (r >> 3 & 1) | ((r >> 4 ^ r >> 2) & 1) << 1;
}

// ds_read_b64_tr_b8: within 16 lanes, lane i gets byte i % 8 of the 8-byte words at the addresses of lanes 2 j + i / 8,
// j = 0..7.  With lane 2 j + h at row j, bytes 8 h, lane i so holds column i of 8 rows.
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2_t;
__device__ __forceinline__ u32x2 lds_tr8(const char *base, int off) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t *)(base + off)));
}

// Four codes from and to fp32 values in the codes' own units.
template <bool INT8>
__device__ __forceinline__ f32x4 kv8_values(uint32_t c) {
    f32x4 v;
    if constexpr (INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = float(int8_t(c >> 8 * i));
    } else {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
        v = f32x4{a[0], a[1], b[0], b[1]};
    }
    return v;
}
template <bool INT8>
__device__ __forceinline__ uint32_t kv8_codes(const f32x4 v) {
    if constexpr (INT8) {
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) c |= uint32_t(uint8_t(int8_t(int(rintf(v[i]))))) << 8 * i;
        return c;
    } else {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], c, true));
    }
}

// Cache row of sequence b, and what is wrong with it and with its lengths (0: nothing).
__device__ __forceinline__ int kv8_err(const fa_kv8_cache &c, int b, int L0, int n, int most_new, int &row) {
    row = c.cache_batch_idx ? c.cache_batch_idx[b] : b;
    const int err = (L0 < 0 || n < 0 || n > most_new || int64_t(L0) + n > c.cache_capacity ? 1 : 0) |
                    (c.cache_batch_idx && (row < 0 || row >= c.cache_batch) ? 2 : 0);
    if (err) row = 0;
    return err;
}

// Attention's plan, made by one workgroup of the launch before, whatever the capacity is: each sequence's keys cut into as
// many pieces as it has times the batch's keys by the places on the chip, all of one length; a sequence without keys has one
// empty piece.
struct Kv8Slot {
    int b, row;         // sequence, its cache row
    int begin, end;     // keys
    int keys;           // of the sequence
    int ch, n_pieces;   // this piece, and how many the sequence has
    int part;           // the piece among those of sequences with several, whose partial results have places
};
static_assert(sizeof(Kv8Slot) == 32, "one scalar load");

// Workspace: counters of the (sequence, KV heads, row tile) items and of every piece that is one of several (a group of pieces
// counts at its first one's), the slots, then those pieces' partial results.
constexpr int kKdRows = 16, kKcRows = 128;  // rows of a tile: few rows, many
constexpr int kKv8Round = 128;              // pieces have a multiple of so many keys: a tile of every wave, or two of a workgroup's
struct Kv8Plan {
    bool many;          // the kernel of many rows (fa_kv8_fwd.hip)
    int heads;          // KV heads that a workgroup takes together
    int row_tiles;      // of a KV head
    int rows_max;       // rows of a tile whose partial results are kept
    int slots;          // at most
    int fixed;          // keys of a piece, where the call says so, or 0
    int want, most;     // slots that fill the chip, and that run at once
    int least;          // keys of a piece at least
    int64_t items;      // batch * nheads_k / heads * row_tiles
    int64_t counters, at_slots, at_ml, at_o, bytes;
};

// Workgroups of an attention call: its (slot, KV head) groups times row tiles.  The tiles of a group read the same codes, so
// they are dealt to one of the eight XCDs (workgroups go to them in turn), where there are groups enough for all.
__host__ __device__ __forceinline__ bool kv8_by_xcd(const Kv8Plan &p, int nheads_k) {
    return p.row_tiles > 1 && (nheads_k % 8 == 0 || int64_t(p.slots) * nheads_k >= 64);
}
static inline int64_t kv8_grid(const Kv8Plan &p, int nheads_k) {
    const int64_t groups = int64_t(p.slots) * nheads_k;
    return (kv8_by_xcd(p, nheads_k) ? (groups + 7) / 8 * 8 : groups) * p.row_tiles;
}
__device__ __forceinline__ bool kv8_item(const Kv8Plan &p, int nheads_k, int wg, int &slot, int &hk, int &rt) {
    int group = wg / p.row_tiles;
    rt = wg - group * p.row_tiles;
    if (kv8_by_xcd(p, nheads_k)) {
        const int turn = wg / (8 * p.row_tiles), in = wg - turn * 8 * p.row_tiles;
        group = turn * 8 + in % 8;
        rt = in / 8;
    }
    slot = group / nheads_k;
    hk = group - slot * nheads_k;
    return slot < p.slots;
}

// First key that a row at position p sees, and its last one.
__device__ __forceinline__ int kv8_first(const fa_kv8_args &a, int p) { return a.window_left >= 0 ? max(p - a.window_left, 0) : 0; }
__device__ __forceinline__ int kv8_last(const fa_kv8_args &a, int p, int L) {
    const int64_t r = a.causal ? p : a.window_right >= 0 ? int64_t(p) + a.window_right : L - 1;
    return int(min(r, int64_t(L - 1)));
}

// Sum of x over the 256 threads of a workgroup and the sum over those before this one.
__device__ __forceinline__ int64_t kv8_scan(int64_t x, int64_t &total) {
    __shared__ int64_t part[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(inc, d);
        if (lane >= d) inc += y;
    }
    __syncthreads();  // the last call's reads are done
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    int64_t base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        base += w < wave ? part[w] : 0;
        total += part[w];
    }
    return base + inc - x;
}

// Sums of four counts over the 256 threads of a workgroup.
__device__ __forceinline__ void kv8_sums(int64_t (&x)[4]) {
    __shared__ int64_t part[4][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], d);
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = part[0][i] + part[1][i] + part[2][i] + part[3][i];
}

// One workgroup: the slots of an attention call.
__device__ __forceinline__ void kv8_make_plan(const fa_kv8_args &a, const Kv8Plan &plan) {
    __shared__ int before[257], parts_before[256];
    __shared__ int keys_of[256], begin_of[256], row_of[256], piece_of[256];
    const int tid = threadIdx.x;
    Kv8Slot *slots = reinterpret_cast<Kv8Slot *>(static_cast<char *>(a.ws) + plan.at_slots);
    auto sequence = [&](int b, int &begin, int &L, int &row) {
        const int L0 = a.cache_seqlens[b], err = kv8_err(a.cache, b, L0, a.seqlen_new, a.seqlen_new, row);
        if (err && a.cache.status) atomicOr(a.cache.status, err);
        L = err ? 0 : L0 + a.seqlen_new;
        begin = min(kv8_first(a, max(L - a.seqlen_q, 0)), L) / 32 * 32;
    };
    int piece = plan.fixed;
    if (piece == 0) {
        int64_t sum = 0, total;
        for (int b = tid; b < a.cache.batch; b += 256) {
            int begin, L, row;
            sequence(b, begin, L, row);
            sum += L - begin;
        }
        kv8_scan(sum, total);
        // x times the even share of n places, a little more for the rounding of 32 bits, in whole rounds.
        auto length = [&](float x, int n) {
            const float share = fminf(float(total) * x / float(n) * 1.000001f, float(1 << 30));
            return int(max(uint32_t(plan.least), (uint32_t(share) / kKv8Round + 1) * kKv8Round));
        };
        piece = length(1.f, plan.want);
        // Few rows, where a piece costs little besides its codes: the shortest of four lengths whose pieces all run at once, at one
        // workgroup a CU or else at two; where none fits, as with lengths far apart, half the share of these: pieces that start as
        // places become free.  Measured (us, one and two a CU): 64 x 8192 172 and 186, 4 x 48000 37 and 40, 2 x 9000 22 and 24;
        // two a CU and half their share: 64 x 1024-16384 188 and 172.
        const int at[8] = {piece, length(1.0625f, plan.want), length(1.125f, plan.want), length(1.25f, plan.want),
                           length(1.f, plan.most), length(1.0625f, plan.most), length(1.125f, plan.most), length(1.25f, plan.most)};
        if (!plan.many && a.cache.batch > 1 && at[3] > plan.least) {
            float inv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) inv[i] = 1.f / float(at[i]);
            // (Counts of 32-bit quotients: a length that is wrongly taken for fitting, or not, is as good.)
            int64_t n[4] = {};  // two counts each
            for (int b = tid; b < a.cache.batch; b += 256) {
                int begin, L, row;
                sequence(b, begin, L, row);
                auto pieces = [&](int i) { return int64_t(max(1, int(float(L - begin - 1) * inv[i]) + 1)); };
#pragma unroll
                for (int i = 0; i < 4; ++i) n[i] += pieces(2 * i) << 32 | pieces(2 * i + 1);
            }
            kv8_sums(n);
            piece = length(0.5f, plan.most);
#pragma unroll
            for (int i = 7; i >= 0; --i)
                if ((i % 2 ? n[i / 2] & 0xffffffff : n[i / 2] >> 32) <= (i < 4 ? plan.want : plan.most)) piece = at[i];
        }
    }
    int64_t done = 0, parts_done = 0;
    for (int b0 = 0; b0 < a.cache.batch; b0 += 256) {
        const int b = b0 + tid;
        int begin = 0, L = 0, row = 0, n = 0;
        if (b < a.cache.batch) {
            sequence(b, begin, L, row);
            n = max(1, int((uint32_t(L - begin) + uint32_t(piece) - 1) / uint32_t(piece)));
        }
        // (Both counts in one sum: a launch has less than 2^24 slots.)
        int64_t totals;
        const int64_t at = kv8_scan(int64_t(n > 1 ? n : 0) << 32 | n, totals);
        const int total = int(totals & 0xffffffff);
        before[tid] = int(at & 0xffffffff);
        parts_before[tid] = int(at >> 32);
        keys_of[tid] = L;
        begin_of[tid] = begin;
        row_of[tid] = row;
        // Pieces of few rows are equal: they end together.  Those of many rows keep the length, whose places run one each, and
        // the short last ones fill what is left: 3 + 2 pieces on 4 places took 204 us equal and 172 us so.
        const uint32_t parts = max(n, 1), even = (uint32_t(L - begin) + parts - 1) / parts;
        piece_of[tid] = plan.fixed || plan.many ? piece : int((even + kKv8Round - 1) / kKv8Round * kKv8Round);
        if (tid == 0) before[256] = total;
        __syncthreads();
        for (int64_t s = tid; s < total && done + s < plan.slots; s += 256) {
            int lo = 0;  // the last sequence whose first slot is at or before s
#pragma unroll
            for (int d = 128; d > 0; d >>= 1)
                if (before[lo + d] <= s) lo += d;
            Kv8Slot x;
            x.b = b0 + lo;
            x.row = row_of[lo];
            x.ch = int(s) - before[lo];
            x.keys = keys_of[lo];
            x.n_pieces = before[lo + 1] - before[lo];
            x.begin = min(x.keys, begin_of[lo] + x.ch * piece_of[lo]);
            x.end = min(x.keys, x.begin + piece_of[lo]);
            x.part = int(parts_done) + parts_before[lo] + x.ch;
            slots[done + s] = x;
        }
        done += total;
        parts_done += totals >> 32;
        __syncthreads();
    }
    for (int64_t s = done + tid; s < plan.slots; s += 256) slots[s].b = -1;
}

// What the attention kernels are called with.  kv8_late reads it anew from where it is used: all of it at once does not fit the
// scalar registers, and what does not is moved to vector lanes and back, which cost a call of one token 1.3 us.
struct Kv8Call {
    fa_kv8_args a;
    Kv8Plan plan;
};
__device__ __forceinline__ const Kv8Call &kv8_late() {
    typedef const __attribute__((address_space(4))) void *Args;
    Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Kv8Call *)p;
}

// Brings the whole of it to the scalar cache at a kernel's start, where all the lines' latencies are one (0.6 us of a call of one token).
__device__ __forceinline__ void kv8_early() {
    typedef const __attribute__((address_space(4))) uint32_t *Args;
    const Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    uint32_t x[(sizeof(Kv8Call) + 63) / 64];
#pragma unroll
    for (size_t i = 0; i < sizeof(x) / 4; ++i) x[i] = p[16 * i];
#pragma unroll
    for (size_t i = 0; i < sizeof(x) / 4; ++i) asm volatile("" ::"s"(x[i]));
}

// A wave-uniform slot, through the scalar cache.
__device__ __forceinline__ Kv8Slot kv8_slot(const fa_kv8_args &a, const Kv8Plan &plan, int i) {
    typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
    const i32x8 *s = reinterpret_cast<const i32x8 *>(static_cast<const char *>(a.ws) + plan.at_slots) + i;
    return __builtin_bit_cast(Kv8Slot, i32x8(*(const __attribute__((address_space(4))) i32x8 *)uniform(s)));
}

// Writes one row of the output: x holds channels d and d + 1 over the sum l.
template <int HD, bool BF>
__device__ __forceinline__ void kv8_store(const fa_kv8_args &a, int b, int hk, int row, int d, f32x2 x, float m, float l) {
    const int G = a.nheads / a.cache.nheads_k, qp = row / G, h = hk * G + row - qp * G;
    // A sum of 0 is that of a row without a visible key (or with scores of -infinity alone); NaN goes on to the output.
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const f16x4 y = l == 0.f ? pack4<BF>(0.f, 0.f, 0.f, 0.f) : pack4<BF>(x[0] * inv, x[1] * inv, 0.f, 0.f);
    f16 *out = (f16 *)a.o.ptr + int64_t(b) * a.o.batch_stride + int64_t(qp) * a.o.row_stride + int64_t(h) * a.o.head_stride + d;
    *reinterpret_cast<uint32_t *>(out) = __builtin_bit_cast(u32x2, y)[0];
    if (d == 0) a.lse[(int64_t(b) * a.nheads + h) * a.seqlen_q + qp] = l == 0.f ? 0.f : (m + log2_fast(l)) * kLn2;
}

// Partial results of a piece: rows_max (maximum, sum) pairs and rows_max x HD / 2 pairs of unnormalised fp32 O.
__device__ __forceinline__ uint64_t *kv8_ml(const fa_kv8_args &a, const Kv8Plan &p, int64_t part) {
    return reinterpret_cast<uint64_t *>(static_cast<char *>(a.ws) + p.at_ml) + part * p.rows_max;
}
template <int HD>
__device__ __forceinline__ uint64_t *kv8_o(const fa_kv8_args &a, const Kv8Plan &p, int64_t part) {
    return reinterpret_cast<uint64_t *>(static_cast<char *>(a.ws) + p.at_o) + part * p.rows_max * (HD / 2);
}
__device__ __forceinline__ void kv8_put(uint64_t *p, f32x2 x) {
    __hip_atomic_store(p, __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 kv8_get(const uint64_t *p) {
    return __builtin_bit_cast(f32x2, __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Counts a piece whose partial results are stored; true in the workgroup that counts last of n.
__device__ __forceinline__ bool kv8_count(int32_t *count, int n, int *ticket) {
    wait_vmem();
    __syncthreads();  // every wave's stores have completed
    if (threadIdx.x == 0) *ticket = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    return *ticket == n - 1;
}

// Pieces of an item are joined in one step, or, where their partial results (bytes each for a KV head) are many, eight at a time
// by the last workgroup of the eight, whose result takes the place of the first one's, and then these: one workgroup would read
// too long.  Measured (us, one step and two): 4 x 48000 tokens in 40 pieces of 4 KB 51.5 and 49.5, 1 x 65536 in 64 pieces of 4 KB
// 38 and 33; 8 heads of 128 channels, 1 x 65536 in 40 pieces of 2 KB 45 and 47.
__device__ __forceinline__ int kv8_group(int n_pieces, int bytes) {
    return n_pieces <= 8 || int64_t(n_pieces) * bytes <= 128 << 10 ? n_pieces : 8;
}
__device__ __forceinline__ int32_t *kv8_counter(const fa_kv8_args &a, int64_t i) { return static_cast<int32_t *>(a.ws) + i; }

// Joins the n pieces of an item in their order, by the 256 threads: thread units of (row, two channels), kKv8Join pieces at a
// time, whose loads are in flight together.  scratch: LDS of ROWS (kKv8Join + 2) floats.  part(i) is the place of piece i's partial
// results, write(row, channel, its and the next one's unnormalised O, maximum, sum) takes the joined ones.
// A row's bits are the same for any ROWS: sums of pieces i, i + 16, .. are kept apart and added in one order.
constexpr int kKv8Join = 64, kKv8Apart = 16;
template <int HD, int ROWS, int UNITS, class Part, class Write>
__device__ __forceinline__ void kv8_join(const fa_kv8_args &a, const Kv8Plan &plan, int rows, int n, float *scratch, Part part,
                                         Write write) {
    constexpr int T = 256 / ROWS, PER = kKv8Join / T;  // threads a row that weigh its pieces, pieces of each
    constexpr int AHEAD = 32 / UNITS;
    constexpr int A = kKv8Apart / T;  // sums of a thread
    static_assert(AHEAD >= 1 && kKv8Join % AHEAD == 0 && kKv8Join % T == 0 && kKv8Apart % T == 0 && PER % A == 0, "whole rounds");
    float *old = scratch, *sum = scratch + ROWS, *weight = scratch + 2 * ROWS;
    const int tid = threadIdx.x, r = tid / T, t = tid % T;
    float mm = -INFINITY, ll[A] = {};
    f32x2 x[UNITS] = {};
    for (int i0 = 0; i0 < n; i0 += kKv8Join) {
        const int k = min(kKv8Join, n - i0);
        f32x2 ml[PER], y[AHEAD][UNITS];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = t + j * T;
            ml[j] = r < rows && i < k ? kv8_get(kv8_ml(a, plan, part(i0 + i)) + r) : f32x2{-INFINITY, 0.f};
        }
        auto load = [&](int i) FA_INLINE {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    const int e = u * 256 + tid;
                    y[j][u] = i + j < k && e < rows * (HD / 2) ? kv8_get(kv8_o<HD>(a, plan, part(i0 + i + j)) + e) : f32x2{0.f, 0.f};
                }
        };
        load(0);
        float top = mm;
#pragma unroll
        for (int j = 0; j < PER; ++j) top = fmaxf(top, ml[j][0]);
#pragma unroll
        for (int d = 1; d < T; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        const float f0 = mm == -INFINITY ? 0.f : exp2_fast(mm - top);
#pragma unroll
        for (int j = 0; j < A; ++j) ll[j] *= f0;
        mm = top;
        __syncthreads();  // the weights before are used up
        if (t == 0) old[r] = f0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float f = ml[j][0] == -INFINITY ? 0.f : exp2_fast(ml[j][0] - top);
            weight[(t + j * T) * ROWS + r] = f;
            ll[j % A] = fmaf(ml[j][1], f, ll[j % A]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const float f = old[min((u * 256 + tid) / (HD / 2), ROWS - 1)];
            x[u][0] *= f;
            x[u][1] *= f;
        }
        for (int i = 0; i < k; i += AHEAD) {
            if (i > 0) load(i);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    const float f = i + j < k ? weight[(i + j) * ROWS + min((u * 256 + tid) / (HD / 2), ROWS - 1)] : 0.f;
                    x[u][0] = fmaf(f, y[j][u][0], x[u][0]);
                    x[u][1] = fmaf(f, y[j][u][1], x[u][1]);
                }
        }
    }
    // (Sums i and i + 8 first, whether they are one thread's or two threads'.)
#pragma unroll
    for (int d = A / 2; d > 0; d >>= 1)
#pragma unroll
        for (int j = 0; j < d; ++j) ll[j] += ll[j + d];
#pragma unroll
    for (int d = T / 2; d > 0; d >>= 1) ll[0] += __shfl_xor(ll[0], d);
    __syncthreads();
    if (t == 0) {
        old[r] = mm;
        sum[r] = ll[0];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int e = u * 256 + tid, row = e / (HD / 2);
        if (row < rows) write(row, 2 * (e % (HD / 2)), x[u], old[row], sum[row]);
    }
}

// The call with its sizes as types: f(head_dim, bf16, int8).
template <class F>
static int kv8_by_type(int head_dim, int dtype, int kind, F f) {
    auto by_kind = [&](auto hd, auto bf) {
        return kind == FA_KV8_INT8 ? f(hd, bf, std::true_type{}) : f(hd, bf, std::false_type{});
    };
    auto by_dtype = [&](auto hd) { return dtype == FA_BF16 ? by_kind(hd, std::true_type{}) : by_kind(hd, std::false_type{}); };
    return head_dim == 128 ? by_dtype(std::integral_constant<int, 128>{}) : by_dtype(std::integral_constant<int, 64>{});
}

}  // namespace fa
