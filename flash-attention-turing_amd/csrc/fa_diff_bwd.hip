// Differential attention, backward.
//
//   dP = dO v^T (shared by both maps), D_m = rowsum(P_m * dP) = dO . O_m
//   dS_1 = P_1 (dP - D_1),  dS_2 = -lam P_2 (dP - D_2)
//   dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dv = (P_1 - lam P_2)^T dO
//   dlam = -D_2, summed over the rows and heads that share a lam
// with P_m = exp(scale S_m - LSE_m), 0 where masked.  o = O_1 - lam O_2 and the
// forward's O_2 give D_2 = dO . O_2 and D_1 = dO . o + lam D_2.
//
// dQ kernel: 4 waves x 32 queries, S^T and dP^T with keys on the MFMA M
// dimension, so a lane owns one query.  dQ_2's factor -lam belongs to the query
// and is applied once at the end.  D_m from 16-bit O_m is off by up to half a
// unit in its last place: enough for dS, where it weighs as the other
// roundings do, but neither for dlam, which is D_2 itself, nor for rows of a few keys, whose dP -
// D_m cancels.  So the kernel sums dS_2, which is D_2's error, in fp32
// (sum_j P_2 (dP - D) = D_2 - D), and rows whose keys lie in the first block
// take both D_m from that block's own P_m and dP.  The matrix cores' sums lean
// towards minus infinity by a small part of a unit (here about 3e-8), the same
// way in every row, and the D_2 of 10^5 rows and more, whose signs vary, sum to
// so little that this showed in a dlam they share (1.5e-4 of it at 2 x 4096
// rows, 8 heads).  So every second query computes with -dO: its lane's sums are the
// negatives, at no cost until the end, and the leanings of neighbours cancel.
//
// dK/dV kernel: 4 waves x 32 keys of one KV head, S and dP with queries on M.
// It loops over the heads of the GQA group and sums them in fp32 registers.
//
// What bounds both is the matrix cores beside the VALU: dQ takes 48 MFMAs and 290
// VALU instructions (64 exponentials) for 32 queries x 64 keys at 128 channels,
// dK/dV 36 (4 of them for the row operands) and 210 for 32 x 32.  Counters: MFMA 48
// to 55 and 58 to 61 % of dQ's and dK/dV's cycles, VALU 60 to 64 and 54 to 57 %.
// b 4, s 4096, 16 heads of 128, causal, bf16: dQ 520 us, dK/dV 655 us (793 and 839
// TFLOP/s of the formulas' products); b 1, s 8192, 32/8 heads, fp16: 925 and 1215 us
// (892 and 905); a library product of 8192^3 runs at 1224 to 1280.
#include <algorithm>
#include <type_traits>

#include "fa_diff_common.h"

namespace fa {

constexpr int kDbThreads = 256;
// The workspace: -D_2 of every row in fp32 (for dlam), then DiffRowOps of every row.
//
// What the dK/dV kernel needs of a query row (its LSEs, D_m and lam) belongs to
// the M dimension of its products, so a lane would need all 16 rows' values of
// its accumulators: 24 16-byte LDS reads per 32 x 32 tile, a quarter of the LDS
// time that bounded the kernel.  Instead the row's values enter the products, as
// one more K step, of bf16 whatever the tensors' type: a value v is the sum of three
// bf16 numbers, each the rounding of what the ones before leave, which is v to 2^-27
// of it (fp32 itself holds 2^-24) over all of fp32's range, and NaN if v is.  (fp16
// pieces with weights held v up to 1.7e7 only, which D passes with a large dO, and
// LSE / scale with a small scale.)  The scores so come out as S_m - LSE_m / scale, with
// log2 |lam| taken off LSE_2, and dP as dP - D_1 and, by one more product, dP - D_2.
// The sign of lam goes in the fourth place, whose weight is 0.
struct DiffRowOps {
    f16x4 lse1, lse2, nd1, e;  // bf16 bits of -LSE_1 / scale, -(LSE_2 - log |lam|) / scale, -D_1, D_1 - D_2
};
static_assert(sizeof(DiffRowOps) == 32, "copied as 32 rows a KiB");

// Scales below this count as 0 in the dK/dV kernel's scores, so that LSE / scale stays within fp32: they
// move the exponent of a raw score up to 2^75 by less than 2^-25 (fp16 products are below 2^39).
constexpr float kDiffFlatScale = 0x1p-100f;

__device__ __forceinline__ f16x4 row_op(float v, float fourth) {
    const float hi = float((__bf16)v), mid = float((__bf16)(v - hi));
    return pack4<true>(hi, mid, (v - hi) - mid, fourth);
}
// B operand that takes the first (which = 0) or second of two row_ops in an A
// operand: K slots 0..3 and 4..7 of the lower lane half, the upper half's are 0.
__device__ __forceinline__ f16x8 row_weights(int which, int hh) {
    const float one = hh ? 0.f : 1.f;
    const f16x4 w = pack4<true>(one, one, one, 0.f), z = pack4<true>(0.f, 0.f, 0.f, 0.f);
    return which ? __builtin_shufflevector(z, w, 0, 1, 2, 3, 4, 5, 6, 7) : __builtin_shufflevector(w, z, 0, 1, 2, 3, 4, 5, 6, 7);
}

__host__ __device__ __forceinline__ int64_t diff_plane(const fa_diff_bwd_args &a) {
    return int64_t(a.batch) * a.nheads * a.lse_seqlen;
}

// Floats from the start of the workspace to the row operands (32-byte aligned from a 32-byte aligned start).
__host__ __device__ __forceinline__ int64_t diff_ops_at(const fa_diff_bwd_args &a) { return (diff_plane(a) + 7) & ~int64_t(7); }

// Shared dK/dV items (diff_dkdv_kernel, SPLIT): split_ws starts with an int32
// counter per (batch, key block, KV head), then, 256-byte aligned, come the fp32
// partial sums.  The dQ kernel, which precedes it on the stream, clears the counters.
__host__ __device__ __forceinline__ int64_t diff_dkdv_items(const fa_diff_bwd_args &a) {
    return int64_t((a.seqlen_k + 127) / 128) * a.batch * a.nheads_k;
}
__host__ __device__ __forceinline__ int64_t diff_dkdv_count_bytes(int64_t items) { return (items * 4 + 255) & ~int64_t(255); }

template <int HD, bool BF, bool CAUSAL>
__global__ __launch_bounds__(kDbThreads, HD == 64 ? 3 : 2) void diff_dq_kernel(const fa_diff_bwd_args a, const int num_m_blocks,
                                                                const int lg) {
    constexpr int NT = kDbThreads, BM = 128, BN = 64;
    constexpr int TILE = BN * HD * 2, STAGE = 2 * TILE;
    constexpr int HG = HD / 32;  // MFMA K steps of one map's channels
    constexpr int PIPE = 3;
    constexpr int KT = HD == 64 ? 1 : 2;  // 32-key tiles at a time
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];

    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (a.split_ws) {
        const int64_t n = diff_dkdv_items(a);
        for (int64_t i = int64_t(blockIdx.x) * NT + tid; i < n; i += int64_t(gridDim.x) * NT)
            static_cast<int32_t *>(a.split_ws)[i] = 0;
    }
    const int packs = a.nheads >> lg, P = BM >> lg;
    int b, h, mb;
    if (a.work_order && a.cu_seqlens_q) {
        const int nnb = (a.seqlen_k + 127) / 128;
        const int it = a.work_order[int64_t(a.batch) * nnb + blockIdx.x / packs];
        if (it < 0) return;
        b = __builtin_amdgcn_readfirstlane(it / num_m_blocks);
        mb = __builtin_amdgcn_readfirstlane(it - b * num_m_blocks);
        h = (blockIdx.x % packs) << lg;
    } else {
        const int bp_count = a.batch * packs, bp = blockIdx.x % bp_count;
        mb = blockIdx.x / bp_count;
        if (CAUSAL) mb = num_m_blocks - 1 - mb;
        b = bp / packs;
        h = (bp - b * packs) << lg;
    }
    const int hk = h / (a.nheads / a.nheads_k);
    const bool packed_q = a.cu_seqlens_q != nullptr, packed_k = a.cu_seqlens_k != nullptr;
    const DiffRows rq = diff_rows(a.cu_seqlens_q, b, a.seqlen_q, a.dq_rows), rk = diff_rows(a.cu_seqlens_k, b, a.seqlen_k, a.dkv_rows);
    const int sq = rq.n, sk = rk.n, m0 = mb * P;
    if (m0 >= sq) return;
    h += wave >> (2 - lg);

    const f16 *kp = (const f16 *)a.k.ptr + base_off(a.k, packed_k, b, rk.start, hk);
    const f16 *vp = (const f16 *)a.v.ptr + base_off(a.v, packed_k, b, rk.start, hk);
    const int64_t krs = a.k.row_stride, vrs = a.v.row_stride;
    const int causal_off = sk - sq;
    int n_end = sk;
    if (CAUSAL) n_end = max(0, min(sk, m0 + P + causal_off));
    const int n_blocks = (n_end + BN - 1) / BN;
    const float cs = uniform(a.softmax_scale * kLog2e);

    DiffCopier<HD, BN, NT> cp;
    cp.init(wave, lane);
    auto issue = [&](int nb, int st) FA_INLINE {
        const int n0 = nb * BN;
        const uint32_t tile = lds_addr(smem) + st * STAGE;
        cp.copy(tile, kp + int64_t(n0) * krs, krs, sk - n0);
        cp.copy(tile + TILE, vp + int64_t(n0) * vrs, vrs, sk - n0);
    };
    if (n_blocks > 0) issue(0, 0);

    // Q^T, dO^T as B operands and this lane's half of the row's D.
    const int q_lo = m0 + 32 * (wave & ((P >> 5) - 1));
    const int qi = q_lo + (lane & 31);
    const bool qv = qi < sq;
    const int qr = qv ? qi : 0;
    const float sgn = qi & 1 ? -1.f : 1.f;  // dO, D_m, dS_m and dQ below are sgn times their values
    f16x8 qB[HD / 16], doB[HD / 16];
    float d1 = 0.f, d2 = 0.f;
    {
        const f16 *qp = (const f16 *)a.q.ptr + base_off(a.q, packed_q, b, rq.start, h) + qr * a.q.row_stride + 8 * hh;
        const f16 *dop =
            (const f16 *)a.dout.ptr + base_off(a.dout, packed_q, b, rq.start, h) + qr * a.dout.row_stride + 8 * hh;
        const f16 *op = (const f16 *)a.o.ptr + base_off(a.o, packed_q, b, rq.start, h) + qr * a.o.row_stride + 8 * hh;
        const f16 *o2p =
            (const f16 *)a.o2.ptr + base_off(a.o2, packed_q, b, rq.start, h) + qr * a.o2.row_stride + 8 * hh;
#pragma unroll
        for (int g = 0; g < HD / 16; ++g) {
            qB[g] = as_h8(qv ? ldg16(qp + 16 * g) : zero_u4());
            const u32x4 dx = qv ? ldg16(dop + 16 * g) : zero_u4();
            doB[g] = as_h8(qi & 1 ? neg_h8(dx) : dx);
            const f16x8 ov = as_h8(qv ? ldg16(op + 16 * g) : zero_u4());
            const f16x8 o2v = as_h8(qv ? ldg16(o2p + 16 * g) : zero_u4());
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float x = elem<BF>(doB[g], t);
                d1 += elem<BF>(ov, t) * x;
                d2 += elem<BF>(o2v, t) * x;
            }
        }
    }
    const float lam = qv ? diff_lam(a.lam, b, rq.start + qi, h) : 0.f;
    const int64_t lrow = (int64_t(b) * a.nheads + h) * a.lse_seqlen;
    const int64_t plane = diff_plane(a);
    const float lse1 = qv ? a.lse[lrow + qi] * kLog2e : 0.f, lse2 = qv ? a.lse[plane + lrow + qi] * kLog2e : 0.f;
    d2 = sum_xor32(d2);
    d1 = fmaf(lam, d2, sum_xor32(d1));
    // All keys of the wave's rows in block 0: D_m from that block.
    const bool one = (CAUSAL ? min(sk, q_lo + 32 + causal_off) : sk) <= 32 * KT;
    if (one) d1 = d2 = 0.f;
    float ds2_sum = 0.f;  // this lane half's sum of P_2 (dP - D_2)

    f32x16 dq[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) dq[i] = zero16();
    TileReader<HD> rd;
    rd.init(lane);

    auto block = [&](int nb, auto mask_tag) FA_INLINE {
        constexpr bool MASK = decltype(mask_tag)::value;
        const int buf = nb & 1, n0 = nb * BN;
        wait_vmem();
        __syncthreads();  // block nb is in LDS; every wave is done with stage buf ^ 1
        if (nb + 1 < n_blocks) issue(nb + 1, buf ^ 1);
        if (CAUSAL && MASK && n0 > q_lo + 31 + causal_off) return;
        if (q_lo >= sq) return;
        const int soff = buf * STAGE;
        static_assert(STAGE % 512 == 0, "stage offsets must be multiples of 512 bytes");
        int ab = rd.a_base + soff, tb0 = rd.tr_base[0] + soff, tb1 = rd.tr_base[1] + soff;
        asm volatile("" : "+v"(ab), "+v"(tb0), "+v"(tb1));
        const int lim = (CAUSAL ? min(sk - 1, qi + causal_off) : sk - 1) - n0;
        f16x8 op[PIPE];
#pragma unroll
        for (int sub = 0; sub < BN / 32; sub += KT) {
            f32x16 dp[KT];
            // dP^T from -D_1 on, so that the product comes out as dP - D_1.
            {
                float nd = -d1;
                asm volatile("" : "+v"(nd));
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[t][i] = nd;
            }
            auto rd_dp = [&](int u) FA_INLINE {
                op[u % PIPE] = rd.a_operand_at(smem + TILE + 32 * (sub + u % KT) * (HD * 2), ab, u / KT);
            };
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < PIPE - 1; ++u) rd_dp(u);
#pragma unroll
            for (int u = 0; u < KT * HD / 16; ++u) {
                if (u + PIPE - 1 < KT * HD / 16) rd_dp(u + PIPE - 1);
                dp[u % KT] = mfma16<BF>(op[u % PIPE], doB[u / KT], dp[u % KT]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                f32x16 s[KT];
                auto rd_k = [&](int u) FA_INLINE {
                    op[u % PIPE] = rd.a_operand_at(smem + 32 * (sub + u % KT) * (HD * 2), ab, m * HG + u / KT);
                };
#pragma unroll
                for (int u = 0; u < PIPE - 1 && u < KT * HG; ++u) rd_k(u);
#pragma unroll
                for (int u = 0; u < KT * HG; ++u) {
                    if (u + PIPE - 1 < KT * HG) rd_k(u + PIPE - 1);
                    s[u % KT] = mfma16<BF>(op[u % PIPE], qB[m * HG + u / KT], u < KT ? zero16() : s[u % KT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // dQ_m^T += K_m^T dS_m^T: step u is key step u / DT, channel tile u % DT of the map;
                // the first reads go out before the exponentials, which cover their latency.
                constexpr int DT = HD / 64;  // 32-channel tiles of a map
                auto rd_dq = [&](int u) FA_INLINE {
                    op[u % PIPE] = rd.tr_operand_at(smem + 16 * (2 * sub + u / DT) * (HD * 2), tb0, tb1, m * DT + u % DT);
                };
#pragma unroll
                for (int u = 0; u < PIPE - 1; ++u) rd_dq(u);
                const float lse = m == 0 ? lse1 : lse2;
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float x = exp2_fast(fmaf(s[t][r], cs, -lse));
                        if constexpr (MASK) x = (sub + t) * 32 + acc_lrow(r, hh) > lim ? 0.f : x;
                        s[t][r] = x;
                    }
                float e = m == 0 ? 0.f : d1 - d2;
                if constexpr (MASK) {
                    if (one && sub == 0) {
                        float d = 0.f;
#pragma unroll
                        for (int t = 0; t < KT; ++t)
#pragma unroll
                            for (int r = 0; r < 16; ++r) d = fmaf(s[t][r], dp[t][r], d);
                        d = sum_xor32(d);
                        e = -d;
                        (m == 0 ? d1 : d2) = d;
                    }
                }
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if (m == 0 && !MASK) {
                            s[t][r] *= dp[t][r];
                        } else {
                            s[t][r] *= dp[t][r] + e;
                            if (m == 1) sum += s[t][r];
                        }
                    }
                if (m == 1) ds2_sum += sum;
                f16x8 dsB[2 * KT];
#pragma unroll
                for (int gg = 0; gg < 2 * KT; ++gg) dsB[gg] = pack16<BF>(s[gg >> 1], 8 * (gg & 1));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < 2 * KT * DT; ++u) {
                    if (u + PIPE - 1 < 2 * KT * DT) rd_dq(u + PIPE - 1);
                    dq[m * DT + u % DT] = mfma16<BF>(op[u % PIPE], dsB[u / DT], dq[m * DT + u % DT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    // Blocks [0, n_full) are fully visible to every row of the workgroup; where
    // a wave's rows see block 0 alone, that block is taken as a masked one.
    int n_full = min(n_blocks, sk / BN);
    if (CAUSAL) n_full = min(n_full, max(0, (m0 + causal_off + 1) / BN));
    if (n_full == 1 && (CAUSAL ? min(sk, m0 + 32 + causal_off) : sk) <= 32 * KT) n_full = 0;
    for (int nb = 0; nb < n_full; ++nb) block(nb, std::false_type{});
    for (int nb = n_full; nb < n_blocks; ++nb) block(nb, std::true_type{});

    ds2_sum = sum_xor32(ds2_sum);
    if (!qv) return;
    if (hh == 0) {
        const float D1 = sgn * d1, D2 = sgn * (d2 + ds2_sum);
        // exp2(cs (S - LSE / cs)); with a scale of 0 the dK/dV kernel takes scores of 0 and cs = 1.
        const float per = fabsf(a.softmax_scale) < kDiffFlatScale ? -1.f : -1.f / cs;
        // A lam of 0 (or subnormal, which the logarithm does not take): 2^-1000 is 0.  (A NaN is neither.)
        const float l2 = fabsf(lam) < 0x1p-126f ? lse2 + 1000.f : lse2 - log2_fast(fabsf(lam));
        a.dsum[lrow + qi] = -D2;
        DiffRowOps *ops = reinterpret_cast<DiffRowOps *>(a.dsum + diff_ops_at(a)) + lrow + qi;
        *ops = DiffRowOps{row_op(lse1 * per, 0.f), row_op(l2 * per, lam < 0.f ? -1.f : 1.f), row_op(-D1, 0.f), row_op(D1 - D2, 0.f)};
    }
    int qo = qi;
    asm volatile("" : "+v"(qo));
    f16 *row = (f16 *)a.dq.ptr + base_off(a.dq, packed_q, b, rq.start, h) + int64_t(qo) * a.dq.row_stride;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) {
        const float f = sgn * (dt < HD / 64 ? a.softmax_scale : -lam * a.softmax_scale);
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4)
            *reinterpret_cast<f16x4 *>(row + dt * 32 + 8 * a4 + 4 * hh) =
                pack4<BF>(dq[dt][4 * a4] * f, dq[dt][4 * a4 + 1] * f, dq[dt][4 * a4 + 2] * f, dq[dt][4 * a4 + 3] * f);
    }
}

// ---------------------------------------------------------------------------
// dK/dV: workgroup = 128 keys of one (batch, KV head), wave w keys 32 w .. + 31.
// K rows live in registers (S's B operands), V rows in LDS (dP's), and every
// 32-query block of Q, dO and the rows' D, LSE and lam goes HBM -> LDS in two
// stages.  With lp = lam P_2: P = P_1 - lp feeds dV, dS_1 = P_1 (dP - D_1) and
// lp (dP - D_2) feed dK; the latter's sign is applied at the end.  At 128 channels
// MFMA and VALU bound it (58 to 61 and 54 to 57 % of the cycles; LDS issue 12 to 13
// %).  At 64 channels neither does (37 and 58 %): its waves wait 31 % of the time, two
// workgroups a CU being too few to fill in, and three spill.  SPLIT: S workgroups
// share the steps (heads of the group x query blocks) of an item and sum their
// dK / dV (diff_dkdv_sum).
//
// Of an item's S workgroups each stores its partial sums and then counts itself;
// the one that counts last, or finds all others counted before it has stored
// anything, adds them in the order of their shares: the sum does not depend on
// who came last, and none waits.  Stores and loads at agent scope, 8 bytes a lane.
template <int HD>
__device__ __forceinline__ bool diff_dkdv_sum(const fa_diff_bwd_args &a, int item, int part, int S, int *ticket,
                                              f32x16 (&dk)[HD / 32], f32x16 (&dv)[HD / 32]) {
    constexpr int N = HD / 2;  // pairs of floats a lane holds: dK, then dV
    const int tid = threadIdx.x;
    int32_t *count = static_cast<int32_t *>(a.split_ws) + item;
    uint64_t *slots = reinterpret_cast<uint64_t *>(static_cast<char *>(a.split_ws) + diff_dkdv_count_bytes(diff_dkdv_items(a))) +
                      int64_t(item) * S * N * kDbThreads + tid;
    if (tid == 0) *ticket = part < 2 ? __hip_atomic_load(count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    __syncthreads();
    if (*ticket != S - 1) {
        uint64_t *own = slots + int64_t(part) * N * kDbThreads;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const f32x16 &t = i < N / 2 ? dk[i / 8] : dv[i / 8 - N / 16];
            const f32x2 x = {t[2 * (i & 7)], t[2 * (i & 7) + 1]};
            __hip_atomic_store(own + i * kDbThreads, __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        }
        wait_vmem();
        __syncthreads();  // every wave's stores have completed
        if (tid == 0) *ticket = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (*ticket != S - 1) return false;
    }
    // Its own share stays in registers when it is one of the first two (x0 + x1 = x1 + x0).
    if (part >= 2) {
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) dk[i] = dv[i] = zero16();
    }
    for (int p = 0; p < S; ++p) {
        if (p == part && part < 2) continue;
        const uint64_t *slot = slots + int64_t(p) * N * kDbThreads;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const f32x2 x = __builtin_bit_cast(
                f32x2, __hip_atomic_load(slot + i * kDbThreads, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            f32x16 &t = i < N / 2 ? dk[i / 8] : dv[i / 8 - N / 16];
            t[2 * (i & 7)] += x[0];
            t[2 * (i & 7) + 1] += x[1];
        }
    }
    return true;
}

template <int HD, bool BF, bool CAUSAL, bool SPLIT>
__global__ __launch_bounds__(kDbThreads, 2) void diff_dkdv_kernel(const fa_diff_bwd_args a, const int nnb, const int S) {
    constexpr int NT = kDbThreads, BN = 128, BM = 32;
    constexpr int QTILE = BM * HD * 2, STAGE = 2 * QTILE + 1024;  // Q, dO, row operands
    constexpr int HG = HD / 32, DT = HD / 64;
    // The last KL of a wave's K operands wait in LDS: with all of them the registers
    // do not hold what the interleaved block below needs.
    constexpr int KL = HD == 128 ? 2 : 0, KR = HD / 16 - KL, KAT = 2 * STAGE + BN * HD * 2;
    __shared__ __attribute__((aligned(16))) char smem[KAT + 4 * KL * 1024];
    __shared__ int ticket;
    static_assert(2 * (KAT + 4 * KL * 1024) <= 160 * 1024, "two workgroups per CU");

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int b, hk, nb, part = 0;
    if (a.work_order && a.cu_seqlens_k) {
        int slot = blockIdx.x / a.nheads_k;
        if constexpr (SPLIT) {
            part = slot % S;
            slot /= S;
        }
        const int it = a.work_order[slot];
        if (it < 0) return;
        b = __builtin_amdgcn_readfirstlane(it / nnb);
        nb = __builtin_amdgcn_readfirstlane(it - b * nnb);
        hk = blockIdx.x % a.nheads_k;
    } else {
        const int bh_count = a.batch * a.nheads_k, bhk = blockIdx.x % bh_count;
        nb = blockIdx.x / bh_count;  // the key blocks that most queries see first
        if constexpr (SPLIT) {
            part = nb % S;
            nb /= S;
        }
        b = bhk / a.nheads_k;
        hk = bhk - b * a.nheads_k;
    }
    const int G = a.nheads / a.nheads_k;
    const bool packed_q = a.cu_seqlens_q != nullptr, packed_k = a.cu_seqlens_k != nullptr;
    const DiffRows rq = diff_rows(a.cu_seqlens_q, b, a.seqlen_q, a.dq_rows), rk = diff_rows(a.cu_seqlens_k, b, a.seqlen_k, a.dkv_rows);
    const int sq = rq.n, sk = rk.n, k0 = nb * BN;
    if (k0 >= sk) return;

    const f16 *kp = (const f16 *)a.k.ptr + base_off(a.k, packed_k, b, rk.start, hk);
    const f16 *vp = (const f16 *)a.v.ptr + base_off(a.v, packed_k, b, rk.start, hk);
    const int causal_off = sk - sq;
    const bool flat = fabsf(a.softmax_scale) < kDiffFlatScale;  // scores of 0: see the dQ kernel
    const float cs = uniform(flat ? 1.f : a.softmax_scale * kLog2e);
    const int64_t qrs = a.q.row_stride, dors = a.dout.row_stride;
    const int kw0 = k0 + wave * 32, key = kw0 + col;
    TileReader<HD> rd;
    rd.init(lane);
    // V rows: row r of each 32-row group at position sigma(r), so that the B
    // operand of key col is the conflict-free A-operand pattern.
    {
        constexpr int KCH = HD / 8;
        char *tile = smem + 2 * STAGE;
#pragma unroll
        for (int i = 0; i < BN * KCH / NT; ++i) {
            const int base = (i * (NT / 64) + wave) * 64;
            const int p = base + lane, pos = p / KCH, c = p % KCH;
            const int64_t r = min(k0 + ((pos & ~31) | sigma(pos & 31)), sk - 1);
            g2l16(vp + r * a.v.row_stride + 8 * (c ^ swz<KCH>(pos)), tile + base * 16);
        }
    }
    f16x8 kreg[KR];
    const int kat = KAT + wave * KL * 1024 + lane * 16;
    {
        const f16 *kr = kp + int64_t(min(key, sk - 1)) * a.k.row_stride + 8 * hh;
        const uint32_t keep = flat ? 0u : ~0u;
#pragma unroll
        for (int g = 0; g < HD / 16; ++g) {
            const f16x8 x = as_h8(ldg16(kr + 16 * g) & keep);
            if (g < KR)
                kreg[g] = x;
            else
                *reinterpret_cast<f16x8 *>(smem + kat + (g - KR) * 1024) = x;
        }
    }
    f32x16 dk[HD / 32], dv[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) dk[i] = dv[i] = zero16();

    const int m_first = CAUSAL ? max(0, k0 - causal_off) / BM : 0;
    const int n_qb = max(0, (sq + BM - 1) / BM - m_first);
    DiffCopier<HD, BM, NT> cp;
    cp.init(wave, lane);
    // Running pointers of the next (head, query block) to copy.
    const f16 *nq = (const f16 *)a.q.ptr + base_off(a.q, packed_q, b, rq.start, hk * G);
    const f16 *ndo = (const f16 *)a.dout.ptr + base_off(a.dout, packed_q, b, rq.start, hk * G);
    const DiffRowOps *ops =
        reinterpret_cast<const DiffRowOps *>(a.dsum + diff_ops_at(a)) + (int64_t(b) * a.nheads + hk * G) * a.lse_seqlen;
    // This workgroup's steps [t0, t1) of the G * n_qb (head slowest).
    int t0 = 0, t1 = G * n_qb;
    if constexpr (SPLIT) {
        t0 = int(int64_t(G * n_qb) * part / S);
        t1 = int(int64_t(G * n_qb) * (part + 1) / S);
    }
    int ni = 0, left = t1 - t0, i0 = 0;  // block of the next copy, steps not yet copied, first block
    if (SPLIT && n_qb > 0) {
        const int h0 = t0 / n_qb;
        ni = i0 = t0 - h0 * n_qb;
        nq += int64_t(h0) * a.q.head_stride;
        ndo += int64_t(h0) * a.dout.head_stride;
        ops += int64_t(h0) * a.lse_seqlen;
    }
    const uint32_t smem_l = lds_addr(smem);
    auto issue_next = [&](int st) FA_INLINE {
        const int q0 = (m_first + ni) * BM;
        const uint32_t tile = smem_l + st * STAGE;
        cp.copy(tile, nq + int64_t(q0) * qrs, qrs, sq - q0);
        cp.copy(tile + QTILE, ndo + int64_t(q0) * dors, dors, sq - q0);
        if (wave == 0)  // 32 rows of 32 bytes, two lanes a row
            g2l16_at(reinterpret_cast<const f16 *>(uniform(ops + q0)), min(lane >> 1, sq - 1 - q0) * 32 + (lane & 1) * 16,
                     __builtin_amdgcn_readfirstlane(tile + 2 * QTILE));
        --left;
        if (++ni == n_qb) {
            ni = 0;
            nq += a.q.head_stride;
            ndo += a.dout.head_stride;
            ops += a.lse_seqlen;
        }
    };
    const int vb0 = rd.a_base + 2 * STAGE + 32 * wave * (HD * 2);
    static_assert(STAGE % 512 == 0 && QTILE % 512 == 0, "tile offsets must be multiples of 512 bytes");

    auto block = [&](int j, int qh0, auto mask_tag) FA_INLINE {
        constexpr bool MASK = decltype(mask_tag)::value;
        const int soff = (j & 1) * STAGE;
        const char *lf = smem + soff + 2 * QTILE;  // 32 rows' DiffRowOps
        int qb = rd.a_base + soff, tb0 = rd.tr_base[0] + soff, tb1 = rd.tr_base[1] + soff, vb = vb0;
        asm volatile("" : "+v"(qb), "+v"(tb0), "+v"(tb1), "+v"(vb));
        constexpr int PIPE = 2, PS = 4, PT = 3, NG = HD / 16;  // operands read ahead: dP, scores, dK and dV
        // The A operands of the products take row sigma(col) of the tile.
        int ro = sigma(col) * 32 + soff + 2 * QTILE;
        asm volatile("" : "+v"(ro));
        f32x16 s[2], dp;
        // Query row c = 16 r8 + u (from qh0 + 8 hh) is live for m_lo <= c < m_hi.
        const int mbase = qh0 + 8 * hh;
        const int m_lo = CAUSAL ? key - causal_off - mbase : -(1 << 30), m_hi = sq - mbase;
        // Rows with a negative lam: bit l for the row of lane l, sigma(l); row 16 r8 + 8 hh + u is lane's
        // 16 r8 + 8 (u / 4) + 4 hh + u % 4.
        const uint64_t neg = __builtin_amdgcn_ballot_w64(*reinterpret_cast<const int16_t *>(smem + 14 + ro) < 0);
        auto exps = [&](int m, int r0, int n) FA_INLINE {
#pragma unroll
            for (int r = r0; r < r0 + n; ++r) {
                s[m][r] = exp2_fast(s[m][r] * cs);
                if constexpr (MASK) {
                    const int c = 16 * (r >> 3) + (r & 7);
                    s[m][r] = c < m_lo || c >= m_hi ? 0.f : s[m][r];
                }
            }
        };
        {
            int h0 = hh;
            asm volatile("" : "+v"(h0));  // formed per block, not held
            const f16x8 w0 = row_weights(0, h0), w1 = row_weights(1, h0);
            const f16x8 lses = lds_ld16(smem, ro);
            // Step u of the scores: map u % 2, K step u / 2 of its channels.
            f16x8 op[PS];
            auto ldq = [&](int u) FA_INLINE { op[u % PS] = rd.a_operand_at(smem, qb, (u & 1) * HG + (u >> 1)); };
#pragma unroll
            for (int u = 0; u < PS - 1; ++u) ldq(u);
            f16x8 kl[KL > 0 ? KL : 1];
#pragma unroll
            for (int i = 0; i < KL; ++i) kl[i] = lds_ld16(smem + i * 1024, kat);
            s[0] = mfma16<true>(lses, w0, zero16());
            s[1] = mfma16<true>(lses, w1, zero16());
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                if (u + PS - 1 < NG) ldq(u + PS - 1);
                const int g = (u & 1) * HG + (u >> 1);
                s[u & 1] = mfma16<BF>(op[u % PS], g < KR ? kreg[g < KR ? g : 0] : kl[g < KR ? 0 : g - KR], s[u & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            // dP, with the exponentials beside its products.
            f16x8 oa[PIPE], va[PIPE];
            auto ldo = [&](int g) FA_INLINE {
                oa[g % PIPE] = rd.a_operand_at(smem + QTILE, qb, g);
                va[g % PIPE] = rd.a_operand_at(smem, vb, g);
            };
#pragma unroll
            for (int g = 0; g < PIPE - 1; ++g) ldo(g);
            asm volatile("" : "+v"(h0));
            dp = mfma16<true>(lds_ld16(smem + 16, ro), row_weights(0, h0), zero16());
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (g + PIPE - 1 < NG) ldo(g + PIPE - 1);
                dp = mfma16<BF>(oa[g % PIPE], va[g % PIPE], dp);
                exps(g * 2 / NG, 32 / NG * (g % (NG / 2)), 32 / NG);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        f16x8 pB[2], d1B[2], d2B[2], tr[PT];
        // Transposed operand u of dV (Q = 0) or dK: channel tile u / 2, query step u % 2.
        auto ldt = [&](int n, int q, int u) FA_INLINE {
            tr[n % PT] = rd.tr_operand_at(smem + (q ? 0 : QTILE) + 16 * (u & 1) * (HD * 2), tb0, tb1, u >> 1);
        };
#pragma unroll
        for (int n = 0; n < PT - 1; ++n) ldt(n, 1, n);
#pragma unroll
        for (int r8 = 0; r8 < 2; ++r8) {
            f32x16 x;
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = s[0][8 * r8 + u] * dp[8 * r8 + u];
            d1B[r8] = pack16<BF>(x, 0);
            asm volatile("" : "+v"(d1B[r8]));
        }
        // dP - D_1 is used up: dP - D_2 takes its place.
        {
            int h0 = hh;
            asm volatile("" : "+v"(h0));
            dp = mfma16<true>(lds_ld16(smem + 16, ro), row_weights(1, h0), dp);
        }
        __builtin_amdgcn_sched_barrier(0);
        // dK of map 1 beside P, dV beside dS_2, dK of map 2.
        constexpr int N1 = 2 * DT, N2 = N1 + 2 * (HD / 32), N3 = N2 + 2 * DT;
        auto ldn = [&](int n) FA_INLINE {
            if (n < N1)
                ldt(n, 1, n);
            else if (n < N2)
                ldt(n, 0, n - N1);
            else
                ldt(n, 1, n - N2 + N1);
        };
        if (neg != 0) {
            const uint32_t m = uint32_t(neg) >> (4 * hh);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[1][r] = __uint_as_float(__float_as_uint(s[1][r]) |
                                          (m << (31 - 16 * (r >> 3) - 8 * (r >> 2 & 1) - (r & 3)) & 0x80000000u));
        }
#pragma unroll
        for (int n = 0; n < N1; ++n) {
            if (n + PT - 1 < N3) ldn(n + PT - 1);
            dk[n >> 1] = mfma16<BF>(tr[n % PT], d1B[n & 1], dk[n >> 1]);
            constexpr int E = 16 / N1;
#pragma unroll
            for (int r = E * n; r < E * n + E; ++r) s[0][r] -= s[1][r];
            if (E * (n + 1) % 8 == 0) pB[E * (n + 1) / 8 - 1] = pack16<BF>(s[0], E * (n + 1) - 8);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = N1; n < N2; ++n) {
            if (n + PT - 1 < N3) ldn(n + PT - 1);
            const int u = n - N1;
            dv[u >> 1] = mfma16<BF>(tr[n % PT], pB[u & 1], dv[u >> 1]);
            constexpr int E = 16 / (N2 - N1);
#pragma unroll
            for (int r = E * u; r < E * u + E; ++r) s[1][r] *= dp[r];
            if (E * (u + 1) % 8 == 0) d2B[E * (u + 1) / 8 - 1] = pack16<BF>(s[1], E * (u + 1) - 8);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = N2; n < N3; ++n) {
            if (n + PT - 1 < N3) ldn(n + PT - 1);
            const int u = n - N2 + N1;
            dk[u >> 1] = mfma16<BF>(tr[n % PT], d2B[u & 1], dk[u >> 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Per head four straight loops: blocks that see none of the wave's keys,
    // diagonal blocks, full blocks, a ragged last block.
    int j = 0;
    auto step = [&](int i, auto mask_tag, bool compute) FA_INLINE {
        wait_vmem();
        __syncthreads();
        if (left > 0) issue_next((j & 1) ^ 1);
        if (compute) block(j, (m_first + i) * BM, mask_tag);
        ++j;
    };
    auto clampi = [](int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); };
    auto first_at = [&](int x) { return ((x + BM - 1) >> 5) - m_first; };
    const int i1 = CAUSAL ? clampi(first_at(kw0 - 31 - causal_off), 0, n_qb) : 0;
    const int i2 = CAUSAL ? clampi(first_at(kw0 + 31 - causal_off), i1, n_qb) : 0;
    const int i3 = clampi(first_at(sq - 31), i2, n_qb);
    if (t1 > t0)
        issue_next(0);
    else
        wait_vmem();
    for (int t = t0, i = i0; t < t1; i = 0) {
        const int end = min(n_qb, i + t1 - t);
        t += end - i;
        for (const int e = min(i1, end); i < e; ++i) step(i, std::true_type{}, false);
        for (const int e = min(i2, end); i < e; ++i) step(i, std::true_type{}, true);
        for (const int e = min(i3, end); i < e; ++i) step(i, std::false_type{}, true);
        for (; i < end; ++i) step(i, std::true_type{}, true);
    }
    if constexpr (SPLIT)
        if (!diff_dkdv_sum<HD>(a, (b * nnb + nb) * a.nheads_k + hk, part, S, &ticket, dk, dv)) return;

    if (key >= sk) return;
    f16 *dkrow = (f16 *)a.dk.ptr + base_off(a.dk, packed_k, b, rk.start, hk) + int64_t(key) * a.dk.row_stride;
    f16 *dvrow = (f16 *)a.dv.ptr + base_off(a.dv, packed_k, b, rk.start, hk) + int64_t(key) * a.dv.row_stride;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) {
        const float f = dt < DT ? a.softmax_scale : -a.softmax_scale;
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4) {
            const int c = 4 * a4;
            *reinterpret_cast<f16x4 *>(dkrow + dt * 32 + 8 * a4 + 4 * hh) =
                pack4<BF>(dk[dt][c] * f, dk[dt][c + 1] * f, dk[dt][c + 2] * f, dk[dt][c + 3] * f);
            *reinterpret_cast<f16x4 *>(dvrow + dt * 32 + 8 * a4 + 4 * hh) =
                pack4<BF>(dv[dt][c], dv[dt][c + 1], dv[dt][c + 2], dv[dt][c + 3]);
        }
    }
}

// ---------------------------------------------------------------------------
// dlam from the rows' -D_2 (the start of the workspace, written by the dQ kernel).
// A lam for each row: one value each, transposed.  One that rows share: one
// workgroup per head sums its rows in fp64 in a fixed order, and for a lam of
// all heads the second launch sums the heads.  It takes a batch's sequences one
// after the other: 10 us for 16 of them, but 1.8 ms for 4096 of 8 tokens (16 heads)
// beside 1.0 ms for the rest of the step.
__global__ __launch_bounds__(1024) void diff_dlam_rows_kernel(const fa_diff_bwd_args a) {
    for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
        const DiffRows rq = diff_rows(a.cu_seqlens_q, b, a.seqlen_q, a.dq_rows);
        const int64_t start = rq.start, n = int64_t(rq.n) * a.nheads;
        for (int64_t i = int64_t(blockIdx.x) * 1024 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 1024) {
            const int64_t row = i / a.nheads;
            const int h = int(i - row * a.nheads);
            a.dlam.ptr[b * a.dlam.batch_stride + (start + row) * a.dlam.row_stride + h * a.dlam.head_stride] =
                a.dsum[(int64_t(b) * a.nheads + h) * a.lse_seqlen + row];
        }
    }
}

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[16];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0;
    for (int i = 0; i < int(blockDim.x >> 6); ++i) s += part[i];
    return s;
}

// Head blockIdx.x; the sum goes to dlam (a lam for each head) or, for a lam of
// all heads, to sums.
__global__ __launch_bounds__(1024) void diff_dlam_head_kernel(const fa_diff_bwd_args a, double *const sums) {
    const int h = blockIdx.x;
    const float *nd2 = a.dsum;
    double x = 0;
    for (int b = 0; b < a.batch; ++b) {
        const int sq = diff_rows(a.cu_seqlens_q, b, a.seqlen_q, a.dq_rows).n;
        const float *row = nd2 + (int64_t(b) * a.nheads + h) * a.lse_seqlen;
        for (int i = threadIdx.x; i < sq; i += 1024) x += row[i];
    }
    x = block_sum(x);
    if (threadIdx.x == 0) {
        if (sums)
            sums[h] = x;
        else
            a.dlam.ptr[h * a.dlam.head_stride] = float(x);
    }
}

__global__ __launch_bounds__(64) void diff_dlam_all_kernel(const fa_diff_bwd_args a, const double *const sums) {
    double x = 0;
    for (int h = threadIdx.x; h < a.nheads; h += 64) x += sums[h];
    x = block_sum(x);
    if (threadIdx.x == 0) a.dlam.ptr[0] = float(x);
}

// Packed batches: work orders (workgroup 0 for dK/dV, 1 for dQ) and zeros in the
// gradients of rows of no sequence.
__global__ __launch_bounds__(kOrderThreads) void diff_bwd_order_kernel(const fa_diff_bwd_args a, const int nnb,
                                                                       const int nmb, const int P, const int order_wgs) {
    if (int(blockIdx.x) >= order_wgs) {
        const int i = blockIdx.x - order_wgs, n = gridDim.x - order_wgs;
        if (a.dq_rows > 0)
            zero_gaps(a.dq, a.cu_seqlens_q, a.batch, a.lse_seqlen, a.dq_rows, a.nheads, a.head_dim, i, n);
        if (a.dkv_rows > 0)
            for (const fa_tensor *t : {&a.dk, &a.dv})
                zero_gaps(*t, a.cu_seqlens_k, a.batch, a.seqlen_k, a.dkv_rows, a.nheads_k, a.head_dim, i, n);
        return;
    }
    const bool dq = blockIdx.x == 1;
    const int per = dq ? nmb : nnb;
    order_items(a.batch * per, [&](int it) {
        const int b = it / per, blk = it - b * per;
        const int sq = diff_rows(a.cu_seqlens_q, b, a.seqlen_q, a.dq_rows).n;
        const int sk = diff_rows(a.cu_seqlens_k, b, a.seqlen_k, a.dkv_rows).n;
        const int at = blk * (dq ? P : 128);
        if (at >= (dq ? sq : sk)) return -1;
        int n;  // keys of a dQ item, queries of a dK/dV item
        if (dq)
            n = a.causal ? min(sk, at + P + sk - sq) : sk;
        else
            n = a.causal ? min(sq, sk - at) : sq;
        return min(max(0, n) >> 6, kOrderBuckets - 1);
    }, a.work_order + (dq ? int64_t(a.batch) * nnb : 0), false);
}

static int check_diff_bwd(const fa_diff_bwd_args *p) {
    if (!p) return FA_ERR_INVALID_ARG;
    const fa_diff_bwd_args &a = *p;
    if (a.head_dim != 64 && a.head_dim != 128) return FA_ERR_UNSUPPORTED;
    if (a.dtype != FA_FP16 && a.dtype != FA_BF16) return FA_ERR_UNSUPPORTED;
    if (a.batch < 0 || a.seqlen_q < 0 || a.seqlen_k < 0 || a.nheads <= 0 || a.nheads_k <= 0 ||
        a.nheads % a.nheads_k != 0 || a.lse_seqlen < a.seqlen_q || (!a.cu_seqlens_q) != (!a.cu_seqlens_k))
        return FA_ERR_INVALID_ARG;
    if (!a.lse || !a.lam.ptr) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.q, &a.k, &a.v, &a.o, &a.o2, &a.dout, &a.dq, &a.dk, &a.dv})
        if (check_tensor(*t, true)) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.q, &a.k, &a.v, &a.dout})
        if (t->row_stride < 0 || t->row_stride > kDiffMaxRowStride) return FA_ERR_INVALID_ARG;
    if (!split_ws_aligned(a.split_ws)) return FA_ERR_INVALID_ARG;
    if (!a.dsum || (reinterpret_cast<uintptr_t>(a.dsum) & 31u) || a.dsum_bytes < int64_t(fa_diff_bwd_ws_bytes(&a)))
        return FA_ERR_WORKSPACE;
    return FA_OK;
}

// Workgroups that share each (batch, key block, KV head) item of dK/dV.  One
// where the grid fills the chip; with few items, or causal ones of very different
// lengths, the longest item decides the kernel's time.  The estimate, in steps of
// 32 queries (about 1.1 us at head_dim 128, two workgroups on a CU): the busiest
// CU's steps (equal items in whole rounds; causal ones, longest first, leave about
// half an item of imbalance), and the partials' traffic.  Packed batches are
// taken as sequences of the mean length, which the packed tensors' rows tell, with
// the longest one's longest item.
static int diff_dkdv_splits(const fa_diff_bwd_args &a) {
    constexpr int kMaxSplits = 16;
    constexpr int64_t kMaxBytes = int64_t(256) << 20;  // of partials
    const int64_t slots = diff_dkdv_items(a), cus = device_cus();
    const int64_t cap = std::min<int64_t>(kMaxSplits, kMaxBytes / std::max<int64_t>(1, slots * 1024 * a.head_dim));
    if (cap < 2 || a.seqlen_q <= 0) return 1;
    const int G = a.nheads / a.nheads_k;
    auto steps_of = [&](int64_t sq, int64_t sk, int64_t &items) {
        const int64_t nnb = (sk + 127) / 128, n_qb = (sq + 31) / 32;
        items += nnb;
        if (!a.causal) return double(G) * n_qb * nnb;
        double t = 0;
        for (int64_t nb = 0; nb < nnb; ++nb) t += double(G) * std::max<int64_t>(0, n_qb - std::max<int64_t>(0, nb * 128 - (sk - sq)) / 32);
        return t;
    };
    const double longest = double(G) * ((a.seqlen_q + 31) / 32);
    int64_t items = 0;
    const bool mean = a.cu_seqlens_q && a.dq_rows > 0 && a.dkv_rows > 0;
    double total = steps_of(mean ? (a.dq_rows + a.batch - 1) / a.batch : a.seqlen_q,
                            mean ? (a.dkv_rows + a.batch - 1) / a.batch : a.seqlen_k, items);
    total *= double(a.batch) * a.nheads_k / cus;
    items *= int64_t(a.batch) * a.nheads_k;
    const bool uneven = a.causal || mean;
    int best = 1;
    double best_t = 0;
    for (int S = 1; S <= cap; ++S) {
        const int64_t wgs = items * S;
        double t = uneven ? std::max(longest / S, total * (1 + 0.5 * cus / wgs))
                          : double((wgs + cus - 1) / cus) * longest / S;
        if (wgs <= cus) t *= 1.1;
        if (S > 1) t += (2 * wgs <= cus ? 2 : 0) + (S - 1) * (0.025 * items + 3);
        if (S == 1 || t < best_t) {
            best = S;
            best_t = t;
        }
    }
    return best;
}

// Bytes of the rows' parts; the heads' fp64 sums follow.
static int64_t plane_bytes(const fa_diff_bwd_args &a) {
    return diff_ops_at(a) * 4 + diff_plane(a) * int64_t(sizeof(DiffRowOps));
}

template <int HD, bool BF>
static int launch_diff_bwd(fa_diff_bwd_args a, hipStream_t s) {
    if (!a.split_ws || a.split_ws_bytes < int64_t(fa_diff_bwd_split_bytes(&a))) a.split_ws = nullptr;
    const int S = a.split_ws ? diff_dkdv_splits(a) : 1;
    if (S == 1) a.split_ws = nullptr;
    const int group = a.nheads / a.nheads_k;
    int lg = 0;  // heads of a GQA group in a dQ workgroup
    while (lg < 2 && group % (2 << lg) == 0) ++lg;
    const int P = 128 >> lg, nmb = (a.lse_seqlen + P - 1) / P, nnb = (a.seqlen_k + 127) / 128;
    const int64_t q_grid = int64_t(nmb) * a.batch * (a.nheads >> lg), k_grid = int64_t(nnb) * a.batch * a.nheads_k * S;
    if (q_grid > 0x7fffffff || k_grid > 0x7fffffff) return FA_ERR_INVALID_ARG;
    int rc;
    if (a.cu_seqlens_q && (a.work_order || a.dq_rows > 0 || a.dkv_rows > 0)) {
        const int order_wgs = a.work_order ? 2 : 0, zero_wgs = a.dq_rows > 0 || a.dkv_rows > 0 ? kZeroBlocks : 0;
        hipLaunchKernelGGL(diff_bwd_order_kernel, dim3(order_wgs + zero_wgs), dim3(kOrderThreads), 0, s, a, nnb, nmb, P,
                           order_wgs);
        if ((rc = int(hipGetLastError()))) return rc;
    }
    if (q_grid > 0) {
        if (a.causal)
            hipLaunchKernelGGL((diff_dq_kernel<HD, BF, true>), dim3(unsigned(q_grid)), dim3(kDbThreads), 0, s, a, nmb, lg);
        else
            hipLaunchKernelGGL((diff_dq_kernel<HD, BF, false>), dim3(unsigned(q_grid)), dim3(kDbThreads), 0, s, a, nmb, lg);
        if ((rc = int(hipGetLastError()))) return rc;
    }
    if (k_grid > 0) {
        auto launch = [&](auto causal, auto split) {
            hipLaunchKernelGGL((diff_dkdv_kernel<HD, BF, decltype(causal)::value, decltype(split)::value>),
                               dim3(unsigned(k_grid)), dim3(kDbThreads), 0, s, a, nnb, S);
        };
        using T = std::true_type;
        using F = std::false_type;
        if (a.causal)
            S > 1 ? launch(T{}, T{}) : launch(T{}, F{});
        else
            S > 1 ? launch(F{}, T{}) : launch(F{}, F{});
        if ((rc = int(hipGetLastError()))) return rc;
    }
    if (!a.dlam.ptr) return FA_OK;
    if (a.dlam.row_stride != 0) {
        if (a.batch == 0 || a.lse_seqlen == 0) return FA_OK;
        const int64_t n = int64_t(a.lse_seqlen) * a.nheads;
        hipLaunchKernelGGL(diff_dlam_rows_kernel, dim3(unsigned(std::min<int64_t>((n + 1023) / 1024, 1024)), std::min(a.batch, 65535)),
                           dim3(1024), 0, s, a);
        return int(hipGetLastError());
    }
    double *sums = a.dlam.head_stride != 0
                       ? nullptr
                       : reinterpret_cast<double *>(reinterpret_cast<char *>(a.dsum) + plane_bytes(a));
    hipLaunchKernelGGL(diff_dlam_head_kernel, dim3(a.nheads), dim3(1024), 0, s, a, sums);
    if ((rc = int(hipGetLastError())) || !sums) return rc;
    hipLaunchKernelGGL(diff_dlam_all_kernel, dim3(1), dim3(64), 0, s, a, sums);
    return int(hipGetLastError());
}

}  // namespace fa

extern "C" size_t fa_diff_bwd_ws_bytes(const fa_diff_bwd_args *a) {
    if (!a || a->batch < 0 || a->nheads <= 0 || a->lse_seqlen < 0) return 0;
    return size_t(fa::plane_bytes(*a) + 8 * int64_t(a->nheads));
}

extern "C" size_t fa_diff_bwd_split_bytes(const fa_diff_bwd_args *p) {
    if (!p || p->batch <= 0 || p->seqlen_q <= 0 || p->seqlen_k <= 0 || p->nheads <= 0 || p->nheads_k <= 0 ||
        (p->head_dim != 64 && p->head_dim != 128))
        return 0;
    const int S = fa::diff_dkdv_splits(*p);
    const int64_t items = fa::diff_dkdv_items(*p);
    return S > 1 ? size_t(fa::diff_dkdv_count_bytes(items) + items * S * 2 * 128 * p->head_dim * 4) : 0;
}

extern "C" size_t fa_diff_bwd_order_len(const fa_diff_bwd_args *a) {
    if (!a || a->batch <= 0) return 0;
    return size_t(a->batch) *
           (size_t((std::max(a->seqlen_k, 0) + 127) / 128) + size_t((std::max(a->lse_seqlen, 0) + 31) / 32));
}

extern "C" int fa_diff_bwd(const fa_diff_bwd_args *args, void *stream) {
    const int rc = fa::check_diff_bwd(args);
    if (rc) return rc;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const fa_diff_bwd_args &a = *args;
    if (a.dtype == FA_BF16)
        return a.head_dim == 128 ? fa::launch_diff_bwd<128, true>(a, s) : fa::launch_diff_bwd<64, true>(a, s);
    return a.head_dim == 128 ? fa::launch_diff_bwd<128, false>(a, s) : fa::launch_diff_bwd<64, false>(a, s);
}
