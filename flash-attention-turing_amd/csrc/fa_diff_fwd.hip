// Differential attention, forward: dense and packed batches, and rows of many
// queries over a key-value cache.
//
//   S_m = scale q_m k_m^T,  P_m = softmax(S_m) over the visible keys  (m = 1, 2)
//   o = (P_1 - lam P_2) v
//
// Each wave owns 32 queries of one head and walks 64-key blocks, keeping for
// both maps a running maximum, a sum and an fp32 O_m of its own (the sums that
// would join them are known at the end only).  S_m^T = K_m Q_m^T puts keys on
// the MFMA M dimension, so a lane owns one query column, and P_m^T feeds
// O_m^T += V^T P_m^T from the accumulators.  One transposed read of V serves
// the products of both maps, which two calls of ordinary attention would read
// twice.  Per 32 queries x 64 keys at head_dim 128: 16 MFMAs for the scores and
// 32 for O, 48 against 40 of ordinary attention's 32, with 32 LDS operand reads.
#include <algorithm>
#include <type_traits>

#include "fa_diff_common.h"

namespace fa {

constexpr int kDiffBN = 64;       // keys per block
constexpr int kDiffThreads = 256;  // 4 waves of 32 queries

// A call as the kernel takes it: the tensors, and the cache that k and v are
// (cache_seqlens set).
struct DiffFwd {
    fa_diff_fwd_args a;
    const int32_t *cache_seqlens, *cache_batch_idx, *block_table;
    int64_t block_table_stride;
    int32_t seqlen_new, page, num_pages, capacity, cache_batch;
    int32_t *status;
};

// One map's 64-key block of S^T -> P^T operands: mask (keys past lim, relative
// to the block), running maximum, rescale of O, exponentials, row sum.  P is
// rounded to 16 bits for the product with V, as in ordinary attention; O and
// the LSE are normalised by the fp32 sum of the unrounded P.
template <int HD, bool BF, bool MASK>
__device__ __forceinline__ void diff_softmax(f32x16 (&s)[2], f16x8 (&pB)[4], f32x16 (&o)[HD / 32], float &m, float &l,
                                             float cscale, int lim, int hh) {
    if constexpr (MASK) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (kt * 32 + acc_lrow(e, hh) > lim) s[kt][e] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kt][e]);
    mx = max_xor32(mx);
    const float mx_t = MASK && mx == -INFINITY ? -INFINITY : mx * cscale;
    if (__builtin_amdgcn_ballot_w64(mx_t > m) != 0) {
        const float m_new = fmaxf(m, mx_t);
        const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m - m_new);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        m = m_new;
    }
    const float m_use = m == -INFINITY ? 0.f : m;
    float rs = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float x = s[kt][e];
            float p = exp2_fast(fmaf(x, cscale, -m_use));
            if constexpr (MASK) p = x == -INFINITY ? 0.f : p;
            s[kt][e] = p;
            rs += p;
        }
    l += rs;
#pragma unroll
    for (int gg = 0; gg < 4; ++gg) pB[gg] = pack16<BF>(s[gg >> 1], 8 * (gg & 1));
}

template <int HD, bool BF, bool CAUSAL, bool CACHE>
__global__ __launch_bounds__(kDiffThreads, 2) void diff_fwd_kernel(const DiffFwd p, const int num_m_blocks,
                                                                   const int lg) {
    constexpr int NT = kDiffThreads, BM = 128, BN = kDiffBN;
    constexpr int TILE = BN * HD * 2, STAGE = 2 * TILE;
    constexpr int HG = HD / 32;  // MFMA K steps of one map's channels
    const fa_diff_fwd_args &a = p.a;
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];

    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The workgroup's rows: gp = 2^lg heads of one GQA group at P = 128 / gp
    // positions from m0, which share the K / V tiles.
    const int gp = 1 << lg, packs = a.nheads >> lg, P = BM >> lg;
    int b, h, mb;
    if (a.work_order && a.cu_seqlens_q) {
        const int it = a.work_order[blockIdx.x / packs];
        b = __builtin_amdgcn_readfirstlane(it / num_m_blocks);
        mb = __builtin_amdgcn_readfirstlane(it - b * num_m_blocks);
        h = (blockIdx.x % packs) * gp;
    } else {
        const int bp_count = a.batch * packs, bp = blockIdx.x % bp_count;
        mb = blockIdx.x / bp_count;
        if (CAUSAL) mb = num_m_blocks - 1 - mb;  // heaviest first
        b = bp / packs;
        h = (bp - b * packs) * gp;
    }
    const int hk = h / (a.nheads / a.nheads_k);
    const bool packed_q = a.cu_seqlens_q != nullptr, packed_k = a.cu_seqlens_k != nullptr;
    SeqInfo si = seq_info(b, a.seqlen_q, a.seqlen_k, a.cu_seqlens_q, a.cu_seqlens_k, nullptr, 0);
    int kb = b;
    if constexpr (CACHE) {
        // A length or a cache row outside the cache leaves the sequence with no
        // keys, and the status word says so: no access leaves the cache.
        const int used = p.cache_seqlens[b];
        if (p.cache_batch_idx) kb = p.cache_batch_idx[b];
        const int err = (used < 0 || int64_t(used) + p.seqlen_new > p.capacity ? 1 : 0) |
                        (p.cache_batch_idx && (kb < 0 || kb >= p.cache_batch) ? 2 : 0);
        si.sk = err ? 0 : used + p.seqlen_new;
        if (err) {
            kb = 0;
            if (p.status && tid == 0) atomicOr(p.status, err);
        }
    }
    const int sq = si.sq, sk = si.sk, m0 = mb * P;
    const int64_t plane = int64_t(a.batch) * a.nheads * a.lse_seqlen;
    float *lse_row = a.lse + (int64_t(b) * a.nheads + h) * a.lse_seqlen;
    if (m0 >= sq) {  // past this sequence: LSE padding is 0
        for (int i = tid; i < gp * P; i += NT) {
            const int row = m0 + i % P;
            if (row < a.lse_seqlen) {
                lse_row[int64_t(i / P) * a.lse_seqlen + row] = 0.f;
                lse_row[plane + int64_t(i / P) * a.lse_seqlen + row] = 0.f;
            }
        }
        return;
    }
    const int causal_off = sk - sq;  // key j is visible to query i iff j <= i + causal_off
    int n_end = sk;
    if (CAUSAL) n_end = max(0, min(sk, m0 + P + causal_off));
    const int n_blocks = (n_end + BN - 1) / BN;
    const float cscale = fabsf(a.softmax_scale) * kLog2e;

    const f16 *kp = (const f16 *)a.k.ptr + base_off(a.k, packed_k, CACHE && p.block_table ? 0 : kb, si.k_start, hk);
    const f16 *vp = (const f16 *)a.v.ptr + base_off(a.v, packed_k, CACHE && p.block_table ? 0 : kb, si.k_start, hk);
    const int64_t krs = a.k.row_stride, vrs = a.v.row_stride;
    TileCopier<HD, BN, NT> kcp, vcp;
    kcp.init(krs, wave, lane);
    vcp.init(vrs, wave, lane);
    // Copies of key block nb into stage st; a block past the sequence's end
    // re-reads its last key (masked).  A page is a multiple of 64 tokens, so a
    // block lies in one.
    auto issue = [&](int nb, int st) FA_INLINE {
        const int n0 = nb * BN;
        int64_t koff = int64_t(n0) * krs, voff = int64_t(n0) * vrs;
        if constexpr (CACHE) {
            if (p.block_table) {
                const int pg = n0 / p.page, in_page = n0 - pg * p.page;
                const int blk = checked_page(p.block_table, p.block_table_stride, b, pg, p.num_pages, p.status);
                koff = int64_t(blk) * a.k.batch_stride + int64_t(in_page) * krs;
                voff = int64_t(blk) * a.v.batch_stride + int64_t(in_page) * vrs;
            }
        }
        if (n0 + BN <= sk) {
            kcp.copy_to(lds_addr(smem) + st * STAGE, kp + koff, krs);
            vcp.copy_to(lds_addr(smem) + st * STAGE + TILE, vp + voff, vrs);
        } else {
            dma_tile<HD, BN, NT>(smem + st * STAGE, kp + koff, krs, 0, sk - 1 - n0, wave, lane);
            dma_tile<HD, BN, NT>(smem + st * STAGE + TILE, vp + voff, vrs, 0, sk - 1 - n0, wave, lane);
        }
    };

    // The wave's 32 rows: head h + wave / (P / 32), positions from q_lo.
    h += wave >> (2 - lg);
    const int q_lo = m0 + 32 * (wave & ((P >> 5) - 1));
    const int qi = q_lo + (lane & 31);
    f16x8 qB[HD / 16];  // B operands: lane (query, hh), K step g covers channels 16g + 8hh + 0..7
    {
        const f16 *qp = (const f16 *)a.q.ptr + base_off(a.q, packed_q, b, si.q_start, h) +
                        int64_t(qi < sq ? qi : 0) * a.q.row_stride + 8 * hh;
#pragma unroll
        for (int g = 0; g < HD / 16; ++g) {
            u32x4 v = qi < sq ? ldg16(qp + 16 * g) : zero_u4();
            if (a.softmax_scale < 0.f) v = neg_h8(v);
            qB[g] = as_h8(v);
        }
    }
    wait_vmem();  // only the tile copies are in flight inside the loop

    f32x16 o[2][HD / 32];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) o[m][i] = zero16();
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    TileReader<HD> rd;
    rd.init(lane);

    auto block = [&](int nb, auto mask_tag) FA_INLINE {
        constexpr bool MASK = decltype(mask_tag)::value;
        const int buf = nb & 1, n0 = nb * BN;
        wait_vmem();
        __syncthreads();  // block nb is in LDS; every wave is done with stage buf ^ 1
        if (nb + 1 < n_blocks) issue(nb + 1, buf ^ 1);
        if (CAUSAL && MASK && n0 > q_lo + 31 + causal_off) return;  // no visible key for this wave
        if (q_lo >= sq) return;
        // Operand reads run PIPE - 1 steps ahead behind scheduling fences, from
        // the lane's bases with the stage added once per block (opaque, so that
        // no read address is held in registers through the loop).
        constexpr int PIPE = 3, NPV = 4 * (HD / 32);
        const int soff = buf * STAGE;
        static_assert(STAGE % 512 == 0, "stage offsets must be multiples of 512 bytes");
        int ab = rd.a_base + soff, tb0 = rd.tr_base[0] + soff, tb1 = rd.tr_base[1] + soff;
        asm volatile("" : "+v"(ab), "+v"(tb0), "+v"(tb1));
        f16x8 op[PIPE];
        f16x8 pB[2][4];
        const int lim = (CAUSAL ? min(sk - 1, qi + causal_off) : sk - 1) - n0;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            // Step u: key tile u % 2 (two independent chains), K step u / 2 of the map.
            f32x16 s[2];
            auto rd_k = [&](int u) FA_INLINE {
                op[u % PIPE] = rd.a_operand_at(smem + 32 * (u & 1) * (HD * 2), ab, m * HG + (u >> 1));
            };
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < PIPE - 1; ++u) rd_k(u);
#pragma unroll
            for (int u = 0; u < 2 * HG; ++u) {
                if (u + PIPE - 1 < 2 * HG) rd_k(u + PIPE - 1);
                s[u & 1] = mfma16<BF>(op[u % PIPE], qB[m * HG + (u >> 1)], u < 2 ? zero16() : s[u & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            diff_softmax<HD, BF, MASK>(s, pB[m], o[m], mx[m], sum[m], cscale, lim, hh);
        }
        auto rd_v = [&](int u) FA_INLINE {
            op[u % PIPE] = rd.tr_operand_at(smem + TILE + 16 * (u & 3) * (HD * 2), tb0, tb1, u >> 2);
        };
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < PIPE - 1; ++u) rd_v(u);
#pragma unroll
        for (int u = 0; u < NPV; ++u) {
            if (u + PIPE - 1 < NPV) rd_v(u + PIPE - 1);
#pragma unroll
            for (int m = 0; m < 2; ++m) o[m][u >> 2] = mfma16<BF>(op[u % PIPE], pB[m][u & 3], o[m][u >> 2]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Blocks [0, n_full) need no mask for any wave of the workgroup.
    int n_full = min(n_blocks, sk / BN);
    if (CAUSAL) n_full = min(n_full, max(0, (m0 + causal_off + 1) / BN));
    if (n_blocks > 0) issue(0, 0);
    for (int nb = 0; nb < n_full; ++nb) block(nb, std::false_type{});
    for (int nb = n_full; nb < n_blocks; ++nb) block(nb, std::true_type{});

    lse_row = a.lse + (int64_t(b) * a.nheads + h) * a.lse_seqlen;
    if (qi >= sq) {
        if (hh == 0 && qi < a.lse_seqlen) lse_row[qi] = lse_row[plane + qi] = 0.f;
        return;
    }
    const float l0 = sum_xor32(sum[0]), l1 = sum_xor32(sum[1]);
    const float lam = diff_lam(a.lam, b, si.q_start + qi, h);
    const float i0 = l0 > 0.f ? 1.f / l0 : 0.f, i1 = l1 > 0.f ? 1.f / l1 : 0.f;
    f16 *orow = (f16 *)a.o.ptr + base_off(a.o, packed_q, b, si.q_start, h) + int64_t(qi) * a.o.row_stride;
    f16 *o2row = a.o2.ptr ? (f16 *)a.o2.ptr + base_off(a.o2, packed_q, b, si.q_start, h) + int64_t(qi) * a.o2.row_stride
                          : nullptr;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4) {
            float x[4], y[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                y[t] = o[1][dt][4 * a4 + t] * i1;
                x[t] = l0 > 0.f ? fmaf(o[0][dt][4 * a4 + t], i0, -lam * y[t]) : 0.f;
            }
            *reinterpret_cast<f16x4 *>(orow + dt * 32 + 8 * a4 + 4 * hh) = pack4<BF>(x[0], x[1], x[2], x[3]);
            if (o2row) *reinterpret_cast<f16x4 *>(o2row + dt * 32 + 8 * a4 + 4 * hh) = pack4<BF>(y[0], y[1], y[2], y[3]);
        }
    if (hh == 0) {
        lse_row[qi] = l0 > 0.f ? (mx[0] + log2_fast(l0)) * kLn2 : 0.f;
        lse_row[plane + qi] = l1 > 0.f ? (mx[1] + log2_fast(l1)) * kLn2 : 0.f;
    }
}

// Packed batches: the (sequence, query block) items, most work first, and zeros
// in the rows of no sequence.
__global__ __launch_bounds__(kOrderThreads) void diff_fwd_order_kernel(const fa_diff_fwd_args a, const int nmb,
                                                                       const int P, const int order_wgs) {
    if (int(blockIdx.x) >= order_wgs) {
        for (const fa_tensor *t : {&a.o, &a.o2})
            if (t->ptr)
                zero_gaps(*t, a.cu_seqlens_q, a.batch, a.lse_seqlen, a.o_rows, a.nheads, a.head_dim,
                          blockIdx.x - order_wgs, gridDim.x - order_wgs);
        return;
    }
    order_items(a.batch * nmb, [&](int it) {
        const int b = it / nmb, mb = it - b * nmb;
        const int sq = a.cu_seqlens_q[b + 1] - a.cu_seqlens_q[b];
        const int sk = a.cu_seqlens_k[b + 1] - a.cu_seqlens_k[b];
        const int m0 = mb * P;
        if (m0 >= sq) return -1;
        const int64_t rows = min(P, sq - m0);
        const int64_t keys = a.causal ? max(0, min(sk, m0 + P + sk - sq)) : max(sk, 0);
        return int(min<int64_t>(rows * keys / (int64_t(P) * 64), kOrderBuckets - 1));
    }, a.work_order, true);
}

// log2 of the heads of a GQA group that a workgroup's rows hold: the largest
// power of two that divides the group and leaves whole 32-row tiles per head.
static int diff_pack_log2(int group) {
    int lg = 0;
    while (lg < 2 && group % (2 << lg) == 0) ++lg;
    return lg;
}

int check_diff_fwd(const fa_diff_fwd_args *p) {
    if (!p) return FA_ERR_INVALID_ARG;
    const fa_diff_fwd_args &a = *p;
    if (a.head_dim != 64 && a.head_dim != 128) return FA_ERR_UNSUPPORTED;
    if (a.dtype != FA_FP16 && a.dtype != FA_BF16) return FA_ERR_UNSUPPORTED;
    if (a.batch < 0 || a.seqlen_q < 0 || a.seqlen_k < 0 || a.nheads <= 0 || a.nheads_k <= 0 ||
        a.nheads % a.nheads_k != 0 || a.lse_seqlen < a.seqlen_q || (!a.cu_seqlens_q) != (!a.cu_seqlens_k))
        return FA_ERR_INVALID_ARG;
    if (!a.lse || !a.lam.ptr) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.q, &a.k, &a.v, &a.o})
        if (check_tensor(*t, true)) return FA_ERR_INVALID_ARG;
    return check_tensor(a.o2, false);
}

template <int HD, bool BF, bool CACHE>
static int launch_diff_fwd(const DiffFwd &p, hipStream_t s) {
    const fa_diff_fwd_args &a = p.a;
    const int lg = diff_pack_log2(a.nheads / a.nheads_k), P = 128 >> lg;
    const int nmb = (a.lse_seqlen + P - 1) / P;
    const int64_t grid = int64_t(nmb) * a.batch * (a.nheads >> lg);
    if (grid > 0x7fffffff) return FA_ERR_INVALID_ARG;
    if (a.cu_seqlens_q && (a.work_order || a.o_rows > 0)) {
        const int order_wgs = a.work_order ? 1 : 0;
        hipLaunchKernelGGL(diff_fwd_order_kernel, dim3(order_wgs + (a.o_rows > 0 ? kZeroBlocks : 0)),
                           dim3(kOrderThreads), 0, s, a, nmb, P, order_wgs);
        const int rc = int(hipGetLastError());
        if (rc) return rc;
    }
    if (grid == 0) return FA_OK;
    if (a.causal)
        hipLaunchKernelGGL((diff_fwd_kernel<HD, BF, true, CACHE>), dim3(unsigned(grid)), dim3(kDiffThreads), 0, s, p,
                           nmb, lg);
    else
        hipLaunchKernelGGL((diff_fwd_kernel<HD, BF, false, CACHE>), dim3(unsigned(grid)), dim3(kDiffThreads), 0, s, p,
                           nmb, lg);
    return int(hipGetLastError());
}

template <bool CACHE>
static int dispatch_diff_fwd(const DiffFwd &p, hipStream_t s) {
    if (p.a.dtype == FA_BF16)
        return p.a.head_dim == 128 ? launch_diff_fwd<128, true, CACHE>(p, s) : launch_diff_fwd<64, true, CACHE>(p, s);
    return p.a.head_dim == 128 ? launch_diff_fwd<128, false, CACHE>(p, s) : launch_diff_fwd<64, false, CACHE>(p, s);
}

// A cache call of many query rows (its append is on the stream before).
int diff_fwd_cache(const fa_diff_kvcache_args &c, hipStream_t s) {
    DiffFwd p{};
    fa_diff_fwd_args &a = p.a;
    a.q = c.q;
    a.k = c.k_cache;
    a.v = c.v_cache;
    a.o = c.o;
    a.lam = c.lam;
    a.lse = c.lse;
    a.batch = c.batch;
    a.seqlen_q = a.lse_seqlen = c.seqlen_q;
    a.seqlen_k = c.cache_capacity;
    a.nheads = c.nheads;
    a.nheads_k = c.nheads_k;
    a.head_dim = c.head_dim;
    a.softmax_scale = c.softmax_scale;
    a.causal = c.causal;
    a.dtype = c.dtype;
    p.cache_seqlens = c.cache_seqlens;
    p.cache_batch_idx = c.cache_batch_idx;
    p.block_table = c.block_table;
    p.block_table_stride = c.block_table_stride;
    p.seqlen_new = c.seqlen_new;
    p.page = c.page_block_size;
    p.num_pages = c.num_pages;
    p.capacity = c.cache_capacity;
    p.cache_batch = c.cache_batch;
    p.status = c.status;
    return dispatch_diff_fwd<true>(p, s);
}

}  // namespace fa

extern "C" size_t fa_diff_fwd_order_len(const fa_diff_fwd_args *a) {
    if (!a || a->batch <= 0 || a->lse_seqlen <= 0) return 0;
    return size_t(a->batch) * size_t((a->lse_seqlen + 31) / 32);  // blocks of 32 positions at the least
}

extern "C" int fa_diff_fwd(const fa_diff_fwd_args *args, void *stream) {
    const int rc = fa::check_diff_fwd(args);
    if (rc) return rc;
    fa::DiffFwd p{};
    p.a = *args;
    return fa::dispatch_diff_fwd<false>(p, reinterpret_cast<hipStream_t>(stream));
}
