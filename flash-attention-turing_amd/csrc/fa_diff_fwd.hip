// Differential attention, forward: dense and packed batches, and rows of many
// queries over a key-value cache.
//
//   S_m = scale q_m k_m^T,  P_m = softmax(S_m) over the visible keys  (m = 1, 2)
//   o = (P_1 - lam P_2) v
//
// Each wave owns 32 queries of one head and walks 64-key blocks, keeping for
// both maps a sum and an fp32 O_m of its own against a maximum that is raised only
// when it must be (diff_exps, below; the sums that would join the maps are known at
// the end only).  S_m^T = K_m Q_m^T puts keys on
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
constexpr int kDiffRows = 128, kDiffThreads = 256;  // 4 waves of 32 rows

// A call as the kernel takes it: the tensors, and the cache that k and v are
// (cache_seqlens set).
struct DiffFwd {
    fa_diff_fwd_args a;
    const int32_t *cache_seqlens, *cache_batch_idx, *block_table;
    int64_t block_table_stride;
    int32_t seqlen_new, page, num_pages, capacity, cache_batch;
    int32_t *status;
};

// The softmax of one map's 32 keys of S^T: exponentials against a maximum m that is
// not looked for.  P and the sum are right against any m near a row's maximum, so m
// stays what it is until a lane's sum of 16 P passes kDiffTop (or is infinite or NaN:
// at first m is -infinity), which 16-bit P would not hold much longer; then the
// tile's scores are taken once more, and m is raised to their maximum and O and the
// sum rescaled.  m is never above the row's maximum, so small P lose nothing either.
// The running maximum that this replaces, kept up lazily, was a quarter of the VALU
// work that bounds the kernel beside its MFMAs, and the exponentials waited for it:
// b 4, s 4096, 16 heads of 128, causal, bf16 505 -> 455 us; 64 channels, s 4096,
// fp16 672 -> 605 us; an exact maximum had cost 15 % more.
// P is rounded to 16 bits for the product with V, as in ordinary attention's forward (its
// 2^-9 in bf16 weighs as the output's own rounding does).  Carrying the remainder, as
// ordinary attention's prompt chunks over a cache and the decode kernel here do, takes 32
// MFMAs more beside 48: two paged chunks of 512 queries over 4 k and 12 k tokens 256 ->
// 361 us, for an error of 1.0 times a plain form's instead of 1.5 (bf16; fp16 1.3).  O
// and the LSE are normalised by the fp32 sum of the unrounded P.
constexpr float kDiffTop = 32768.f;

// P of keys up to lim (relative to the first) in place of their scores; returns their sum.
template <bool MASK>
__device__ __forceinline__ float diff_exps(f32x16 &s, float m, float cscale, int lim, int hh) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float x = fmaf(s[e], cscale, -m);
        if constexpr (MASK) x = acc_lrow(e, hh) > lim ? -INFINITY : x;
        s[e] = exp2_fast(x);
        sum += s[e];
    }
    return sum;
}

// Raises m to the maximum of the visible scores, O and the sum l with it.
template <int HD, bool MASK>
__device__ __forceinline__ void diff_raise(const f32x16 &s, f32x16 (&o)[HD / 32], float &m, float &l, float cscale,
                                           int lim, int hh) {
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, MASK && acc_lrow(e, hh) > lim ? -INFINITY : s[e]);
    mx = max2_xor32(mx);
    const float m_new = fmaxf(m, mx == -INFINITY ? mx : mx * cscale);
    const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m - m_new);
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    m = m_new;
}

// A workgroup's work: gp = 2^lg heads of one GQA group at P = 128 / gp positions
// from m0, which share the K / V tiles; a wave takes 32 rows of one head.
struct DiffWork {
    int b, h, hk, q_start, sq, sk, m0, P, causal_off, n_keys;  // n_keys: keys that some row sees
    const f16 *kp, *vp;
    bool live;
};

// The sequence of rank r when a cache's sequences are sorted by length, longest
// first (as they come where a wave has no lane for each).
__device__ __forceinline__ int diff_nth_longest(const int32_t *lens, int batch, int r) {
    if (batch == 1 || batch > 64) return r;
    const int lane = threadIdx.x & 63, mine = lens[min(lane, batch - 1)];
    int rank = 0;
    for (int j = 0; j < batch; ++j) {
        const int other = __builtin_amdgcn_readlane(mine, j);
        rank += other > mine || (other == mine && j < lane);
    }
    return __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(lane < batch && rank == r)) - 1;
}

template <bool CAUSAL, bool CACHE, int NG>
__device__ __forceinline__ DiffWork diff_work(const DiffFwd &p, int num_m_blocks, int lg, int bid) {
    const fa_diff_fwd_args &a = p.a;
    DiffWork w;
    const int gp = 1 << lg, packs = a.nheads >> lg;
    int mb;
    w.P = kDiffRows / NG >> lg;
    if (a.work_order && a.cu_seqlens_q) {
        const int it = a.work_order[bid / packs];
        w.b = __builtin_amdgcn_readfirstlane(it / num_m_blocks);
        mb = __builtin_amdgcn_readfirstlane(it - w.b * num_m_blocks);
        w.h = (bid % packs) * gp;
    } else if (CACHE && NG == 2) {
        const int per = num_m_blocks * packs, r = bid / per;
        w.b = __builtin_amdgcn_readfirstlane(diff_nth_longest(p.cache_seqlens, a.batch, r));
        mb = (bid - r * per) / packs;
        w.h = (bid - r * per - mb * packs) * gp;
        if (CAUSAL) mb = num_m_blocks - 1 - mb;
    } else {
        const int bp_count = a.batch * packs, bp = bid % bp_count;
        mb = bid / bp_count;
        if (CAUSAL) mb = num_m_blocks - 1 - mb;  // heaviest first
        w.b = bp / packs;
        w.h = (bp - w.b * packs) * gp;
    }
    w.hk = w.h / (a.nheads / a.nheads_k);
    const bool packed_k = a.cu_seqlens_k != nullptr;
    const DiffRows qr = diff_rows(a.cu_seqlens_q, w.b, a.seqlen_q, a.o_rows);
    DiffRows kr = diff_rows(a.cu_seqlens_k, w.b, a.seqlen_k, a.k_rows);
    int kb = w.b;
    if constexpr (CACHE) {
        // A length or a cache row outside the cache leaves the sequence with no
        // keys, and the status word says so: no access leaves the cache.
        const int used = p.cache_seqlens[w.b];
        if (p.cache_batch_idx) kb = p.cache_batch_idx[w.b];
        const int err = (used < 0 || int64_t(used) + p.seqlen_new > p.capacity ? 1 : 0) |
                        (p.cache_batch_idx && (kb < 0 || kb >= p.cache_batch) ? 2 : 0);
        kr.n = err ? 0 : used + p.seqlen_new;
        if (err) {
            kb = 0;
            if (p.status && threadIdx.x == 0) atomicOr(p.status, err);
        }
        if (p.block_table) kb = 0;
    }
    w.q_start = qr.start;
    w.sq = qr.n;
    w.sk = kr.n;
    w.m0 = mb * w.P;
    w.causal_off = w.sk - w.sq;  // key j is visible to query i iff j <= i + causal_off
    w.n_keys = CAUSAL ? max(0, min(w.sk, w.m0 + w.P + w.causal_off)) : w.sk;
    w.kp = (const f16 *)a.k.ptr + base_off(a.k, packed_k, kb, kr.start, w.hk);
    w.vp = (const f16 *)a.v.ptr + base_off(a.v, packed_k, kb, kr.start, w.hk);
    w.live = w.m0 < w.sq;
    return w;
}

// LSE rows of a block past its sequence: 0.
__device__ __forceinline__ void diff_pad_lse(const fa_diff_fwd_args &a, const DiffWork &w, int lg) {
    const int64_t plane = int64_t(a.batch) * a.nheads * a.lse_seqlen;
    float *lse = a.lse + (int64_t(w.b) * a.nheads + w.h) * a.lse_seqlen;
    for (int i = threadIdx.x; i < w.P << lg; i += blockDim.x) {
        const int row = w.m0 + i % w.P;
        if (row < a.lse_seqlen) lse[int64_t(i / w.P) * a.lse_seqlen + row] = lse[plane + int64_t(i / w.P) * a.lse_seqlen + row] = 0.f;
    }
}

// Q^T of query qi of head h as B operands: lane (query, hh), K step g covers channels 16g + 8hh + 0..7.
template <int HD>
__device__ __forceinline__ void diff_load_q(const fa_diff_fwd_args &a, const DiffWork &w, int h, int qi, int hh,
                                            f16x8 (&qB)[HD / 16]) {
    const f16 *qp = (const f16 *)a.q.ptr + base_off(a.q, a.cu_seqlens_q != nullptr, w.b, w.q_start, h) +
                    int64_t(qi < w.sq ? qi : 0) * a.q.row_stride + 8 * hh;
#pragma unroll
    for (int g = 0; g < HD / 16; ++g) {
        u32x4 v = qi < w.sq ? ldg16(qp + 16 * g) : zero_u4();
        if (a.softmax_scale < 0.f) v = neg_h8(v);
        qB[g] = as_h8(v);
    }
}

// Channel tiles [D0, D1) of a row of o (and o2), from both maps' O, maxima and
// sums; the LSEs go with the first one.
template <int HD, bool BF, int D0, int D1>
__device__ __forceinline__ void diff_store(const fa_diff_fwd_args &a, const DiffWork &w, int h, int qi, int hh,
                                           const f32x16 (&o)[2][HD / 32], const float (&mx)[2], const float (&sum)[2]) {
    const int64_t plane = int64_t(a.batch) * a.nheads * a.lse_seqlen;
    float *lse_row = a.lse + (int64_t(w.b) * a.nheads + h) * a.lse_seqlen;
    if (qi >= w.sq) {
        if (D0 == 0 && hh == 0 && qi < a.lse_seqlen) lse_row[qi] = lse_row[plane + qi] = 0.f;
        return;
    }
    const float l0 = sum[0], l1 = sum[1];
    const bool packed_q = a.cu_seqlens_q != nullptr;
    const float lam = diff_lam(a.lam, w.b, w.q_start + qi, h);
    // A sum of 0 is that of a map without a visible key (or with scores of -infinity alone); one that is NaN goes on
    // to the outputs.
    const bool none = l0 == 0.f && l1 == 0.f;
    const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
    f16 *orow = (f16 *)a.o.ptr + base_off(a.o, packed_q, w.b, w.q_start, h) + int64_t(qi) * a.o.row_stride + 4 * hh;
    f16 *o2row = a.o2.ptr ? (f16 *)a.o2.ptr + base_off(a.o2, packed_q, w.b, w.q_start, h) +
                                int64_t(qi) * a.o2.row_stride + 4 * hh
                          : nullptr;
#pragma unroll
    for (int dt = D0; dt < D1; ++dt)
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4) {
            float x[4], y[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                y[t] = o[1][dt][4 * a4 + t] * i1;
                x[t] = none ? 0.f : fmaf(o[0][dt][4 * a4 + t], i0, -lam * y[t]);
            }
            *reinterpret_cast<f16x4 *>(orow + dt * 32 + 8 * a4) = pack4<BF>(x[0], x[1], x[2], x[3]);
            if (o2row) *reinterpret_cast<f16x4 *>(o2row + dt * 32 + 8 * a4) = pack4<BF>(y[0], y[1], y[2], y[3]);
        }
    if (D0 == 0 && hh == 0) {
        lse_row[qi] = l0 == 0.f ? 0.f : (mx[0] + log2_fast(l0)) * kLn2;
        lse_row[plane + qi] = l1 == 0.f ? 0.f : (mx[1] + log2_fast(l1)) * kLn2;
    }
}

// First rows of K and V tiles of a dense tensor or of the pages of a cache, block
// after block.  A tile lies in one page (pages are multiples of 64 tokens).
template <bool CACHE>
struct DiffTiles {
    const f16 *k, *v;  // the next block
    int left = 0;      // blocks left in its page
    int next = 0;      // the table's entry after that page
    __device__ __forceinline__ void init(const DiffFwd &p, const DiffWork &w) {
        k = w.kp;
        v = w.vp;
        if (CACHE && p.block_table && w.n_keys > 0) next = scalar_load_ahead(p.block_table + int64_t(w.b) * p.block_table_stride);
    }
    // Goes to block n0 / kDiffBN, which follows the one before.
    __device__ __forceinline__ void step(const DiffFwd &p, const DiffWork &w, int n0) {
        const fa_diff_fwd_args &a = p.a;
        if (CACHE && p.block_table && left-- == 0) {
            const int blk = checked_page(next, p.num_pages, p.status);
            k = w.kp + int64_t(blk) * a.k.batch_stride;
            v = w.vp + int64_t(blk) * a.v.batch_stride;
            left = p.page / kDiffBN - 1;
            // Loaded a page ahead: its latency would stall every wave once a page.
            const int last = (w.n_keys - 1) / p.page;
            next = scalar_load_ahead(p.block_table + int64_t(w.b) * p.block_table_stride + min(n0 / p.page + 1, last));
        } else if (n0 > 0) {
            k += kDiffBN * a.k.row_stride;
            v += kDiffBN * a.v.row_stride;
        }
    }
};

// NG = 1: four waves of 32 rows each.  NG = 2, for grids that do not fill the chip:
// 64 rows, and the two pairs of waves take the two halves of each key block and
// merge through LDS, so that there are twice the workgroups with half the chain
// of products each.  Of these the first workgroup on a CU gets one of the longest
// items and the second one of the shortest; a cache's sequences are sorted by
// length for it.  launch_diff_fwd has what both measured.
template <int HD, bool BF, bool CAUSAL, bool CACHE, int NG>
__global__ __launch_bounds__(kDiffThreads, HD == 64 ? 3 : 2) void diff_fwd_kernel(const DiffFwd p, const int num_m_blocks,
                                                                                    const int lg, const int cus) {
    constexpr int NT = kDiffThreads, BN = kDiffBN;
    constexpr int TILE = BN * HD * 2, STAGE = 2 * TILE;
    constexpr int HG = HD / 32;  // MFMA K steps of one map's channels
    const fa_diff_fwd_args &a = p.a;
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];

    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave4 = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave = NG == 1 ? wave4 : wave4 & 1, grp = NG == 1 ? 0 : wave4 >> 1;
    int bid = blockIdx.x;
    if (NG == 2 && int(gridDim.x) <= 2 * cus && bid >= cus) bid = gridDim.x - 1 - (bid - cus);
    const DiffWork w = diff_work<CAUSAL, CACHE, NG>(p, num_m_blocks, lg, bid);
    if (!w.live) return diff_pad_lse(a, w, lg);
    const int n_blocks = (w.n_keys + BN - 1) / BN;
    const float cscale = uniform(fabsf(a.softmax_scale) * kLog2e);

    DiffCopier<HD, BN, NT> cp;
    cp.init(wave4, lane);
    DiffTiles<CACHE> tiles;
    tiles.init(p, w);
    auto issue = [&](int nb, int st) FA_INLINE {
        tiles.step(p, w, nb * BN);
        const uint32_t tile = lds_addr(smem) + st * STAGE;
        cp.copy(tile, tiles.k, a.k.row_stride, w.sk - nb * BN);
        cp.copy(tile + TILE, tiles.v, a.v.row_stride, w.sk - nb * BN);
    };

    // The wave's 32 rows: head h, positions from q_lo.
    const int h = w.h + (wave >> (3 - NG - lg));
    const int q_lo = w.m0 + 32 * (wave & ((w.P >> 5) - 1));
    const int qi = q_lo + (lane & 31);
    f16x8 qB[HD / 16];
    diff_load_q<HD>(a, w, h, qi, hh, qB);
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
        const int buf = nb & 1, n0 = nb * BN + 32 * grp;
        wait_vmem();
        __syncthreads();  // block nb is in LDS; every wave is done with stage buf ^ 1
        if (nb + 1 < n_blocks) issue(nb + 1, buf ^ 1);
        if (NG > 1 && MASK && n0 >= w.sk) return;
        if (CAUSAL && MASK && n0 > q_lo + 31 + w.causal_off) return;  // no visible key for this wave
        if (q_lo >= w.sq) return;
        // 32 keys at a time: the scores of both maps take as many registers as
        // those of 64 keys of one, with the two O that is what fits.
        // Operand reads run PIPE - 1 steps ahead behind scheduling fences, from
        // the lane's bases with the stage added once per block (opaque, so that
        // no read address is held in registers through the loop).
        constexpr int PIPE = 3, NS = 2 * HG, NPV = 2 * (HD / 32);
        const int soff = buf * STAGE + 32 * grp * (HD * 2);
        static_assert(STAGE % 512 == 0, "stage offsets must be multiples of 512 bytes");
        int ab = rd.a_base + soff, tb0 = rd.tr_base[0] + soff, tb1 = rd.tr_base[1] + soff;
        asm volatile("" : "+v"(ab), "+v"(tb0), "+v"(tb1));
        f16x8 op[PIPE];
        const int lim = (CAUSAL ? min(w.sk - 1, qi + w.causal_off) : w.sk - 1) - n0;
#pragma unroll
        for (int sub = 0; sub < BN / 32 / NG; ++sub) {
            // Step u: map u % 2, K step u / 2 of the map's channels.
            f32x16 s[2];
            auto rd_k = [&](int u) FA_INLINE {
                op[u % PIPE] = rd.a_operand_at(smem + 32 * sub * (HD * 2), ab, (u & 1) * HG + (u >> 1));
            };
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < PIPE - 1; ++u) rd_k(u);
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                if (u + PIPE - 1 < NS) rd_k(u + PIPE - 1);
                s[u & 1] = mfma16<BF>(op[u % PIPE], qB[(u & 1) * HG + (u >> 1)], u < 2 ? zero16() : s[u & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            // Step u: key step u % 2, channel tile u / 2; one V operand for both maps.
            // The first reads go out before the softmax, which covers their latency.
            auto rd_v = [&](int u) FA_INLINE {
                op[u % PIPE] = rd.tr_operand_at(smem + TILE + 16 * (2 * sub + (u & 1)) * (HD * 2), tb0, tb1, u >> 1);
            };
#pragma unroll
            for (int u = 0; u < PIPE - 1; ++u) rd_v(u);
            float part[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) part[m] = diff_exps<MASK>(s[m], mx[m], cscale, lim - 32 * sub, hh);
            // (Each by itself: a maximum of both would pass over a NaN, which scores of -infinity give while m is -infinity.)
            if (__builtin_amdgcn_ballot_w64(!(part[0] <= kDiffTop) || !(part[1] <= kDiffTop)) != 0) {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    f32x16 t = zero16();
#pragma unroll
                    for (int g = 0; g < HG; ++g)
                        t = mfma16<BF>(rd.a_operand_at(smem + 32 * sub * (HD * 2), ab, m * HG + g), qB[m * HG + g], t);
                    diff_raise<HD, MASK>(t, o[m], mx[m], sum[m], cscale, lim - 32 * sub, hh);
                    part[m] = diff_exps<MASK>(t, mx[m] == -INFINITY ? 0.f : mx[m], cscale, lim - 32 * sub, hh);
                    s[m] = t;
                }
            }
            f16x8 pB[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                sum[m] += part[m];
                pB[m][0] = pack16<BF>(s[m], 0);
                pB[m][1] = pack16<BF>(s[m], 8);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < NPV; ++u) {
                if (u + PIPE - 1 < NPV) rd_v(u + PIPE - 1);
#pragma unroll
                for (int m = 0; m < 2; ++m) o[m][u >> 1] = mfma16<BF>(op[u % PIPE], pB[m][u & 1], o[m][u >> 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    // Iterations whose blocks need no mask for any wave of the workgroup come first.
    int n_full = min(n_blocks, w.sk / BN);
    if (CAUSAL) n_full = min(n_full, max(0, (w.m0 + w.causal_off + 1) / BN));
    if (n_blocks > 0) issue(0, 0);
    for (int nb = 0; nb < n_full; ++nb) block(nb, std::false_type{});
    for (int nb = n_full; nb < n_blocks; ++nb) block(nb, std::true_type{});

    sum[0] = sum_xor32(sum[0]);
    sum[1] = sum_xor32(sum[1]);
    if constexpr (NG == 1) {
        diff_store<HD, BF, 0, HD / 32>(a, w, h, qi, hh, o, mx, sum);
    } else {
        // Each group finishes half of the channels of both maps: it hands the other
        // half, and its maxima and sums, to the other group.
        constexpr int H = HD / 64;  // 32-channel tiles of a half
        __shared__ f32x2 ml[2][2][kDiffRows / 2];
        f32x4 *xo = reinterpret_cast<f32x4 *>(smem);  // [group][2 maps * 4 H][GT threads]
        constexpr int GT = NT / 2;
        const int t4 = tid & (GT - 1), r = 32 * wave + (lane & 31);
        static_assert(2 * 2 * 4 * H * GT * 16 <= 2 * STAGE, "the exchange fits the stages");
        __syncthreads();  // every wave is done with the tiles
        if (hh == 0) {
            ml[grp][0][r] = f32x2{mx[0], sum[0]};
            ml[grp][1][r] = f32x2{mx[1], sum[1]};
        }
        auto finish = [&](auto grp_tag) FA_INLINE {
            constexpr int GRP = decltype(grp_tag)::value;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4 * H; ++i) {
                    const f32x16 &t = o[m][(1 - GRP) * H + i / 4];
                    const int e = 4 * (i & 3);
                    xo[((GRP * 2 + m) * 4 * H + i) * GT + t4] = f32x4{t[e], t[e + 1], t[e + 2], t[e + 3]};
                }
            __syncthreads();
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const f32x2 other = ml[1 - GRP][m][r];
                const float top = fmaxf(mx[m], other[0]);
                const float f_own = mx[m] == -INFINITY ? 0.f : exp2_fast(mx[m] - top);
                const float f_other = other[0] == -INFINITY ? 0.f : exp2_fast(other[0] - top);
#pragma unroll
                for (int i = 0; i < 4 * H; ++i) {
                    const f32x4 x = xo[(((1 - GRP) * 2 + m) * 4 * H + i) * GT + t4];
                    f32x16 &t = o[m][GRP * H + i / 4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[4 * (i & 3) + e] = fmaf(x[e], f_other, t[4 * (i & 3) + e] * f_own);
                }
                // In group order, so that both groups have the same bits.
                sum[m] = GRP == 0 ? fmaf(other[1], f_other, sum[m] * f_own) : fmaf(sum[m], f_own, other[1] * f_other);
                mx[m] = top;
            }
            diff_store<HD, BF, GRP * H, GRP * H + H>(a, w, h, qi, hh, o, mx, sum);
        };
        if (grp == 0)
            finish(std::integral_constant<int, 0>{});
        else
            finish(std::integral_constant<int, 1>{});
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
        const int sq = diff_rows(a.cu_seqlens_q, b, a.seqlen_q, a.o_rows).n;
        const int sk = diff_rows(a.cu_seqlens_k, b, a.seqlen_k, a.k_rows).n;
        const int m0 = mb * P;
        if (m0 >= sq) return -1;
        const int64_t rows = min(P, sq - m0);
        const int64_t keys = a.causal ? max(0, min(sk, m0 + P + sk - sq)) : max(sk, 0);
        return int(min<int64_t>(rows * keys / (int64_t(P) * 64), kOrderBuckets - 1));
    }, a.work_order, true);
}

// log2 of the heads of a GQA group that a workgroup's BM rows hold: the largest
// power of two that divides the group and leaves whole 32-row tiles per head.
static int diff_pack_log2(int group, int BM) {
    int lg = 0;
    while ((64 << lg) <= BM && group % (2 << lg) == 0) ++lg;
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
    for (const fa_tensor *t : {&a.k, &a.v})
        if (t->row_stride < 0 || t->row_stride > kDiffMaxRowStride) return FA_ERR_INVALID_ARG;
    return check_tensor(a.o2, false);
}

template <int HD, bool BF, bool CACHE>
static int launch_diff_fwd(const DiffFwd &p, hipStream_t s) {
    const fa_diff_fwd_args &a = p.a;
    int lg, P, nmb;
    int64_t grid;
    auto rows = [&](int BM) {
        lg = diff_pack_log2(a.nheads / a.nheads_k, BM);
        P = BM >> lg;
        nmb = (a.lse_seqlen + P - 1) / P;
        grid = int64_t(nmb) * a.batch * (a.nheads >> lg);
    };
    rows(kDiffRows);
    const int cus = device_cus();
    // Measured with NG = 1 and NG = 2 (fp16, 128 channels, us): 128 tokens, batch 4, 16/4
    // heads 10.8 and 9.2; 16 heads, 1024 tokens 36 and 27; 2048 tokens (grid = CUs) 74 and 67,
    // causal 67 and 47; 20 heads, 2048 tokens, causal (1.25 of the CUs) 72 and 51; batch 3,
    // 1024 tokens, causal 43 and 39; two paged chunks of 512 queries over 4 k and 12 k
    // tokens 401 and 289.  Twice the CUs, 2048 tokens: 118 and 129, causal 79 and 81.
    const bool uneven = a.causal || CACHE;
    const int groups = 2 * grid <= (uneven ? 3 : 2) * cus && a.seqlen_k > 32 ? 2 : 1;
    if (groups == 2) rows(kDiffRows / 2);
    if (grid > 0x7fffffff) return FA_ERR_INVALID_ARG;
    if (a.cu_seqlens_q && (a.work_order || a.o_rows > 0)) {
        const int order_wgs = a.work_order ? 1 : 0;
        hipLaunchKernelGGL(diff_fwd_order_kernel, dim3(order_wgs + (a.o_rows > 0 ? kZeroBlocks : 0)),
                           dim3(kOrderThreads), 0, s, a, nmb, P, order_wgs);
        const int rc = int(hipGetLastError());
        if (rc) return rc;
    }
    if (grid == 0) return FA_OK;
    auto launch = [&](auto causal) {
        constexpr bool C = decltype(causal)::value;
        if (groups == 2)
            hipLaunchKernelGGL((diff_fwd_kernel<HD, BF, C, CACHE, 2>), dim3(unsigned(grid)), dim3(kDiffThreads), 0, s, p,
                               nmb, lg, cus);
        else
            hipLaunchKernelGGL((diff_fwd_kernel<HD, BF, C, CACHE, 1>), dim3(unsigned(grid)), dim3(kDiffThreads), 0, s, p,
                               nmb, lg, cus);
    };
    if (a.causal)
        launch(std::true_type{});
    else
        launch(std::false_type{});
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
