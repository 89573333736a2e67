// Attention of many query rows over a key-value cache in 8 bits (prompt chunks).
//
// A workgroup takes 128 rows of a KV head (its query heads times the query positions) and one piece of the
// sequence's keys, 64 at a time.  Codes go from memory straight to a ring of four LDS stages and stay 8 bits there: half the
// LDS traffic, and each wave converts what it reads.  (Converted once for the workgroup, through registers and 16-bit LDS, a
// call took 183 us against 172: the barriers and writes cost more than the conversions.)  Scales multiply scores and
// probabilities.  Four waves of 32 rows: S^T = K Q^T, so that a lane owns a row, and P^T feeds O^T += V^T P^T from the
// accumulators, half a tile behind.
//
// P times V's scale is rounded to fp16 for both types of q, as P is in the forward kernels: codes make the products exact,
// and 11 bits are no fewer than the output keeps.  Against 64 bits a bf16 output is as far off as one that is rounded alone
// (0.0017 of its norm), an fp16 output up to 1.4 times (0.00027 and 0.00021).  P as hi + lo, which the kernel of few rows has, where
// the product with V costs nothing, would not add that, but half of the products: 175 -> 238 us at 2 x 512 queries over 4k to
// 12k keys, 1145 -> 1605 at 2048 over 32768.  fp16's range suffices because O has a reference of its own, a row's largest
// score + log2(V's scale) so far: keys that a row does not see, or whose probability is small, take no bits from the others,
// whatever their V is.  What rounds to 0 is 2^-30 of the row's largest p * scale.
//
// What bounds it: matrix and vector instructions of the same SIMDs, 43 and 65 % of the cycles at 2 x 512 queries over 4k to
// 12k tokens (32/8 heads of 128, e4m3, bf16: 173 us a call, 0.86 PFLOP/s), 0.99 PFLOP/s at 2048 queries over 32768 (1148 us); int8
// takes a quarter to a third longer (218 and 1482): 10 or 12 instructions convert an operand where e4m3 has 4.  Row tiles of a
// KV head share an XCD's L2 (kv8_item).
#include <algorithm>

#include "fa_kv8_common.h"

namespace fa {

constexpr int kKcThreads = 256, kKcKeys = 64, kKcHalves = kKcThreads;
// P is 2^5 at its reference, which is raised when the sum of a lane's 16, or their softmax sum, passes 2^15: fp16 holds it,
// with all its bits down to 2^-19 of the reference.
constexpr float kKcTop = 32768.f, kKcLift = 5.f, kKcNoLift = -160.f;

template <int HD, bool BF, bool INT8>
__global__ __launch_bounds__(kKcThreads, 2) void kv8_chunk_kernel(const Kv8Call call) {
    kv8_early();
    const fa_kv8_args &a = call.a;
    const Kv8Plan &plan = call.plan;
    constexpr int CH = HD / 16, TILE = kKcKeys * HD, STAGE = 2 * TILE, NST = 4;
    constexpr int DT = HD / 32;
    __shared__ __attribute__((aligned(1024))) char smem[NST * STAGE];
    // Halves of tiles (32 keys, which lie in one page and one block of scales): where their codes begin, k's scale with the
    // softmax's, V's as what it adds to the exponents of P, and what it adds to scores: 0 or NaN.
    struct Half {
        const char *k, *v;
        float k_scale, lift, nan, pad;
    };
    __shared__ __attribute__((aligned(16))) Half halves[kKcHalves];
    __shared__ int ticket;

    const fa_kv8_cache &c = a.cache;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int HI = c.nheads_k * plan.row_tiles;
    int slot_i, hk, rt;
    if (!kv8_item(plan, c.nheads_k, blockIdx.x, slot_i, hk, rt)) return;
    const int hi_i = hk * plan.row_tiles + rt;
    const Kv8Slot sl = kv8_slot(a, plan, slot_i);
    if (sl.b < 0) return;
    const int G = a.nheads / c.nheads_k, R = G * a.seqlen_q, L = sl.keys, shift = L - a.seqlen_q;
    const int w_row0 = rt * kKcRows + wave * 32, row = w_row0 + col;
    const bool row_ok = row < R;
    const int qpos = row_ok ? row / G : 0, hq = hk * G + (row_ok ? row - qpos * G : 0);
    const int first = kv8_first(a, qpos + shift), last = kv8_last(a, qpos + shift, L);
    // Query positions of the workgroup's rows, and of the wave's.
    const int g_lo = rt * kKcRows / G, g_hi = (min(rt * kKcRows + kKcRows, R) - 1) / G;
    const int w_lo = min(w_row0, R - 1) / G, w_hi = (min(w_row0 + 32, R) - 1) / G;
    const int s0 = max(sl.begin, kv8_first(a, g_lo + shift)) / 32 * 32, s1 = min(sl.end, kv8_last(a, g_hi + shift, L) + 1);
    // Keys that some row of the wave sees, and that all see.
    const int any_first = kv8_first(a, w_lo + shift), any_last = w_row0 < R ? kv8_last(a, w_hi + shift, L) : -1;
    const int all_first = kv8_first(a, w_hi + shift), all_last = min(kv8_last(a, w_lo + shift, L), s1 - 1);

    // Q^T as B operands.
    const float cscale = fabsf(a.softmax_scale) * kLog2e;
    f16x8 qB[HD / 16];  // step g: channels 32 (g / 2) + 16 hh + 8 (g % 2) + 0..7
    {
        const f16 *qp = (const f16 *)a.q.ptr + int64_t(sl.b) * a.q.batch_stride + int64_t(qpos) * a.q.row_stride +
                        int64_t(hq) * a.q.head_stride + 16 * hh;
#pragma unroll
        for (int g = 0; g < HD / 16; ++g) {
            qB[g] = as_h8(row_ok ? ldg16(qp + 32 * (g / 2) + 8 * (g % 2)) : zero_u4());
        }
    }

    // Copies of a tile's codes to LDS, straight from memory: chunk c of row r of a half lies at chunk c ^ kv8_swz(r).  A wave
    // takes one half of K (waves 0, 1) or V.
    constexpr int RPC = 1024 / HD, CPH = 32 / RPC;  // rows of a copy, copies of a half
    const int64_t rs = wave < 2 ? c.k.row_stride : c.v.row_stride;  // (at most 2^23)
    const int row0 = lane / CH;
    uint32_t off[CPH];
#pragma unroll
    for (int i = 0; i < CPH; ++i) off[i] = uint32_t(row0) * uint32_t(rs) + 16 * (lane % CH ^ kv8_swz<HD>(row0 + i * RPC));
    const uint32_t lds0 = lds_addr(smem) + wave * (32 * HD);
    auto issue = [&](int x, int base) FA_INLINE {
        const int h = 2 * x + (wave & 1), most = L - 1 - min(base + 32 * h, (L - 1) / 32 * 32);
        const uint32_t to = lds0 + (x % NST) * STAGE;
        const char *from = uniform(wave < 2 ? halves[h].k : halves[h].v);
        if (most >= 31) {
#pragma unroll
            for (int i = 0; i < CPH; ++i) g2l16_at((const f16 *)(from + i * RPC * rs), off[i], to + i * 1024);
        } else {
            // Rows past the sequence re-read its last one, so that no stale code reaches a product.
#pragma unroll
            for (int i = 0; i < CPH; ++i)
                g2l16_at((const f16 *)from, uint32_t(min(row0 + i * RPC, most)) * uint32_t(rs) + off[i] - uint32_t(row0) * uint32_t(rs), to + i * 1024);
        }
    };
    // Operand reads: rows sigma(col) of K, 16 codes of two steps; V transposed, eight keys of a channel.
    const int kr = sigma(col), k_at = kr * HD + ((hh ^ kv8_swz<HD>(kr)) << 4);
    const int vr = 8 * hh + (lane & 15) / 2, v_at = vr * HD + ((((lane >> 4) & 1) ^ kv8_swz<HD>(vr)) << 4) + 8 * (lane & 1);
    f32x16 o[DT], s[2];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = zero16();
    float m = -INFINITY, mo = -INFINITY, l = 0.f;  // references of the sum and of O, the sum
    constexpr int NS = HD / 16, NPV = 2 * DT, EPS = 16 / NS;  // EPS: exponentials of a step
    constexpr int KP = HD == 128 ? 3 : 2, VP = 4;  // reads in flight, and the next
    u32x4 kc[KP];
    u32x2 vc[VP];
    for (int base = s0; base < s1; base += 32 * kKcHalves) {
        const int n_tiles = (min(s1 - base, 32 * kKcHalves) + kKcKeys - 1) / kKcKeys;
        {
            // The places and scales of the next halves, one a thread; halves behind the sequence repeat its last.
            const int p0 = min(base + 32 * tid, (L - 1) / 32 * 32);
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
            const float ks = c.k_scale.ptr[line * c.k_scale.batch_stride + int64_t(blk) * c.k_scale.row_stride + int64_t(hk) * c.k_scale.head_stride];
            const float vs = c.v_scale.ptr[line * c.v_scale.batch_stride + int64_t(blk) * c.v_scale.row_stride + int64_t(hk) * c.v_scale.head_stride];
            halves[tid].k = (const char *)c.k.ptr + line * c.k.batch_stride + int64_t(at) * c.k.row_stride + int64_t(hk) * c.k.head_stride;
            halves[tid].v = (const char *)c.v.ptr + line * c.v.batch_stride + int64_t(at) * c.v.row_stride + int64_t(hk) * c.v.head_stride;
            __syncthreads();
            for (int x = 0; x < min(3, n_tiles); ++x) issue(x, base);  // (the waits below are theirs, too)
            // V's scale as a power of P (of 0: under that of any number); where one of the two is not finite, the scores of its
            // keys are NaN.
            f32x4 h;
            h[0] = ks * cscale;
            h[2] = ks * 0.f + vs * 0.f;
            h[1] = fmaxf(log2_fast(h[2] == 0.f ? vs : 0.f), kKcNoLift);
            h[3] = 0.f;
            *reinterpret_cast<f32x4 *>(&halves[tid].k_scale) = h;
            wait_vmem();
            if (base == s0 && a.softmax_scale < 0.f) {
#pragma unroll
                for (int g = 0; g < HD / 16; ++g) qB[g] = as_h8(neg_h8(__builtin_bit_cast(u32x4, qB[g])));
            }
            __syncthreads();
        }
        // Scores of 32 keys: step u of NS, a read of 16 codes for two.
        auto k_read = [&](const char *tile, int j) FA_INLINE { kc[j % KP] = *reinterpret_cast<const u32x4 *>(tile + (k_at ^ (j << 5))); };
        auto k_operand = [&](int u) FA_INLINE {
            const u32x4 q = kc[u / 2 % KP];
            return kv8_decode<INT8, BF>(u % 2 ? u32x2{q[2], q[3]} : u32x2{q[0], q[1]});
        };
#pragma unroll
        for (int u = 0; u < NS; ++u) {
            if (u % 2 == 0) k_read(smem, u / 2);
            s[0] = mfma16<BF>(k_operand(u), qB[u], u < 1 ? zero16() : s[0]);
        }
        for (int t = 0; t < n_tiles; ++t) {
            // Tile t + 1 has landed for this wave, and after the barrier for all (t + 2 may be on its way); every wave is done
            // with tile t - 1, whose place t + 3 takes.
            if (t + 2 < n_tiles)
                wait_vmem_n<CPH>();
            else
                wait_vmem();
            __syncthreads();
            if (t + 3 < n_tiles) issue(t + 3, base);
            // Half h of tile t, with its scores in s[h]: its softmax runs between the products of the next half's scores.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x16 &sc = s[h], &sn = s[1 - h];
                const int p0 = base + t * kKcKeys + 32 * h;
                const bool some = p0 <= any_last && p0 + 32 > any_first;  // (of the wave)
                const char *kt = smem + (h == 0 ? t % NST : (t + 1) % NST) * STAGE + (h == 0 ? 32 * HD : 0);
                const char *vt = smem + t % NST * STAGE + TILE + 32 * h * HD;
                // Step u: channel tile u % DT, 16 keys u / DT (row bit 4 is bit HD / 2 of the swizzle).
                auto v_read = [&](int u) FA_INLINE { vc[u % VP] = lds_tr8(vt, 16 * (u / DT) * HD + (v_at ^ (u % DT << 5) ^ u / DT * (HD / 2))); };
                if (some) {
                    const f32x4 x4 = *reinterpret_cast<const f32x4 *>(&halves[2 * t + h].k_scale);
                    float sk = uniform(x4[0]), d = x4[2];
                    if (p0 < all_first || p0 + 31 > all_last) {
                        const int lo = first - p0 - 8 * hh, hi = min(last, s1 - 1) - p0 - 8 * hh;
                        d = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int key = acc_lrow(r, 0);
                            const float x = fmaf(sc[r], sk, x4[2]);
                            sc[r] = key < lo || key > hi ? -INFINITY : x;
                        }
                        sk = 1.f;
                    }
                    // Exponentials of the half, with its largest at most 2^15 over the references, which are those of the last
                    // raise: their sum says so.  p is what scores are raised by: V's scale over O's reference, or 2^-64 over
                    // the sum's where that is more.  (Such keys are 0 in P, and still all there in the sum.)
                    auto power = [&]() FA_INLINE { return m == -INFINITY ? 0.f : fmaxf(x4[1] - mo, -64.f - m); };
                    float p = power(), sum = 0.f;
                    const float dm = p + d;
                    f16x8 pB[2];
                    __builtin_amdgcn_s_setprio(1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < KP - 1; ++j) k_read(kt, j);
#pragma unroll
                    for (int u = 0; u < NS; ++u) {
                        if (u % 2 == 0 && u / 2 + KP - 1 < NS / 2) k_read(kt, u / 2 + KP - 1);
                        if (u >= NS - (VP - 1)) v_read(u - (NS - (VP - 1)));
                        sn = mfma16<BF>(k_operand(u), qB[u], u < 1 ? zero16() : sn);
#pragma unroll
                        for (int e = u * EPS; e < u * EPS + EPS; ++e) {
                            sc[e] = exp2_fast(fmaf(sc[e], sk, dm));
                            sum += sc[e];
                            if (e % 8 == 7) pB[e / 8] = pack8(sc, e - 7);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    // A row without a reference gets one from the first half that shows it a key, whatever the sum: scores far
                    // below 0 leave a sum of 0.
                    const bool fresh = m == -INFINITY && max(first, p0) <= min(min(last, s1 - 1), p0 + 31);
                    float sum_l = m == -INFINITY ? sum : sum * exp2_fast(-p - m);
                    if (__builtin_amdgcn_ballot_w64(sum > kKcTop || sum_l > kKcTop || fresh) != 0) {
                        // The scores again, their maximum as the new reference; with V's scale for O's.
                        const char *kt0 = smem + t % NST * STAGE + 32 * h * HD;
                        f32x16 x = zero16();
#pragma unroll
                        for (int u = 0; u < NS; ++u) {
                            const u32x4 q = *reinterpret_cast<const u32x4 *>(kt0 + (k_at ^ (u / 2 << 5)));
                            x = mfma16<BF>(kv8_decode<INT8, BF>(u % 2 ? u32x2{q[2], q[3]} : u32x2{q[0], q[1]}), qB[u], x);
                        }
                        const int lo = first - p0 - 8 * hh, hi = min(last, s1 - 1) - p0 - 8 * hh;
                        float top = -INFINITY;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int key = acc_lrow(r, 0);
                            x[r] = key < lo || key > hi ? -INFINITY : fmaf(x[r], x4[0], x4[2]);
                            top = fmaxf(top, x[r]);
                        }
                        top = max2_xor32(top);
                        const float m_new = fmaxf(m, top), mo_new = fmaxf(mo, top + x4[1] - kKcLift);
                        const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(mo - mo_new);
                        l *= m_new == -INFINITY ? 1.f : exp2_fast(m - m_new);
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
                        m = m_new;
                        mo = mo_new;
                        p = power();
                        sum = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            x[r] = exp2_fast(x[r] + p);
                            sum += x[r];
                        }
                        pB[0] = pack8(x, 0);
                        pB[1] = pack8(x, 8);
                        sum_l = m == -INFINITY ? sum : sum * exp2_fast(-p - m);
                    }
                    l += sum_l;
#pragma unroll
                    for (int u = 0; u < NPV; ++u) {
                        const f16x8 v = kv8_decode<INT8, false>(vc[u % VP]);
                        if (u + VP - 1 < NPV) v_read(u + VP - 1);
                        o[u % DT] = mfma16<false>(v, pB[u / DT], o[u % DT]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    __builtin_amdgcn_s_setprio(0);
                } else {
#pragma unroll
                    for (int u = 0; u < NS; ++u) {
                        if (u % 2 == 0) k_read(kt, u / 2);
                        sn = mfma16<BF>(k_operand(u), qB[u], u < 1 ? zero16() : sn);
                    }
                }
            }
        }
        __syncthreads();  // every wave is done with the table and the tiles
    }

    const Kv8Call &late = kv8_late();
    // O on the sum's reference.
    const float out_scale = m == -INFINITY ? 1.f : exp2_fast(mo - m);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= out_scale;
    l = sum_xor32(l);
    if (sl.n_pieces > 1) {
        // Partial results lane by lane: (maximum, sum) of every row, then register pairs of O by wave and lane.
        const int F = kv8_group(sl.n_pieces, kKcRows * HD * 4), g0 = sl.ch / F * F, in_group = min(F, sl.n_pieces - g0), groups = (sl.n_pieces + F - 1) / F;
        const int64_t part0 = int64_t(sl.part - sl.ch) * HI + hi_i;
        auto ml_at = [&](int i) { return kv8_ml(late.a, late.plan, part0 + int64_t(i) * HI) + wave * 32 + col; };
        auto o_at = [&](int i, int j) { return kv8_o<HD>(late.a, late.plan, part0 + int64_t(i) * HI) + (wave * (HD / 4) + j) * 64 + lane; };
        auto put = [&](int i) FA_INLINE {
            if (hh == 0) kv8_put(ml_at(i), f32x2{m, l});
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; r += 2) kv8_put(o_at(i, dt * 8 + r / 2), f32x2{o[dt][r], o[dt][r + 1]});
        };
        // Pieces first, first + step, .. (n of them) in their order; the own one's results are still in registers.
        auto join = [&](int first, int step, int n, int own_i) FA_INLINE {
            float mm = m;
            for (int k = 0; k < n; ++k)
                if (first + k * step != own_i) mm = fmaxf(mm, kv8_get(ml_at(first + k * step))[0]);
            const float own = m == -INFINITY ? 0.f : exp2_fast(m - mm), l_own = l;
            f32x16 sum[DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) sum[dt] = zero16();
            l = 0.f;
            for (int k = 0; k < n; ++k) {
                const int i = first + k * step;
                if (i == own_i) {
                    l = fmaf(l_own, own, l);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int r = 0; r < 16; ++r) sum[dt][r] = fmaf(own, o[dt][r], sum[dt][r]);
                    continue;
                }
                const f32x2 ml = kv8_get(ml_at(i));
                f32x2 y[DT * 8];
#pragma unroll
                for (int j = 0; j < DT * 8; ++j) y[j] = kv8_get(o_at(i, j));
                const float f = ml[0] == -INFINITY ? 0.f : exp2_fast(ml[0] - mm);
                l = fmaf(ml[1], f, l);
#pragma unroll
                for (int j = 0; j < DT * 8; ++j) {
                    sum[j / 8][j % 8 * 2] = fmaf(f, y[j][0], sum[j / 8][j % 8 * 2]);
                    sum[j / 8][j % 8 * 2 + 1] = fmaf(f, y[j][1], sum[j / 8][j % 8 * 2 + 1]);
                }
            }
            m = mm;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = sum[dt];
        };
        put(sl.ch);
        if (!kv8_count(kv8_counter(late.a, late.plan.items + part0 + int64_t(g0) * HI), in_group, &ticket)) return;
        join(g0, 1, in_group, sl.ch);
        if (groups > 1) {
            put(g0);
            if (!kv8_count(kv8_counter(late.a, int64_t(sl.b) * HI + hi_i), groups, &ticket)) return;
            join(0, F, groups, g0);
        }
    }
    // Opaque to the optimiser: the row's output addresses are formed here, not before the loop and held through it.
    int orow = row;
    asm volatile("" : "+v"(orow));
    if (orow >= R) return;
    const int oq = orow / G, oh = hk * G + orow - oq * G;
    // A sum of 0 is that of a row without a visible key (or with scores of -infinity alone); NaN goes on to the output.
    const float inv = l == 0.f ? 0.f : 1.f / l;
    f16 *out = (f16 *)late.a.o.ptr + int64_t(sl.b) * late.a.o.batch_stride + int64_t(oq) * late.a.o.row_stride + int64_t(oh) * late.a.o.head_stride + 4 * hh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            f16x4 y = pack4<BF>(o[dt][r] * inv, o[dt][r + 1] * inv, o[dt][r + 2] * inv, o[dt][r + 3] * inv);
            if (l == 0.f) y = pack4<BF>(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<f16x4 *>(out + 32 * dt + 2 * r) = y;
        }
    if (hh == 0) late.a.lse[(int64_t(sl.b) * late.a.nheads + oh) * late.a.seqlen_q + oq] = l == 0.f ? 0.f : (m + log2_fast(l)) * kLn2;
}

int kv8_chunk(const fa_kv8_args &a, const Kv8Plan &plan, hipStream_t s) {
    const unsigned grid = unsigned(kv8_grid(plan, a.cache.nheads_k));
    return kv8_by_type(a.cache.head_dim, a.dtype, a.cache.kind, [&](auto hd, auto bf, auto int8) {
        hipLaunchKernelGGL((kv8_chunk_kernel<decltype(hd)::value, decltype(bf)::value, decltype(int8)::value>), dim3(grid),
                           dim3(kKcThreads), 0, s, Kv8Call{a, plan});
        return int(hipGetLastError());
    });
}

}  // namespace fa
