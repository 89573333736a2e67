// Attention of many query rows over a key-value cache in 8 bits (prompt chunks).
//
// A workgroup takes 128 rows of a KV head (its query heads times the query positions) and one piece of the
// sequence's keys, 64 at a time.  Codes come from memory through registers, are converted once for the workgroup and lie in
// LDS in 16 bits, in the layout from which the products of ordinary attention are fed; their scales multiply
// scores and probabilities.  Four waves of 32 rows: S^T = K Q^T, so that a lane owns a row, and P^T feeds
// O^T += V^T P^T from the accumulators.  P is fp16 for both types of q, which codes allow: exact products
// and 11 bits where bf16 has 8.
#include <algorithm>

#include "fa_kv8_common.h"

namespace fa {

constexpr int kKcThreads = 256, kKcKeys = 64;
// P is kept times 2^7 and its maximum within 2^8 of the reference, so at most 2^15 in fp16; it loses bits under 2^-21.
constexpr float kKcRaise = 8.f, kKcLift = 7.f;

template <int HD, bool BF, bool INT8>
__global__ __launch_bounds__(kKcThreads, 2) void kv8_chunk_kernel(const fa_kv8_args a, const Kv8Plan plan) {
    constexpr int CH = HD / 16, TILE = kKcKeys * HD * 2, STAGE = 2 * TILE;
    constexpr int CPT = kKcKeys * CH / kKcThreads;  // chunks of 16 codes a thread for K or V of a tile
    constexpr int DT = HD / 32;
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
    __shared__ int ticket;

    const fa_kv8_cache &c = a.cache;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int HI = c.nheads_k * plan.row_tiles;
    const int slot_i = blockIdx.x / HI, hi_i = blockIdx.x % HI, hk = hi_i / plan.row_tiles, rt = hi_i % plan.row_tiles;
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
    const int n_tiles = s0 < s1 ? (s1 - s0 + kKcKeys - 1) / kKcKeys : 0;
    // Keys that some row of the wave sees, and that all see.
    const int any_first = kv8_first(a, w_lo + shift), any_last = w_row0 < R ? kv8_last(a, w_hi + shift, L) : -1;
    const int all_first = kv8_first(a, w_hi + shift), all_last = min(kv8_last(a, w_lo + shift, L), s1 - 1);

    // Q^T as B operands.
    const bool neg = a.softmax_scale < 0.f;
    const float cscale = fabsf(a.softmax_scale) * kLog2e;
    f16x8 qB[HD / 16];
    {
        const f16 *qp = (const f16 *)a.q.ptr + int64_t(sl.b) * a.q.batch_stride + int64_t(qpos) * a.q.row_stride +
                        int64_t(hq) * a.q.head_stride + 8 * hh;
#pragma unroll
        for (int g = 0; g < HD / 16; ++g) {
            u32x4 v = row_ok ? ldg16(qp + 16 * g) : zero_u4();
            qB[g] = as_h8(neg ? neg_h8(v) : v);
        }
    }

    // Codes of a tile in registers, the scales of its halves of 32 keys.  A half lies in one page and one block of scales.
    u32x4 kr[CPT], vr[CPT];
    struct Half {
        float k, v;
    } next[2], now[2];
    const int my_row = tid / CH, my_ch = tid % CH;
    auto load = [&](int t) FA_INLINE {
        const char *kb[2], *vb[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int p0 = min(s0 + t * kKcKeys + 32 * h, (L - 1) / 32 * 32);  // keys past the sequence: any of its blocks
            int64_t line = sl.row;
            int at = p0;
            if (c.block_table) {
                const int pg = p0 / c.page_block_size;
                line = checked_page(scalar_load_ahead(c.block_table + int64_t(sl.b) * c.block_table_stride + pg), c.num_pages, c.status);
                at = p0 - pg * c.page_block_size;
            }
            const int blk = at / c.scale_block;
            next[h].k = scalar_float(c.k_scale.ptr + line * c.k_scale.batch_stride + int64_t(blk) * c.k_scale.row_stride +
                                     int64_t(hk) * c.k_scale.head_stride);
            next[h].v = scalar_float(c.v_scale.ptr + line * c.v_scale.batch_stride + int64_t(blk) * c.v_scale.row_stride +
                                     int64_t(hk) * c.v_scale.head_stride);
            kb[h] = (const char *)c.k.ptr + line * c.k.batch_stride + int64_t(at) * c.k.row_stride + int64_t(hk) * c.k.head_stride;
            vb[h] = (const char *)c.v.ptr + line * c.v.batch_stride + int64_t(at) * c.v.row_stride + int64_t(hk) * c.v.head_stride;
        }
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
            const int r = i * (kKcThreads / CH) + my_row;  // HD 128: half i; HD 64: half wave / 2
            const int h = CPT == 2 ? i : wave >> 1;
            // Rows past the sequence re-read its last one, so that no stale code reaches a product.
            const int p0 = min(s0 + t * kKcKeys + 32 * h, (L - 1) / 32 * 32), rr = min(r & 31, L - 1 - p0);
            kr[i] = *reinterpret_cast<const u32x4 *>(kb[h] + int64_t(rr) * c.k.row_stride + 16 * my_ch);
            vr[i] = *reinterpret_cast<const u32x4 *>(vb[h] + int64_t(rr) * c.v.row_stride + 16 * my_ch);
        }
    };
    // The codes in 16 bits to LDS.  Odd rows write their upper eight first: 16 lanes then cover all banks.
    auto store = [&](int st) FA_INLINE {
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
            const int r = i * (kKcThreads / CH) + my_row, odd = r & 1, sw = swz<HD / 8>(r);
            char *const base = smem + st * STAGE + r * (HD * 2);
            const int c0 = ((2 * my_ch + odd) ^ sw) << 4, c1 = ((2 * my_ch + 1 - odd) ^ sw) << 4;
            const f16x8 k0 = kv8_decode<INT8, BF>(u32x2{kr[i][0], kr[i][1]}), k1 = kv8_decode<INT8, BF>(u32x2{kr[i][2], kr[i][3]});
            const f16x8 v0 = kv8_decode<INT8, false>(u32x2{vr[i][0], vr[i][1]}), v1 = kv8_decode<INT8, false>(u32x2{vr[i][2], vr[i][3]});
            *reinterpret_cast<f16x8 *>(base + c0) = odd ? k1 : k0;
            *reinterpret_cast<f16x8 *>(base + c1) = odd ? k0 : k1;
            *reinterpret_cast<f16x8 *>(base + TILE + c0) = odd ? v1 : v0;
            *reinterpret_cast<f16x8 *>(base + TILE + c1) = odd ? v0 : v1;
        }
    };
    TileReader<HD> rd;
    rd.init(lane);
    f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = zero16();
    float m = -INFINITY, l = 0.f, vref = 0.f;
    if (n_tiles > 0) {
        load(0);
        store(0);
        now[0] = next[0];
        now[1] = next[1];
        if (n_tiles > 1) load(1);
        __syncthreads();
    }
    for (int t = 0; t < n_tiles; ++t) {
        const int p0 = s0 + t * kKcKeys;
        const char *ks = smem + (t & 1) * STAGE, *vs = ks + TILE;
        const bool some = p0 <= any_last && p0 + kKcKeys > any_first;  // (of the wave)
        f32x16 s[2];
        if (some) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[h] = mfma16<BF>(rd.a_operand(ks, 32 * h, 0), qB[0], zero16());
#pragma unroll
                for (int g = 1; g < HD / 16; ++g) s[h] = mfma16<BF>(rd.a_operand(ks, 32 * h, g), qB[g], s[h]);
            }
        }
        const Half cur[2] = {now[0], now[1]};
        if (t + 1 < n_tiles) {
            store((t + 1) & 1);
            now[0] = next[0];
            now[1] = next[1];
            if (t + 2 < n_tiles) load(t + 2);
        }
        if (some) {
            // V's scale over a reference of the workgroup's, as a power of P; where it is not finite, it reaches the scores
            // of its keys as NaN.
            float lift[2], sv0[2], sk[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sv0[h] = cur[h].v * 0.f;
                sk[h] = cur[h].k * cscale;
                const float sv = sv0[h] == 0.f ? cur[h].v : 0.f;
                if (sv > vref) {
                    const float f = vref / (4.f * sv);  // room for scales that grow a little
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[dt][r] *= f;
                    vref = 4.f * sv;
                }
                lift[h] = sv > 0.f ? sv : 0.f;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) lift[h] = fmaxf(log2_fast(lift[h] / fmaxf(vref, kKv8MinScale)), -64.f) + kKcLift;
            const bool cut = p0 < all_first || p0 + kKcKeys - 1 > all_last;
            float top = -INFINITY;
            if (cut) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int key = p0 + 32 * h + acc_lrow(r, hh);
                        const float x = fmaf(s[h][r], sk[h], sv0[h]);
                        s[h][r] = key < first || key > last || key >= s1 ? -INFINITY : x;
                    }
                sk[0] = sk[1] = 1.f;
                sv0[0] = sv0[1] = 0.f;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = max3(s[h][0], s[h][1], s[h][2]);
#pragma unroll
                for (int r = 3; r < 15; r += 2) x = max3(x, s[h][r], s[h][r + 1]);
                x = max3(x, s[h][15], x);
                top = fmaxf(top, cut ? x : x * sk[h]);
            }
            if (__builtin_amdgcn_ballot_w64(top > m + kKcRaise) != 0) {
                const float m_new = fmaxf(m, max2_xor32(top));
                const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m - m_new);
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
                m = m_new;
            }
            const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float d = lift[h] - m_use + sv0[h];
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[h][r] = exp2_fast(fmaf(s[h][r], sk[h], d));
                    sum += s[h][r];
                }
                l = fmaf(sum, exp2_fast(-lift[h]), l);
#pragma unroll
                for (int gg = 0; gg < 2; ++gg) {
                    const f16x8 p = pack8(s[h], 8 * gg);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt] = mfma16<false>(rd.tr_operand(vs, 32 * h + 16 * gg, dt), p, o[dt]);
                }
            }
        }
        __syncthreads();
    }

    // P's lift and the reference of V's scales leave O.
    const float out_scale = vref * exp2_fast(-kKcLift);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= out_scale;
    l = sum_xor32(l);
    if (sl.n_pieces > 1) {
        // Partial results lane by lane: (maximum, sum) of every row, then register pairs of O by wave and lane.
        const int64_t part = int64_t(slot_i) * HI + hi_i;
        auto ml_at = [&](int i) { return kv8_ml(a, plan, part + int64_t(i - sl.ch) * HI) + wave * 32 + col; };
        auto o_at = [&](int i, int j) { return kv8_o<HD>(a, plan, part + int64_t(i - sl.ch) * HI) + (wave * (HD / 4) + j) * 64 + lane; };
        if (hh == 0) kv8_put(ml_at(sl.ch), f32x2{m, l});
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; r += 2) kv8_put(o_at(sl.ch, dt * 8 + r / 2), f32x2{o[dt][r], o[dt][r + 1]});
        int32_t *count = static_cast<int32_t *>(a.ws) + int64_t(sl.b) * HI + hi_i;
        if (!kv8_count(count, sl.n_pieces, &ticket)) return;
        m = -INFINITY;
        for (int i = 0; i < sl.n_pieces; ++i) m = fmaxf(m, kv8_get(ml_at(i))[0]);
        l = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = zero16();
        for (int i = 0; i < sl.n_pieces; ++i) {
            const f32x2 ml = kv8_get(ml_at(i));
            const float f = ml[0] == -INFINITY ? 0.f : exp2_fast(ml[0] - m);
            l = fmaf(ml[1], f, l);
            f32x2 y[DT * 8];
#pragma unroll
            for (int j = 0; j < DT * 8; ++j) y[j] = kv8_get(o_at(i, j));
#pragma unroll
            for (int j = 0; j < DT * 8; ++j) {
                o[j / 8][j % 8 * 2] = fmaf(f, y[j][0], o[j / 8][j % 8 * 2]);
                o[j / 8][j % 8 * 2 + 1] = fmaf(f, y[j][1], o[j / 8][j % 8 * 2 + 1]);
            }
        }
    }
    if (!row_ok) return;
    // A sum of 0 is that of a row without a visible key (or with scores of -infinity alone); NaN goes on to the output.
    const float inv = l == 0.f ? 0.f : 1.f / l;
    f16 *out = (f16 *)a.o.ptr + int64_t(sl.b) * a.o.batch_stride + int64_t(qpos) * a.o.row_stride + int64_t(hq) * a.o.head_stride + 4 * hh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            f16x4 y = pack4<BF>(o[dt][r] * inv, o[dt][r + 1] * inv, o[dt][r + 2] * inv, o[dt][r + 3] * inv);
            if (l == 0.f) y = pack4<BF>(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<f16x4 *>(out + 32 * dt + 2 * r) = y;
        }
    if (hh == 0) a.lse[(int64_t(sl.b) * a.nheads + hq) * a.seqlen_q + qpos] = l == 0.f ? 0.f : (m + log2_fast(l)) * kLn2;
}

int kv8_chunk(const fa_kv8_args &a, const Kv8Plan &plan, hipStream_t s) {
    const unsigned grid = unsigned(plan.slots) * unsigned(a.cache.nheads_k * plan.row_tiles);
    return kv8_by_type(a.cache.head_dim, a.dtype, a.cache.kind, [&](auto hd, auto bf, auto int8) {
        hipLaunchKernelGGL((kv8_chunk_kernel<decltype(hd)::value, decltype(bf)::value, decltype(int8)::value>), dim3(grid),
                           dim3(kKcThreads), 0, s, a, plan);
        return int(hipGetLastError());
    });
}

}  // namespace fa
