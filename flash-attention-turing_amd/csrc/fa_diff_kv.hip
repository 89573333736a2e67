// Differential attention over a key-value cache: append, and few query rows
// (decode steps, drafted tokens) split over the cache's length.
//
// What bounds it is reading K and V once: 4 * head_dim bytes a token and KV
// head.  The rows of a KV head are its query heads times the query positions;
// a tile of 16 of them fills the 32 columns of one MFMA with both maps: column
// c < 16 is row c's map 1, whose query operand is 0 on map 2's channels,
// column 16 + c its map 2.  So the scores of both maps take the products of one
// whole K row, and both products with V are one; the waste is in MFMA slots, which
// wait for memory here.
//
// A workgroup takes one chunk of the keys of one (sequence, KV head, row tile);
// chunks have the same length for all sequences, so the items are of equal work
// whatever the lengths.  That length follows from num_splits and the capacity, and
// a row's sum does not depend on the rest of the batch; with num_splits 0 it is
// chosen by the batch's items too (diff_kv_chunk).  A workgroup's four waves walk
// 32-key tiles (tile t to wave t % 4), each through LDS slots of its own: operands
// go to registers, the next copy into the same slot goes out, then the tile is
// computed, with no barrier in the loop.  The waves merge through LDS.  Of a
// sequence's chunks, the workgroup that counts last adds all partial results in
// the order of the chunks; none waits.
//
// Measured (32/8 heads of 128): 64 sequences of 1 k to 16 k tokens, paged, bf16,
// one query each: 307 us for 1.73 GB, 5.6 TB/s (a large copy reaches 4.7); one
// sequence of 1500 tokens, where the chain of latencies counts (arguments, length,
// tiles, partial results, counter, join): 11 us, 3 more for the append.  Both in
// tables no wider than the longest sequence.  The host knows the capacity only, not
// the lengths, so a wider table means longer chunks and fewer of them: the one
// sequence in a table of 131072 tokens 25 us a call against 15, eight of 8000 tokens
// 69 against 59, the 64 sequences 300 against 299.
#include <algorithm>

#include "fa_diff_common.h"

namespace fa {

constexpr int kDkThreads = 256, kDkTile = 32, kDkRows = 16;

// g2l16 (fa_common.h) for bytes that are read once (one row tile): the caches are
// asked not to keep them, and so evict nothing for them.  64 sequences of 1 k to
// 16 k tokens, 32/8 heads of 128: 335 -> 305 us.  After other work has filled the
// 256 MB memory-side cache: 404 -> 327, 32 x 500 to 5000 tokens 128 -> 81, 16 x 500
// to 12000 120 -> 79 us; the last one repeated with nothing between, so that its
// 240 MB stay there, 54 -> 67 us.
__device__ __forceinline__ void g2l16_once(const void *g, char *lds_base) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off nt\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(g), "s"(__builtin_amdgcn_readfirstlane(lds_addr(lds_base)))
        : "memory");
}

// A wave's copy of kDkTile rows of K or V, swizzled as TileReader reads them; rows past last_row re-read it.
template <int HD, bool ONCE>
__device__ __forceinline__ void diff_kv_tile(char *tile, const f16 *src, int64_t rs, int last_row, int lane) {
    constexpr int KCH = HD / 8;
#pragma unroll
    for (int i = 0; i < kDkTile * KCH / 64; ++i) {
        const int p = i * 64 + lane, row = p / KCH, c = p % KCH;
        const f16 *g = src + min(row, last_row) * rs + 8 * (c ^ swz<KCH>(row));
        if constexpr (ONCE)
            g2l16_once(g, tile + i * 1024);
        else
            g2l16(g, tile + i * 1024);
    }
}

__device__ __forceinline__ int diff_kv_err(const fa_diff_kvcache_args &a, int b, int &L0, int &row) {
    L0 = a.cache_seqlens[b];
    row = a.cache_batch_idx ? a.cache_batch_idx[b] : b;
    const int err = (L0 < 0 || int64_t(L0) + a.seqlen_new > a.cache_capacity ? 1 : 0) |
                    (a.cache_batch_idx && (row < 0 || row >= a.cache_batch) ? 2 : 0);
    if (err) L0 = row = 0;
    return err;
}

// Append (one 16-byte chunk of K and of V a thread) after clear_wgs workgroups
// that clear the split counters.
__global__ __launch_bounds__(256) void diff_kv_prep_kernel(const fa_diff_kvcache_args a, int32_t *const count,
                                                           const int n_count, const int clear_wgs) {
    if (int(blockIdx.x) < clear_wgs) {
        const int i = blockIdx.x * 256 + threadIdx.x;
        if (i < n_count) count[i] = 0;
        return;
    }
    const int kch = a.head_dim / 8;
    const int64_t idx = int64_t(blockIdx.x - clear_wgs) * 256 + threadIdx.x;
    if (idx >= int64_t(a.batch) * a.seqlen_new * a.nheads_k * kch) return;
    const int c = int(idx % kch);
    int64_t rest = idx / kch;
    const int hk = int(rest % a.nheads_k);
    rest /= a.nheads_k;
    const int t = int(rest % a.seqlen_new), b = int(rest / a.seqlen_new);
    int L0, row;
    const int err = diff_kv_err(a, b, L0, row);
    if (err) {
        if (a.status && t == 0 && hk == 0 && c == 0) atomicOr(a.status, err);
        return;
    }
    int pos = L0 + t;
    int64_t line = row;
    if (a.block_table) {
        const int pg = pos / a.page_block_size;
        line = a.block_table[int64_t(b) * a.block_table_stride + pg];
        pos -= pg * a.page_block_size;
        if (line < 0 || line >= a.num_pages) {
            if (a.status && hk == 0 && c == 0) atomicOr(a.status, FA_KV_BAD_PAGE);
            return;
        }
    }
    auto src = [&](const fa_tensor &x) {
        return (const f16 *)x.ptr + int64_t(b) * x.batch_stride + int64_t(t) * x.row_stride + int64_t(hk) * x.head_stride;
    };
    auto dst = [&](const fa_tensor &x) {
        return (f16 *)x.ptr + line * x.batch_stride + int64_t(pos) * x.row_stride + int64_t(hk) * x.head_stride;
    };
    *reinterpret_cast<u32x4 *>(dst(a.k_cache) + 8 * c) = ldg16(src(a.k_new) + 8 * c);
    *reinterpret_cast<u32x4 *>(dst(a.v_cache) + 8 * c) = ldg16(src(a.v_new) + 8 * c);
}

// Workspace of a call in n_chunks chunks: the counters of the (sequence, KV
// head, row tile) items, then (256-byte aligned) each chunk's (maximum, sum) of
// 2 R columns and its 2 R x head_dim unnormalised fp32 O, R the rows of a tile.
__host__ __device__ __forceinline__ int diff_kv_rows(const fa_diff_kvcache_args &a) {
    const int rows = a.nheads / a.nheads_k * a.seqlen_q;
    return rows < kDkRows ? rows : kDkRows;
}
__host__ __device__ __forceinline__ int64_t diff_kv_items(const fa_diff_kvcache_args &a) {
    const int64_t rows = int64_t(a.nheads / a.nheads_k) * a.seqlen_q;
    return a.batch * int64_t(a.nheads_k) * ((rows + kDkRows - 1) / kDkRows);
}
__host__ __device__ __forceinline__ int64_t diff_kv_count_bytes(int64_t items) { return (items * 4 + 255) & ~int64_t(255); }

template <int HD, bool BF>
__global__ __launch_bounds__(kDkThreads, 2) void diff_kv_kernel(const fa_diff_kvcache_args a, const int row_tiles,
                                                                const int chunk, const int n_chunks) {
    constexpr int KCH = HD / 8, TILE = kDkTile * HD * 2, STAGE = 2 * TILE;
    constexpr int NST = HD == 64 ? 2 : 1;          // tiles in flight per wave
    constexpr int CPW = kDkTile * KCH / 64;        // copies a lane for K or V of a tile
    constexpr int MERGE = 33;                      // row stride of the waves' O^T at the merge
    constexpr int WAVE_LDS = NST * STAGE > HD * MERGE * 4 ? NST * STAGE : HD * MERGE * 4;
    constexpr int HG = HD / 32;
    static_assert(WAVE_LDS % 512 == 0, "tile bases must be multiples of 512 bytes");
    __shared__ __attribute__((aligned(16))) char smem[4 * WAVE_LDS];
    __shared__ f32x2 ml[4][32];
    __shared__ int ticket;

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rt = blockIdx.x % row_tiles;
    int rest = blockIdx.x / row_tiles;
    const int hk = rest % a.nheads_k;
    rest /= a.nheads_k;
    const int b = rest % a.batch, ch = rest / a.batch;
    const int G = a.nheads / a.nheads_k, R = G * a.seqlen_q;  // row = query position * G + head of the group
    int L0, cache_row;
    const int err = diff_kv_err(a, b, L0, cache_row);
    if (err && a.status && ch == 0 && tid == 0) atomicOr(a.status, err);
    const int L = err ? 0 : L0 + a.seqlen_new;
    const int live_chunks = max(1, (L + chunk - 1) / chunk);  // an empty sequence has one empty chunk
    if (ch >= live_chunks) return;
    const int s0 = ch * chunk, s1 = min(L, s0 + chunk);

    const int map = col >> 4, row = rt * kDkRows + (col & 15);
    const bool row_ok = row < R;
    const int qpos = row_ok ? row / G : 0, hq = hk * G + (row_ok ? row - qpos * G : 0);
    const int lim = a.causal ? qpos + L - a.seqlen_q : L - 1;                     // last visible key
    const int lim_min = a.causal ? (rt * kDkRows) / G + L - a.seqlen_q : L - 1;  // ... of the tile's first row
    const float cscale = fabsf(a.softmax_scale) * kLog2e;
    f32x16 o[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) o[i] = zero16();
    float m = -INFINITY, l = 0.f;

    const int t_first = s0 / kDkTile, t_end = (s1 + kDkTile - 1) / kDkTile;
    const int my_first = t_first + wave;
    const int n_my = my_first < t_end ? (t_end - my_first + 3) / 4 : 0;
    const int64_t krs = a.k_cache.row_stride, vrs = a.v_cache.row_stride;
    char *const slot = smem + wave * WAVE_LDS;
    // Copies of tile t into the wave's slot st (keys past L re-read key L - 1; masked).
    auto issue = [&](int t, int st) FA_INLINE {
        const int p0 = t * kDkTile;
        int64_t line = cache_row;
        int at = p0;
        if (a.block_table) {
            const int pg = p0 / a.page_block_size;
            line = checked_page(scalar_load(a.block_table + int64_t(b) * a.block_table_stride + pg), a.num_pages, a.status);
            at = p0 - pg * a.page_block_size;
        }
        const f16 *kb = (const f16 *)a.k_cache.ptr + line * a.k_cache.batch_stride + int64_t(at) * krs +
                        int64_t(hk) * a.k_cache.head_stride;
        const f16 *vb = (const f16 *)a.v_cache.ptr + line * a.v_cache.batch_stride + int64_t(at) * vrs +
                        int64_t(hk) * a.v_cache.head_stride;
        char *const ks = slot + st * STAGE;
        if (row_tiles == 1) {
            diff_kv_tile<HD, true>(ks, kb, krs, L - 1 - p0, lane);
            diff_kv_tile<HD, true>(ks + TILE, vb, vrs, L - 1 - p0, lane);
        } else {
            diff_kv_tile<HD, false>(ks, kb, krs, L - 1 - p0, lane);
            diff_kv_tile<HD, false>(ks + TILE, vb, vrs, L - 1 - p0, lane);
        }
    };
    TileReader<HD> rd;
    rd.init(lane);
    if (n_my > 0) issue(my_first, 0);
    if (NST > 1 && n_my > 1) issue(my_first + 4, 1);
    // Q^T as B operands, behind the first copies: the two latencies run together.
    f16x8 qB[HD / 16];
    {
        const f16 *qp = (const f16 *)a.q.ptr + int64_t(b) * a.q.batch_stride + int64_t(qpos) * a.q.row_stride +
                        int64_t(hq) * a.q.head_stride + 8 * hh;
#pragma unroll
        for (int g = 0; g < HD / 16; ++g) {
            u32x4 v = row_ok && g / HG == map ? ldg16(qp + 16 * g) : zero_u4();
            if (a.softmax_scale < 0.f) v = neg_h8(v);
            qB[g] = as_h8(v);
        }
    }
    wait_vmem();  // only tile copies are in flight inside the loop
    for (int k = 0; k < n_my; ++k) {
        const int st = k % NST, p0 = (my_first + 4 * k) * kDkTile;
        if (k + 1 < n_my)
            wait_vmem_n<(NST - 1) * 2 * CPW>();  // the newer tile may stay in flight
        else
            wait_vmem();
        const char *ks = slot + st * STAGE, *vs = ks + TILE;
        f16x8 ka[HD / 16], va[HD / 32][2];
#pragma unroll
        for (int g = 0; g < HD / 16; ++g) ka[g] = rd.a_operand(ks, 0, g);
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
            for (int gg = 0; gg < 2; ++gg) va[dt][gg] = rd.tr_operand(vs, 16 * gg, dt);
        wait_lds();
        if (k + NST < n_my) issue(my_first + 4 * (k + NST), st);
        // Each map's channels apart, of which a column takes its own map's: a key's infinity or NaN in the other
        // map's channels, times the query operand's 0, would be NaN.
        f32x16 s = mfma16<BF>(ka[0], qB[0], zero16()), s2 = mfma16<BF>(ka[HG], qB[HG], zero16());
#pragma unroll
        for (int g = 1; g < HG; ++g) {
            s = mfma16<BF>(ka[g], qB[g], s);
            s2 = mfma16<BF>(ka[HG + g], qB[HG + g], s2);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = map ? s2[r] : s[r];
        if (p0 + kDkTile > s1 || p0 + kDkTile - 1 > lim_min) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = p0 + acc_lrow(r, hh);
                if (key >= s1 || key > lim) s[r] = -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = max_xor32(mx);
        const float mx_t = mx == -INFINITY ? -INFINITY : mx * cscale;
        if (__builtin_amdgcn_ballot_w64(mx_t > m) != 0) {
            const float m_new = fmaxf(m, mx_t);
            const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m - m_new);
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
            m = m_new;
        }
        const float m_use = m == -INFINITY ? 0.f : m;
        float rs = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float x = s[r];
            const float e = x == -INFINITY ? 0.f : exp2_fast(fmaf(x, cscale, -m_use));
            s[r] = e;
            rs += e;
        }
        l += rs;
        // P keeps 32 bits through the product, as hi + lo in the tensors' type: the matrix cores wait for memory here
        // (64 sequences of 1 k to 16 k tokens, bf16: 306.5 -> 307.3 us, and 1.4 times a plain form's error -> the same;
        // one of 1500: 13.4 -> 13.6; four of 4096, 4 queries each, fp16: 31 -> 33).
#pragma unroll
        for (int gg = 0; gg < 2; ++gg) {
            const f16x8 hi = pack16<BF>(s, 8 * gg);
            f32x16 rest;
#pragma unroll
            for (int u = 0; u < 8; ++u) rest[u] = s[8 * gg + u] - elem<BF>(hi, u);
            const f16x8 lo = pack16<BF>(rest, 0);
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt) {
                o[dt] = mfma16<BF>(va[dt][gg], hi, o[dt]);
                o[dt] = mfma16<BF>(va[dt][gg], lo, o[dt]);
            }
        }
    }

    // Merge the four waves: O^T to LDS, then every thread sums elements of (column, channel).
    l = sum_xor32(l);
    float *ow = reinterpret_cast<float *>(slot);
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) ow[(dt * 32 + acc_row(r, hh)) * MERGE + col] = o[dt][r];
    if (hh == 0) ml[wave][col] = f32x2{m, l};
    __syncthreads();

    const int rows = min(kDkRows, R - rt * kDkRows), R16 = diff_kv_rows(a);
    // Column c's merged maximum, sum and unnormalised O at channels d, d + 1.
    auto merged = [&](int c, int d, float &mm, float &ll) FA_INLINE {
        mm = fmaxf(fmaxf(ml[0][c][0], ml[1][c][0]), fmaxf(ml[2][c][0], ml[3][c][0]));
        ll = 0.f;
        f32x2 x = {0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ml[w][c][0] == -INFINITY ? 0.f : exp2_fast(ml[w][c][0] - mm);
            const float *ow = reinterpret_cast<const float *>(smem + w * WAVE_LDS);
            ll = fmaf(ml[w][c][1], f, ll);
            x[0] = fmaf(ow[d * MERGE + c], f, x[0]);
            x[1] = fmaf(ow[(d + 1) * MERGE + c], f, x[1]);
        }
        return x;
    };
    auto store = [&](int r, int d, f32x2 x1, float m1, float l1, f32x2 x2, float m2, float l2) FA_INLINE {
        const int row = rt * kDkRows + r, qp = row / G, h = hk * G + row - qp * G;
        const float lam = diff_lam(a.lam, b, qp, h);
        // A sum of 0 is that of a map without a visible key (or with scores of -infinity alone); one that is NaN goes
        // on to the outputs.
        const float i1 = l1 == 0.f ? 0.f : 1.f / l1, i2 = l2 == 0.f ? 0.f : lam / l2;
        f16 *out = (f16 *)a.o.ptr + int64_t(b) * a.o.batch_stride + int64_t(qp) * a.o.row_stride +
                   int64_t(h) * a.o.head_stride + d;
        const f16x4 y = l1 == 0.f && l2 == 0.f
                            ? pack4<BF>(0.f, 0.f, 0.f, 0.f)
                            : pack4<BF>(x1[0] * i1 - x2[0] * i2, x1[1] * i1 - x2[1] * i2, 0.f, 0.f);
        *reinterpret_cast<uint32_t *>(out) = __builtin_bit_cast(u32x2, y)[0];
        if (d == 0) {
            float *lse = a.lse + (int64_t(b) * a.nheads + h) * a.seqlen_q + qp;
            lse[0] = l1 == 0.f ? 0.f : (m1 + log2_fast(l1)) * kLn2;
            lse[int64_t(a.batch) * a.nheads * a.seqlen_q] = l2 == 0.f ? 0.f : (m2 + log2_fast(l2)) * kLn2;
        }
    };
    if (live_chunks == 1) {
        for (int e = tid; e < rows * (HD / 2); e += kDkThreads) {
            const int r = e / (HD / 2), d = 2 * (e % (HD / 2));
            float m1, l1, m2, l2;
            const f32x2 x1 = merged(r, d, m1, l1), x2 = merged(16 + r, d, m2, l2);
            store(r, d, x1, m1, l1, x2, m2, l2);
        }
        return;
    }
    // Partial results: 2 R16 columns of (maximum, sum), then of HD / 2 pairs, for each (item, chunk).
    const int64_t item = (int64_t(b) * a.nheads_k + hk) * row_tiles + rt, items = diff_kv_items(a);
    int32_t *count = static_cast<int32_t *>(a.ws) + item;
    uint64_t *mls = reinterpret_cast<uint64_t *>(static_cast<char *>(a.ws) + diff_kv_count_bytes(items));
    uint64_t *os = mls + items * n_chunks * 2 * R16;
    mls += item * n_chunks * 2 * R16;
    os += item * n_chunks * 2 * R16 * (HD / 2);
    for (int e = tid; e < 2 * rows * (HD / 2); e += kDkThreads) {
        const int c = e / (HD / 2), d2 = e % (HD / 2);
        float mm, ll;
        const f32x2 x = merged(c < rows ? c : 16 + c - rows, 2 * d2, mm, ll);
        __hip_atomic_store(os + (int64_t(ch) * 2 * R16 + c) * (HD / 2) + d2, __builtin_bit_cast(uint64_t, x),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d2 == 0)
            __hip_atomic_store(mls + ch * 2 * R16 + c, __builtin_bit_cast(uint64_t, f32x2{mm, ll}), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
    }
    wait_vmem();
    __syncthreads();  // every wave's stores have completed
    if (tid == 0) ticket = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (ticket != live_chunks - 1) return;

    // The last chunk's workgroup: wave w takes rows w, w + 4, .., a lane two channels.
    auto load = [](const uint64_t *p) FA_INLINE {
        return __builtin_bit_cast(f32x2, __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    };
    const int d2 = lane % (HD / 2);
    for (int r = wave; r < rows; r += 4) {
        // Lane i holds chunk i's maxima and sums; both maps' loads, and eight chunks', are in flight together.
        float mm[2] = {-INFINITY, -INFINITY}, ll[2] = {0.f, 0.f};
        f32x2 x[2] = {}, own[2];
        for (int i0 = 0; i0 < live_chunks; i0 += 64)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f32x2 y = load(mls + min(i0 + lane, live_chunks - 1) * 2 * R16 + k * rows + r);
                if (i0 == 0) own[k] = y;
                mm[k] = fmaxf(mm[k], y[0]);
            }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1)
#pragma unroll
            for (int k = 0; k < 2; ++k) mm[k] = fmaxf(mm[k], __shfl_xor(mm[k], d));
        for (int i0 = 0; i0 < live_chunks; i0 += 64) {
            const int n = min(64, live_chunks - i0);
            float f[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (i0 > 0) own[k] = load(mls + (i0 + min(lane, n - 1)) * 2 * R16 + k * rows + r);
                f[k] = lane < n && own[k][0] != -INFINITY ? exp2_fast(own[k][0] - mm[k]) : 0.f;
                ll[k] = fmaf(own[k][1], f[k], ll[k]);
            }
            for (int i = 0; i < n; i += 8) {
                f32x2 y[8][2];
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        y[j][k] = i + j < n ? load(os + (int64_t(i0 + i + j) * 2 * R16 + k * rows + r) * (HD / 2) + d2)
                                            : f32x2{0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f[k]), i + j));
                        x[k][0] = fmaf(w, y[j][k][0], x[k][0]);
                        x[k][1] = fmaf(w, y[j][k][1], x[k][1]);
                    }
            }
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1)
#pragma unroll
            for (int k = 0; k < 2; ++k) ll[k] += __shfl_xor(ll[k], d);
        if (lane < HD / 2) store(r, 2 * d2, x[0], mm[0], ll[0], x[1], mm[1], ll[1]);
    }
}

// Whether the forward kernel takes the call: more rows than one tile (with one,
// this kernel reads the cache once, which nothing beats), and less time by these
// estimates in us, the tokens counted as the capacity.  This kernel: its launches
// and the join, and the chip's rate of 32-key tiles.  The forward kernel: one
// workgroup's walk over the keys, longer with a second one on its CU.
// Measured (128 channels, 4 heads a KV head, bf16; this kernel, the forward one):
//   1 x 1000 tokens, 8 KV heads,  32 / 64 / 128 rows   20 / 20 / 25      27 / 27 / 29 us
//   1 x 8192                                           37 / 43 / 59      150 / 151 / 152
//   16 x 4096                                          99 / 178 / 335    94 / 96 / 97
static bool diff_kv_many_rows(const fa_diff_kvcache_args &a) {
    const int G = a.nheads / a.nheads_k;
    if (int64_t(G) * a.seqlen_q <= kDkRows) return false;
    const int heads = G % 2 == 0 ? 2 : 1, P = 64 / heads;  // of a forward workgroup of 64 rows
    const double cus = device_cus(), cap = a.cache_capacity;
    const double w = double(a.batch) * (a.nheads / heads) * ((a.seqlen_q + P - 1) / P) / cus;
    return 8 + cap / 64 * std::max(1 + 0.5 * w, w) < 15 + cap * double(diff_kv_items(a)) / (50 * cus);
}

// Keys of a chunk, a multiple of the 128 that four waves take at a time.  Chunks of
// one sequence are equal: as many as find room on the chip at once.  With more
// sequences, whose lengths differ, half as many again, so that the rounds fill.
// Under 256 keys a chunk's start and the join cost more than its keys.  Measured
// (decode, 32/8 heads of 128 channels; 2 or 3 chunks per CU, us): 1 x 32 k
// tokens 38 and 46; 32 sequences of 500 to 5000 78 and 66; at least 128, 256 or 512
// keys: 1 x 8192 30, 21 and 20.5, 1 x 1500 13.2, 13.2 and 15.4.
static int diff_kv_chunk(const fa_diff_kvcache_args &a) {
    const int64_t cap = std::max(a.cache_capacity, 1), items = diff_kv_items(a);
    int64_t chunk;
    if (a.num_splits > 0)
        chunk = (cap + a.num_splits - 1) / a.num_splits;
    else
        chunk = std::min<int64_t>(std::max<int64_t>(cap * items / ((a.batch == 1 ? 2 : 3) * device_cus()), 256), 4096);
    return int((chunk + 127) / 128 * 128);
}

int diff_fwd_cache(const fa_diff_kvcache_args &a, hipStream_t s);  // fa_diff_fwd.hip

static int check_diff_kv(const fa_diff_kvcache_args *p) {
    if (!p) return FA_ERR_INVALID_ARG;
    const fa_diff_kvcache_args &a = *p;
    if (a.head_dim != 64 && a.head_dim != 128) return FA_ERR_UNSUPPORTED;
    if (a.dtype != FA_FP16 && a.dtype != FA_BF16) return FA_ERR_UNSUPPORTED;
    if (a.batch < 0 || a.seqlen_q < 0 || a.seqlen_new < 0 || a.nheads <= 0 || a.nheads_k <= 0 ||
        a.nheads % a.nheads_k != 0 || a.num_splits < 0 || a.cache_capacity < 0)
        return FA_ERR_INVALID_ARG;
    if (a.batch == 0) return FA_OK;  // tensors of no sequences have no address
    const bool queries = a.seqlen_q > 0;  // none: an append alone
    if (!a.cache_seqlens || (queries && (!a.lse || !a.lam.ptr))) return FA_ERR_INVALID_ARG;
    if (a.block_table && (a.cache_batch_idx || a.page_block_size <= 0 || a.page_block_size % 64 != 0 || a.num_pages <= 0))
        return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.q, &a.o})
        if (check_tensor(*t, queries)) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.k_cache, &a.v_cache})
        if (check_tensor(*t, true)) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.k_cache, &a.v_cache})
        if (t->row_stride < 0 || t->row_stride > kDiffMaxRowStride) return FA_ERR_INVALID_ARG;
    for (const fa_tensor *t : {&a.k_new, &a.v_new})
        if (check_tensor(*t, a.seqlen_new > 0)) return FA_ERR_INVALID_ARG;
    if (a.ws_bytes < int64_t(fa_diff_kvcache_ws_bytes(&a)) || (reinterpret_cast<uintptr_t>(a.ws) & 255u) ||
        (!a.ws && fa_diff_kvcache_ws_bytes(&a) > 0))
        return FA_ERR_WORKSPACE;
    return FA_OK;
}

template <int HD, bool BF>
static int launch_diff_kv(const fa_diff_kvcache_args &a, int chunk, int n_chunks, hipStream_t s) {
    const int64_t items = diff_kv_items(a), grid = items * n_chunks;
    if (grid > 0x7fffffff) return FA_ERR_INVALID_ARG;
    const int row_tiles = int(items / (int64_t(a.batch) * a.nheads_k));
    hipLaunchKernelGGL((diff_kv_kernel<HD, BF>), dim3(unsigned(grid)), dim3(kDkThreads), 0, s, a, row_tiles, chunk,
                       n_chunks);
    return int(hipGetLastError());
}

}  // namespace fa

extern "C" size_t fa_diff_kvcache_ws_bytes(const fa_diff_kvcache_args *a) {
    if (!a || a->batch <= 0 || a->seqlen_q <= 0 || a->nheads <= 0 || a->nheads_k <= 0 || fa::diff_kv_many_rows(*a))
        return 0;
    const int chunk = fa::diff_kv_chunk(*a);
    const int64_t n = (int64_t(std::max(a->cache_capacity, 1)) + chunk - 1) / chunk, items = fa::diff_kv_items(*a);
    if (n == 1) return 0;
    return size_t(fa::diff_kv_count_bytes(items) + items * n * 2 * fa::diff_kv_rows(*a) * (8 + 4 * int64_t(a->head_dim)));
}

extern "C" int fa_diff_kvcache(const fa_diff_kvcache_args *args, void *stream) {
    using namespace fa;
    int rc = check_diff_kv(args);
    if (rc) return rc;
    const fa_diff_kvcache_args &a = *args;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (a.batch == 0) return FA_OK;
    const bool many = diff_kv_many_rows(a);
    const int chunk = diff_kv_chunk(a);
    const int n_chunks = int((int64_t(std::max(a.cache_capacity, 1)) + chunk - 1) / chunk);
    const int64_t items = diff_kv_items(a);
    const int64_t n_count = many || a.seqlen_q == 0 || n_chunks == 1 ? 0 : items;
    const int64_t pieces = int64_t(a.batch) * a.seqlen_new * a.nheads_k * (a.head_dim / 8);
    const int64_t clear_wgs = (n_count + 255) / 256, grid = clear_wgs + (pieces + 255) / 256;
    if (grid > 0x7fffffff || items > 0x7fffffff) return FA_ERR_INVALID_ARG;
    if (grid > 0) {
        hipLaunchKernelGGL(diff_kv_prep_kernel, dim3(unsigned(grid)), dim3(256), 0, s, a, static_cast<int32_t *>(a.ws),
                           int(n_count), int(clear_wgs));
        if ((rc = int(hipGetLastError()))) return rc;
    }
    if (a.seqlen_q == 0) return FA_OK;
    if (many) return diff_fwd_cache(a, s);
    if (a.dtype == FA_BF16)
        return a.head_dim == 128 ? launch_diff_kv<128, true>(a, chunk, n_chunks, s)
                                 : launch_diff_kv<64, true>(a, chunk, n_chunks, s);
    return a.head_dim == 128 ? launch_diff_kv<128, false>(a, chunk, n_chunks, s)
                             : launch_diff_kv<64, false>(a, chunk, n_chunks, s);
}
