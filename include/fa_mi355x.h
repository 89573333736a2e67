/*
 * fa_mi355x.h - C ABI of the MI355X (gfx950) FlashAttention kernels.
 *
 * This is the boundary between the host layer (the `flash_attn_turing`
 * PyTorch extension, or any FFI: ctypes, cgo, JNI) and the hand-written HIP
 * kernels in libfa_mi355x.so.  Every entry point takes plain device pointers,
 * sizes and strides (in elements, 64-bit), never allocates, launches on the
 * given HIP stream (a `hipStream_t` passed as `void *`, NULL = default
 * stream) and returns FA_OK or an error code (see fa_error_string).
 *
 * Tensor convention (reference: flash_attention_interface.py:457-462, 530-539;
 * flash_api.cpp:188-256): q/o [batch][seqlen][heads][head_dim] fp16 with the
 * last dimension contiguous; k/v [batch][seqlen_k][heads_k][head_dim].  For
 * packed varlen tensors ([total][heads][head_dim]) batch_stride is ignored and
 * the row offset of batch b is cu_seqlens[b].  LSE is fp32
 * [batch][heads][lse_seqlen].  head_dim is 64 or 128 (flash_api.cpp:10-14).
 * Rows, heads and the base pointer must be 16-byte aligned (strides multiple
 * of 8 elements).
 */
#ifndef FA_MI355X_H
#define FA_MI355X_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    FA_OK = 0,
    FA_ERR_INVALID_ARG = -1,   /* shape / pointer / alignment check failed   */
    FA_ERR_UNSUPPORTED = -2,   /* head_dim not in {64, 128} and similar      */
    FA_ERR_WORKSPACE = -3,     /* missing or too small workspace             */
    FA_ERR_SCRATCH = -4        /* request beyond fa_fwd_kvcache_noalloc's static scratch */
    /* positive values are hipError_t codes from the launch                  */
};

/* A strided fp16 tensor [batch][row][head][head_dim]; strides in elements. */
typedef struct fa_tensor {
    void *ptr;
    int64_t batch_stride;
    int64_t row_stride;
    int64_t head_stride;
} fa_tensor;

/*
 * Forward attention.  Replaces the reference's run_mha_fwd(Flash_fwd_params&)
 * (flash_api.cpp:174-179, params from set_params_fprop :39-106) used by
 * mha_fwd (:188-256), mha_varlen_fwd (:353-416) and the KV-cache chunk path
 * (:686-714).
 */
typedef struct fa_fwd_args {
    fa_tensor q, k, v, o;           /* fp16; o is written for every valid row   */
    float *lse;                     /* fp32 [batch][nheads][lse_seqlen]          */
    const int32_t *cu_seqlens_q;    /* [batch+1] or NULL (dense)                 */
    const int32_t *cu_seqlens_k;    /* [batch+1] or NULL (dense)                 */
    const int32_t *seqused_k;       /* [batch] keys used per batch, or NULL      */
    const int32_t *k_batch_idx;     /* [batch] k/v batch read by q batch b, or NULL */
    int32_t seqused_k_add;          /* added to seqused_k[b] (appended tokens)   */
    int32_t batch, seqlen_q, seqlen_k, nheads, nheads_k, head_dim;
    int32_t lse_seqlen;             /* seqlen_q, or max_seqlen_q for varlen      */
    float softmax_scale;
    int32_t causal;                 /* bottom-right aligned (mask.h:52)          */
    /* KV-cache chunk checks, done on the device (no host read; replaces the
     * reference's host-side checks flash_api.cpp:627, 634-641): with seqused_k,
     * a batch whose key count is negative or above seqlen_k, or whose
     * k_batch_idx is outside [0, k_batch), is given no keys (O = 0, LSE = 0)
     * and, when status is set, ORs 1 (capacity) or 2 (cache row) into *status. */
    int32_t k_batch;                /* batches of k/v bounding k_batch_idx, 0 = unchecked */
    int32_t *status;                /* device int32 error word, or NULL          */
    /* Optional workspace for varlen calls (cu_seqlens_q set), fa_fwd_order_len(args)
     * int32s: fa_fwd then first lists the (sequence, query block) work items on
     * the device, most work first, and launches the workgroups in that order;
     * NULL keeps the natural order.  Results are the same either way. */
    int32_t *work_order;
    /* Optional workspace of split_ws_bytes >= fa_fwd_split_bytes(args) bytes,
     * 256-byte aligned (else FA_ERR_INVALID_ARG), when that is not 0: the grid of query blocks is too small
     * for the chip, and several workgroups then share each block's keys and sum
     * their fp32 partial results in it.  NULL (or a smaller one): one each. */
    void *split_ws;
    int64_t split_ws_bytes;
    /* Rows of the packed o tensor (varlen calls), or 0.  When set, o's rows that no
     * sequence covers (before cu_seqlens_q[0], from cu_seqlens_q[batch] on, and past
     * lse_seqlen within a sequence) are zeroed on the device; 0 leaves them as they are. */
    int32_t o_rows;
} fa_fwd_args;

/* Length in int32s of fa_fwd's work_order workspace: batch * ceil(lse_seqlen / 32).
 * No counterpart in the reference (its grid is in natural order). */
size_t fa_fwd_order_len(const fa_fwd_args *args);
/* Bytes of fa_fwd's split_ws workspace, 0 when the grid fills the chip by itself and
 * for varlen calls.  It depends on the sizes, head counts, head_dim, causal and the
 * current device's CU count alone.  No counterpart in the reference. */
size_t fa_fwd_split_bytes(const fa_fwd_args *args);
int fa_fwd(const fa_fwd_args *args, void *stream);

/*
 * Backward attention.  Replaces run_mha_bwd(Flash_bwd_params&) (flash_api.cpp:181-186)
 * and run_flash_bwd's three launches (flash_bwd_launch_template.h:69-146), plus
 * the GQA dK/dV reduction done with torch::sum_out (flash_api.cpp:338-348,
 * 493-503): dk/dv are written per KV head, the group is summed in-kernel.
 */
typedef struct fa_bwd_args {
    fa_tensor q, k, v, o, dout;     /* fp16 inputs                               */
    fa_tensor dq, dk, dv;           /* fp16 outputs, every valid row written     */
    const float *lse;               /* fp32 [batch][nheads][lse_seqlen]          */
    float *dsum;                    /* workspace fp32 [2][batch][nheads][lse_seqlen]: -rowsum(dO*O),
                                       then LSE*log2(e) (written by fa_bwd_dq / fa_bwd_preprocess) */
    const int32_t *cu_seqlens_q;
    const int32_t *cu_seqlens_k;
    int32_t batch, seqlen_q, seqlen_k, nheads, nheads_k, head_dim;
    int32_t lse_seqlen;
    float softmax_scale;
    int32_t causal;
    /* Optional workspace for varlen calls, fa_bwd_order_len(args) int32s:
     * fa_bwd_dkdv (cu_seqlens_k set) first lists the (sequence, key block)
     * work items on the device, most query rows first, and launches the dK/dV
     * workgroups in that order, and fa_bwd_dq (cu_seqlens_q set) does the same
     * for its (sequence, query block) items, most keys first, in the second
     * part of the workspace; NULL keeps the natural order, which is longest
     * first only when every sequence has the same length.  Results are the same
     * either way (each item is computed independently). */
    int32_t *work_order;
    /* Optional workspace of split_ws_bytes >= fa_bwd_split_bytes(args) bytes,
     * 256-byte aligned (else FA_ERR_INVALID_ARG), when that is not 0: the grid of dK/dV key blocks is too
     * small for the chip, and several workgroups then share each key block's
     * queries and sum their fp32 partial dK / dV in it.  Only dK/dV reads it, and
     * every call clears its counters itself, whatever ran before.
     * NULL (or a smaller one) gives each key block to one workgroup. */
    void *split_ws;
    int64_t split_ws_bytes;
    /* Rows of the packed dq and of the packed dk / dv, or 0, as fa_fwd_args.o_rows:
     * fa_bwd_dq zeroes dq's rows of no sequence (and past lse_seqlen within one),
     * fa_bwd_dkdv those of dk and dv (past seqlen_k). */
    int32_t dq_rows, dkv_rows;
} fa_bwd_args;

/* Length in int32s of the work_order workspace: batch * (ceil(seqlen_k / 128) +
 * ceil(lse_seqlen / 32)).  No counterpart in the reference (its grids are in
 * natural order). */
size_t fa_bwd_order_len(const fa_bwd_args *args);
/* Bytes of the split_ws workspace, 0 when the dK/dV grid fills the chip by
 * itself.  It depends on the sizes, head counts, head_dim, causal and the current
 * device's CU count alone.  No counterpart in the reference. */
size_t fa_bwd_split_bytes(const fa_bwd_args *args);
/* D = rowsum(dO * O) (flash_bwd_preprocess_kernel.h:23-96), stored negated in dsum plane 0. */
int fa_bwd_preprocess(const fa_bwd_args *args, void *stream);
/* dQ kernel (flash_bwd_kernel.h:25-609); computes and stores the dsum workspace itself. */
int fa_bwd_dq(const fa_bwd_args *args, void *stream);
/* dK/dV kernel with in-kernel GQA accumulation (flash_bwd_kernel.h:613-1344); reads the
 * dsum workspace written by fa_bwd_dq or fa_bwd_preprocess. */
int fa_bwd_dkdv(const fa_bwd_args *args, void *stream);
/* dQ (with the dsum workspace) then dK/dV, in stream order. */
int fa_bwd(const fa_bwd_args *args, void *stream);

/*
 * KV-cache attention.  Replaces run_kvcache_paged_append (kvcache_native.cu:956-993),
 * the contiguous append loop (flash_api.cpp:643-654) and run_mha_fwd_kvcache_native
 * (kvcache_native.cu:995-1218) called from mha_fwd_kvcache (flash_api.cpp:508-715).
 * Attention runs over L_b = cache_seqlens[b] + seqlen_new keys.
 */
typedef struct fa_kvcache_args {
    fa_tensor q;                    /* [batch][seqlen_q][nheads][head_dim]       */
    fa_tensor k_cache, v_cache;     /* contiguous [batch_cache][capacity][nheads_k][d]
                                       or paged [num_blocks][page_block_size][nheads_k][d] */
    fa_tensor k_new, v_new;         /* [batch][seqlen_new][nheads_k][d]; ptr NULL = no append */
    fa_tensor o;                    /* [batch][seqlen_q][nheads][head_dim]       */
    float *lse;                     /* [batch][nheads][seqlen_q]                 */
    const int32_t *cache_seqlens;   /* [batch] tokens in the cache before append */
    const int32_t *cache_batch_idx; /* [batch] cache row of batch b, or NULL     */
    const int32_t *block_table;     /* [batch][block_table_stride], or NULL      */
    int64_t block_table_stride;
    int32_t batch, seqlen_q, nheads, nheads_k, head_dim;
    int32_t seqlen_new;             /* tokens appended per sequence (0 = none)   */
    int32_t page_block_size;        /* paged: multiple of 256; contiguous: 0     */
    int32_t num_splits;             /* >= 1, as resolved by fa_kv_num_splits     */
    float softmax_scale;
    int32_t causal;
    float *out_accum;               /* workspace [num_splits][batch*nheads*seqlen_q][d] fp32, 8-byte aligned */
    float *lse_accum;               /* workspace [num_splits][batch*nheads*seqlen_q] fp32    */
    int32_t *batch_order;           /* workspace [batch + 1]: sequences longest first and a work
                                       counter (filled by fa_kv_splitkv or fa_fwd_kvcache where
                                       the call has more items than the device has CUs, else
                                       left as they are), or NULL for the natural order        */
    /* Device-side input checks (replace the host reads of flash_api.cpp:627,
     * 634-641 and interface.py:855, so a decode step needs no host sync): a
     * sequence with cache_seqlens[b] < 0, cache_seqlens[b] + seqlen_new >
     * cache_capacity, or cache_batch_idx[b] outside [0, cache_batch) is not
     * appended to and is attended over no keys (O = 0, LSE = 0); with status
     * set, 1 (capacity) or 2 (cache row) is ORed into *status.  0 = unchecked. */
    int32_t cache_capacity;         /* tokens one sequence's cache holds (paged: pages * page size) */
    int32_t cache_batch;            /* rows of a contiguous cache (bounds cache_batch_idx); paged: pages of the
                                       cache (a table entry in use outside them reads page 0, is not appended to
                                       and ORs FA_KV_BAD_PAGE into *status), or 0: the table is not checked */
    int32_t *status;                /* device int32 error word, or NULL                            */
    /* Upstream FlashAttention options the reference's signature takes but rejects
     * (flash_attention_interface.py:617-634), with upstream's semantics: query i
     * (at key position p = i + L - seqlen_q) sees keys [p - window_left, p + window_right]
     * (a negative bound is unbounded; causal also caps the right side at p), and
     * softcap > 0 replaces the scaled score x by softcap * tanh(x / softcap),
     * ALiBi adds -slope[h] * |p - j| to the score of key j, and key j < cache_leftpad[b]
     * does not exist for sequence b (positions unchanged).  Zero-initialised, all are off. */
    int32_t local_window;           /* 1: apply window_left / window_right; 0: no window */
    int32_t window_left, window_right;
    float softcap;                  /* > 0: softcapping on                                          */
    const int32_t *cache_leftpad;   /* [batch] first valid key of each sequence, or NULL            */
    const float *alibi_slopes;      /* fp32 [nheads] (batch stride 0) or [batch][nheads], or NULL   */
    int64_t alibi_batch_stride;
    /* Rotary embedding on append (upstream FlashAttention's, also rejected by the
     * reference): with rotary_dim > 0 (a multiple of 16, at most head_dim; k_new
     * required), channels [0, rotary_dim) of appended key t of sequence b are
     * rotated at position cache_seqlens[b] + t before the store, and those of
     * query row i at cache_seqlens[b] + i when causal or local_window, else at
     * cache_seqlens[b]; position p's angles are row p of rotary_cos / rotary_sin
     * (fp16 [rotary_seqlen][rotary_dim / 2], contiguous, 16-byte aligned; a
     * position past the last row takes the last row).  Interleaved rotates
     * channel pairs (2j, 2j + 1) by angle j, otherwise (j, j + rotary_dim / 2). */
    const void *rotary_cos, *rotary_sin;
    int32_t rotary_dim;             /* 0: no rotary embedding                                       */
    int32_t rotary_seqlen;
    int32_t rotary_interleaved;
    /* Workspace of fa_kv_split_count_len(args) int32s, or NULL.  With it, batch_order
     * and num_splits > 1, the split kernel combines the partials itself: the last of
     * the num_splits items of each (batch, kv head, row tile) to finish reads them
     * and writes o and lse, so fa_kv_combine has nothing left to do (it returns at
     * once) and fa_fwd_kvcache runs two kernels (append with ordering, split) instead
     * of four.  Every call zeroes these counts itself. */
    int32_t *split_count;
} fa_kvcache_args;

/* Split count for a request (kvcache_native.cu:913-952 choose_num_splits);
 * requested > 0 is returned unchanged.  fa_kv_args_num_splits takes the call itself
 * (sizes, options, cache_capacity; num_splits and the workspaces are not read, and
 * batch_order and split_count are taken to be given), fa_kv_num_splits only the sizes
 * of a call without options, and where many rows per KV head ask for more splits than
 * fa_fwd_kvcache_noalloc's scratch holds it returns as many as fit.
 * fa_kv_args_num_splits has no counterpart in the reference. */
int fa_kv_args_num_splits(const fa_kvcache_args *args, int requested, int num_cus);
int fa_kv_num_splits(int requested, int seqlen_k_capacity, int head_dim, int seqlen_q,
                     int batch, int nheads, int nheads_k, int num_cus);
/* Bytes of the split accumulators for args->num_splits (0 when num_splits == 1);
 * batch_order, when used, needs (batch + 1) * 4 more. */
size_t fa_kv_workspace_bytes(const fa_kvcache_args *args);
/* int32s of the split_count workspace: batch * nheads_k * ceil(nheads / nheads_k *
 * seqlen_q / 32) when num_splits > 1, else 0. */
size_t fa_kv_split_count_len(const fa_kvcache_args *args);
/* In-place append of k_new/v_new at cache_seqlens (contiguous, remapped or paged). */
int fa_kv_append(const fa_kvcache_args *args, void *stream);
/* Split-KV partial attention; writes o/lse directly when num_splits == 1, or with
 * batch_order and split_count. */
int fa_kv_splitkv(const fa_kvcache_args *args, void *stream);
/* Log-sum-exp combine of the split partials into o/lse (kvcache_native.cu:676-729);
 * nothing to do when fa_kv_splitkv combined them (batch_order and split_count set). */
int fa_kv_combine(const fa_kvcache_args *args, void *stream);
/* append + split-KV + combine in stream order (with batch_order the append and the
 * ordering share one launch). */
int fa_fwd_kvcache(const fa_kvcache_args *args, void *stream);

/*
 * Allocation-free variant of fa_fwd_kvcache.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, serving loops, harnesses that forbid hipMalloc).  The
 * same kernels run; out_accum, lse_accum, batch_order and split_count in args
 * are ignored and taken instead from a static device array of
 * FA_NOALLOC_SCRATCH_BYTES per device, held until the process ends (the calling
 * thread's current device must be the stream's).  A request needing more than
 * that, i.e. fa_kv_workspace_bytes(args) + 4 * (batch + 1 +
 * fa_kv_split_count_len(args)) bytes, returns FA_ERR_SCRATCH.
 * No allocation or free happens in the call.  Calls on one device share its
 * array: calls that overlap on one device (on different streams) race, and
 * their results are undefined.  (No kernel waits for a word in memory, so the
 * kernels end all the same.)
 */
#define FA_NOALLOC_SCRATCH_BYTES (16u << 20)
int fa_fwd_kvcache_noalloc(const fa_kvcache_args *args, void *stream);

/*
 * Differential attention.  A head's q and k hold two maps in the two halves of
 * their head_dim channels (map 1 the first half, map 2 the second), v has
 * head_dim channels:
 *   o = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v.
 * All tensors are laid out as those of fa_fwd / fa_bwd, with row strides of 0 to
 * 2^23 elements (o, o2 and the gradients: any); dtype is FA_FP16 or FA_BF16 for
 * all of them.  No counterpart in the reference.
 */
enum { FA_FP16 = 0, FA_BF16 = 1, FA_FP32 = 2 /* rotary tables alone */ };

/* lam, fp32: element [batch b][row i][head h] at ptr + b * batch_stride + i *
 * row_stride + h * head_stride (strides in elements, 0 where it is shared; for
 * packed tensors the row counts from the first packed row and batch_stride is 0). */
typedef struct fa_diff_lam {
    const float *ptr;
    int64_t batch_stride, row_stride, head_stride;
} fa_diff_lam;

typedef struct fa_diff_fwd_args {
    fa_tensor q, k, v, o;
    fa_tensor o2;                   /* map 2's own output softmax(S2) v, which the backward reads, or ptr NULL */
    fa_diff_lam lam;
    float *lse;                     /* fp32 [2][batch][nheads][lse_seqlen], map 1's first */
    const int32_t *cu_seqlens_q;    /* [batch+1], both or neither                */
    const int32_t *cu_seqlens_k;
    int32_t batch, seqlen_q, seqlen_k, nheads, nheads_k, head_dim;
    int32_t lse_seqlen;             /* seqlen_q, or max_seqlen_q for packed batches */
    float softmax_scale;
    int32_t causal;                 /* bottom-right aligned                      */
    int32_t dtype;
    int32_t o_rows;                 /* rows of the packed q and o, as fa_fwd_args.o_rows */
    int32_t k_rows;                 /* rows of the packed k and v, or 0; a packed sequence is cut to these
                                       rows and to seqlen_q / seqlen_k, whatever cu_seqlens hold */
    int32_t *work_order;            /* fa_diff_fwd_order_len(args) int32s for packed batches, or NULL */
} fa_diff_fwd_args;

size_t fa_diff_fwd_order_len(const fa_diff_fwd_args *args);
int fa_diff_fwd(const fa_diff_fwd_args *args, void *stream);

/* dlam as fa_diff_lam, written. */
typedef struct fa_diff_dlam {
    float *ptr;
    int64_t batch_stride, row_stride, head_stride;
} fa_diff_dlam;

typedef struct fa_diff_bwd_args {
    fa_tensor q, k, v, o, o2, dout; /* inputs; o and o2 as the forward wrote them */
    fa_tensor dq, dk, dv;           /* outputs, every row of a sequence written   */
    fa_diff_lam lam;
    fa_diff_dlam dlam;              /* gradient of lam, or ptr NULL: row_stride not 0 gives every row
                                       its own (each row of a sequence written); else the sum over all rows, of each
                                       head (head_stride not 0) or of all of them (one value) */
    const float *lse;               /* as the forward wrote it                    */
    const int32_t *cu_seqlens_q, *cu_seqlens_k;
    int32_t batch, seqlen_q, seqlen_k, nheads, nheads_k, head_dim, lse_seqlen;
    float softmax_scale;
    int32_t causal, dtype;
    int32_t dq_rows, dkv_rows;      /* as o_rows and k_rows, and as in fa_bwd_args */
    int32_t *work_order;            /* fa_diff_bwd_order_len(args) int32s for packed batches, or NULL */
    float *dsum;                    /* workspace of dsum_bytes >= fa_diff_bwd_ws_bytes(args), 32-byte aligned */
    int64_t dsum_bytes;
    void *split_ws;                 /* fa_diff_bwd_split_bytes(args) bytes, 256-byte aligned, as fa_bwd_args.split_ws, or NULL */
    int64_t split_ws_bytes;
} fa_diff_bwd_args;

size_t fa_diff_bwd_ws_bytes(const fa_diff_bwd_args *args);
size_t fa_diff_bwd_split_bytes(const fa_diff_bwd_args *args);
size_t fa_diff_bwd_order_len(const fa_diff_bwd_args *args);
int fa_diff_bwd(const fa_diff_bwd_args *args, void *stream);

/*
 * Differential attention over a key-value cache, laid out and checked on the
 * device as in fa_kvcache_args: k_new / v_new are appended at cache_seqlens,
 * then seqlen_q queries attend over L = cache_seqlens + seqlen_new keys.  With
 * seqlen_q 0 the append alone runs (q, o, lam and lse may be NULL).
 */
typedef struct fa_diff_kvcache_args {
    fa_tensor q, k_cache, v_cache, k_new, v_new, o;
    fa_diff_lam lam;                /* [batch][seqlen_q][nheads] by its strides   */
    float *lse;                     /* fp32 [2][batch][nheads][seqlen_q]          */
    const int32_t *cache_seqlens;   /* [batch] tokens before the append           */
    const int32_t *cache_batch_idx; /* [batch] or NULL (contiguous caches)        */
    const int32_t *block_table;     /* [batch][block_table_stride] or NULL        */
    int64_t block_table_stride;
    int32_t batch, seqlen_q, nheads, nheads_k, head_dim, seqlen_new;
    int32_t page_block_size;        /* paged: a multiple of 64                    */
    int32_t num_pages;              /* paged: pages of the cache; a table entry in use outside them reads page
                                       0, is not appended to and ORs FA_KV_BAD_PAGE into *status */
    int32_t num_splits;             /* pieces of cache_capacity, 0: chosen (calls of few query rows) */
    float softmax_scale;
    int32_t causal, dtype;
    int32_t cache_capacity;         /* tokens one sequence's cache holds          */
    int32_t cache_batch;            /* rows of a contiguous cache                 */
    int32_t *status;                /* device word: 1 (capacity) or 2 (cache row) is ORed in, or NULL */
    void *ws;                       /* fa_diff_kvcache_ws_bytes(args) bytes, 256-byte aligned */
    int64_t ws_bytes;
} fa_diff_kvcache_args;

size_t fa_diff_kvcache_ws_bytes(const fa_diff_kvcache_args *args);
int fa_diff_kvcache(const fa_diff_kvcache_args *args, void *stream);

/*
 * Pages of a paged key-value cache.  page_refs[p] is the number of block_table
 * entries that name page p (0: free); a table entry of -1 names none.  All arrays
 * are on the device, nothing is read on the host, and what is wrong is ORed into
 * *status (a call that gives out pages then changes nothing).  No counterpart in
 * the reference.
 */
enum {
    FA_KV_BAD_PAGE = 4,  /* a block_table entry in use names no page of the cache */
    FA_KV_NO_PAGES = 8,  /* fewer free pages than the call needs                   */
    FA_KV_BAD_LIST = 16  /* a list's row or page is out of range, taken or named twice */
};

typedef struct fa_kvpages_args {
    fa_tensor k_cache, v_cache;     /* [num_pages][page_block_size][nheads_k][head_bytes], strides in BYTES, multiples of 16 */
    int32_t nheads_k, head_bytes;
    int32_t page_block_size, num_pages;
    int32_t *block_table;           /* [rows][max_pages]                          */
    int64_t block_table_stride;
    int32_t rows, max_pages;
    int32_t *cache_seqlens;         /* [rows] tokens in the cache                 */
    int32_t *page_refs;             /* [num_pages]                                */
    const int32_t *from, *to;       /* [n]: pages (copy), parents and children (fork), rows (free: from) */
    int32_t n;
    int32_t seqlen_new;             /* alloc: tokens that every row makes room for ... */
    const int32_t *seqlens_new;     /* ... or [rows], or NULL                     */
    int32_t *out_table;             /* compact: [rows][max_pages], apart from block_table */
    int64_t out_table_stride;
    int32_t *out_refs, *out_used;   /* compact: [num_pages], apart from page_refs; [1] pages in use */
    int32_t *status;                /* device int32 error word, or NULL           */
    void *ws;                       /* fa_kvpages_ws_bytes(args) bytes (not for copy and free) */
    int64_t ws_bytes;
} fa_kvpages_args;

size_t fa_kvpages_ws_bytes(const fa_kvpages_args *args);
/* Rows get pages for tokens [cache_seqlens, cache_seqlens + new), lowest free pages first, in row order. */
int fa_kvpages_alloc(const fa_kvpages_args *args, void *stream);
/* Page to[i] = page from[i], all at once; pairs that touch each other's pages are not copied (FA_KV_BAD_LIST). */
int fa_kvpages_copy(const fa_kvpages_args *args, void *stream);
/* Row to[i] (empty) shares the full pages of row from[i] and gets a page with a copy of the tokens of a last, partly
 * filled one.  (This and compact move one pair of pools: not the codes of a cache in 8 bits, whose scales would stay.) */
int fa_kvpages_fork(const fa_kvpages_args *args, void *stream);
/* Rows from[i] give their pages back and become empty. */
int fa_kvpages_free(const fa_kvpages_args *args, void *stream);
/* The used pages move to the front of the pool: out_table and out_refs are the table and the counts afterwards. */
int fa_kvpages_compact(const fa_kvpages_args *args, void *stream);

/*
 * Rotary positions: cosines and sines of angles, and q and k rotated by them.  A pair
 * (x1, x2) of channels of a row at position p becomes (x1 c - x2 s, x2 c + x1 s), in
 * fp32 and rounded once.  fa_kvcache_args has the same rotation for fp16 caches; here it is
 * for training (inverse is the gradient), packed batches, bf16 and tables of 32 bits.
 * No counterpart in the reference.
 */
#define FA_ROTARY_MAX_DIM 256
/* Positions of the tables: up to here, to either side, angles in 64 bits are right to half a step of fp32 (2^-25). */
#define FA_ROTARY_MAX_POSITION (1 << 26)

/* cos and sin, [seqlen][rotary_dim / 2] of dtype: entry (i, j) is attention_factor times the
 * cosine / sine of (offset + i) * f_j, computed in 64 bits, f_j = base ^ (-2 j / rotary_dim).
 * factor != 1 divides the frequencies: all of them (original_seqlen 0), or, by the turns t that
 * a pair makes in original_seqlen tokens, f_j (keep + (1 - keep) / factor) with
 * keep = (t - low_turns) / (high_turns - low_turns) cut to [0, 1].  All positions lie within
 * FA_ROTARY_MAX_POSITION of 0. */
typedef struct fa_rotary_tables_args {
    void *cos, *sin;                /* 16-byte aligned                           */
    int32_t seqlen, rotary_dim;     /* rotary_dim: a multiple of 16 up to FA_ROTARY_MAX_DIM */
    int32_t dtype;                  /* FA_FP16, FA_BF16 or FA_FP32               */
    int64_t offset;
    double base, factor, original_seqlen, low_turns, high_turns, attention_factor;
} fa_rotary_tables_args;

int fa_rotary_tables(const fa_rotary_tables_args *args, void *stream);

/* q and k (ptr NULL: none) to q_out and k_out, apart from them.  Row i of sequence b is at position
 * positions[b * positions_stride + i], or else offset + seqlen_offsets[b] + i; packed (cu_seqlens): i
 * counts from the sequence's first row, and rows of no sequence become 0.  A row whose
 * position is outside the tables gets NaN in the rotated channels. */
typedef struct fa_rotary_args {
    fa_tensor q, k, q_out, k_out;   /* fp16 or bf16                              */
    const void *cos, *sin;          /* [table_rows][rotary_dim / 2], 16-byte aligned rows */
    int64_t cos_stride, sin_stride; /* between their rows, elements              */
    const int32_t *positions;       /* [batch][seqlen], packed [seqlen], or NULL */
    int64_t positions_stride;
    const int32_t *seqlen_offsets;  /* [batch] or NULL                           */
    const int32_t *cu_seqlens;      /* [batch + 1]: packed, or NULL              */
    int32_t batch, seqlen;          /* seqlen: rows a sequence, or all packed rows */
    int32_t nheads, nheads_k, head_dim, rotary_dim, table_rows;
    int32_t offset;
    int32_t interleaved;            /* pairs (2j, 2j + 1), else (j, j + rotary_dim / 2) */
    int32_t inverse;                /* rotates back: the gradient of q and k from those of q_out and k_out */
    int32_t dtype, table_dtype;
} fa_rotary_args;

int fa_rotary(const fa_rotary_args *args, void *stream);

/*
 * A key-value cache in 8 bits: codes of one byte and one fp32 scale for each block of
 * scale_block tokens of a head; a value is code * scale.  fa_kv8_append quantises k_new and v_new
 * as it writes them at cache_seqlens: a block's scale becomes the smallest power of two s >= 2^-126
 * with max|x| <= most * s over the block's new values (most: 448 for e4m3, 127 for int8), or
 * the old scale where the block holds earlier tokens and that is larger, and codes are x / s rounded to
 * nearest even; earlier tokens' codes are rounded again where the scale grows.  A NaN or an
 * infinity among the new values makes the scale NaN, and so every value of the block.
 * Attention takes any finite codes and scales >= 0; rows that see a block with a scale that is NaN or infinite become
 * NaN.  Lengths, rows and pages are checked on the device as in
 * fa_diff_kvcache_args.  No counterpart in the reference.
 */
enum { FA_KV8_E4M3 = 0, FA_KV8_INT8 = 1 };

/* Scale of (page or cache row, block of tokens, head) at ptr + row * batch_stride + block *
 * row_stride + head * head_stride (strides in elements). */
typedef struct fa_kv8_scales {
    float *ptr;
    int64_t batch_stride, row_stride, head_stride;
} fa_kv8_scales;

typedef struct fa_kv8_cache {
    fa_tensor k, v;                 /* codes [pages or rows][tokens][nheads_k][head_dim], strides multiples of 16 bytes, tokens at most 2^23 apart */
    fa_kv8_scales k_scale, v_scale; /* [pages or rows][tokens / scale_block][nheads_k] */
    const int32_t *cache_batch_idx; /* [batch] or NULL (contiguous caches)        */
    const int32_t *block_table;     /* [batch][block_table_stride] or NULL        */
    int64_t block_table_stride;
    int32_t batch, nheads_k, head_dim;
    int32_t scale_block;            /* 32, 64, 128 or 256; divides the tokens of a page or row */
    int32_t kind;                   /* FA_KV8_E4M3 or FA_KV8_INT8                 */
    int32_t page_block_size, num_pages;
    int32_t cache_capacity;         /* tokens one sequence's cache holds          */
    int32_t cache_batch;            /* rows of a contiguous cache                 */
    int32_t *status;                /* device error word, or NULL                 */
} fa_kv8_cache;

typedef struct fa_kv8_args {
    fa_kv8_cache cache;
    fa_tensor k_new, v_new;         /* [batch][seqlen_new][nheads_k][head_dim] of dtype */
    const int32_t *cache_seqlens;   /* [batch] tokens before the append           */
    const int32_t *seqlens_new;     /* [batch] new tokens of each sequence, 0 to seqlen_new, or NULL: all of them (fa_kv8_append alone) */
    int32_t seqlen_new;
    int32_t dtype;                  /* FA_FP16 or FA_BF16: q, o, k_new and v_new  */
    /* Attention alone. */
    fa_tensor q, o;                 /* [batch][seqlen_q][nheads][head_dim]        */
    float *lse;                     /* fp32 [batch][nheads][seqlen_q]             */
    int32_t seqlen_q, nheads;
    int32_t causal;                 /* bottom-right aligned                       */
    int32_t window_left, window_right; /* keys that a query sees to either side of its own position, -1: all */
    int32_t num_splits;             /* pieces of cache_capacity, 0: chosen        */
    float softmax_scale;
    void *ws;                       /* fa_kv8_ws_bytes(args) bytes, 256-byte aligned */
    int64_t ws_bytes;
} fa_kv8_args;

int fa_kv8_append(const fa_kv8_args *args, void *stream);
size_t fa_kv8_ws_bytes(const fa_kv8_args *args);
/* The append (seqlen_new > 0), then seqlen_q queries over cache_seqlens + seqlen_new keys. */
int fa_kv8_attention(const fa_kv8_args *args, void *stream);

/* The first cu_seqlens[b + 1] - cu_seqlens[b] tokens of each sequence b as values of dtype, in rows cu_seqlens[b]
 * and on of k_out and v_out; rows that no sequence covers, and those of a sequence that is longer than the cache's
 * capacity, become 0. */
typedef struct fa_kv8_read_args {
    fa_kv8_cache cache;
    fa_tensor k_out, v_out;         /* packed [total][nheads_k][head_dim]         */
    const int32_t *cu_seqlens;      /* [batch + 1]                                */
    int32_t total, dtype;
} fa_kv8_read_args;

int fa_kv8_read(const fa_kv8_read_args *args, void *stream);

/* Human-readable text for a return code (FA_* or hipError_t). */
const char *fa_error_string(int code);

/*
 * Version of the argument-struct layouts above.  It changes whenever a struct
 * gains, loses or moves a field (4: fa_bwd_args.split_ws and split_ws_bytes
 * appended; 5: the same for fa_fwd_args; 6:
 * fa_fwd_args.o_rows, fa_bwd_args.dq_rows and dkv_rows).  A caller compiled against this
 * header checks fa_abi_version() == FA_ABI_VERSION once after loading the
 * library and refuses a mismatch: the entry points themselves cannot tell a
 * shorter struct from an older caller.  No counterpart in the reference (its
 * bindings are compiled together with its kernels).
 */
#define FA_ABI_VERSION 6
int fa_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* FA_MI355X_H */
