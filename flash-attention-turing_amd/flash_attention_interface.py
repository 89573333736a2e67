"""Python interface of the MI355X FlashAttention (drop-in for the reference's
flash_attention_interface.py).

Public API, argument order, defaults, validation order and error messages follow
the reference module (flash_attention_interface.py:448-922):

    flash_attn_func, flash_attn_qkvpacked_func, flash_attn_kvpacked_func,
    flash_attn_varlen_func, flash_attn_varlen_qkvpacked_func,
    flash_attn_varlen_kvpacked_func, flash_attn_with_kvcache

Beside them, without a counterpart in the reference: differential attention

    flash_diff_attn_func, flash_diff_attn_varlen_func, flash_diff_attn_with_kvcache

and the pages of a paged cache

    flash_attn_kvcache_alloc, flash_attn_kvcache_copy_pages, flash_attn_kvcache_fork,
    flash_attn_kvcache_free, flash_attn_kvcache_compact

and rotary positions

    flash_attn_rotary_tables, flash_attn_rotary_func

and a KV cache in 8 bits

    flash_attn_kvcache_append_q8, flash_attn_kvcache_read_q8, flash_attn_with_kvcache_q8

and the autograd classes FlashAttnFunc, FlashAttnQKVPackedFunc,
FlashAttnKVPackedFunc, FlashAttnVarlenFunc, FlashAttnVarlenQKVPackedFunc,
FlashAttnVarlenKVPackedFunc (:172-445).  Every call goes to the native
``flash_attn_turing`` extension (HIP kernels for gfx950); there is no Python
math fallback: a missing or incompatible extension raises at import or call.
"""

import math
from typing import Optional, Tuple, Union

import torch  # noqa: F401  (loads the HIP runtime before the extension)

import flash_attn_turing as flash_attn_gpu


def maybe_contiguous(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Copy only tensors whose last dimension is strided (interface.py:9-10)."""
    if x is None or x.stride(-1) == 1:
        return x
    return x.contiguous()


def _default_scale(q: torch.Tensor, softmax_scale: Optional[float]) -> float:
    # interface.py:183: head_dim ** -0.5 unless given.
    return q.shape[-1] ** (-0.5) if softmax_scale is None else softmax_scale


# ---------------------------------------------------------------------------
# Thin wrappers over the extension (interface.py:13-169).


def _flash_attn_forward(q, k, v, softmax_scale: float, causal: bool):
    q, k, v = (maybe_contiguous(t) for t in (q, k, v))
    out, lse = flash_attn_gpu.fwd(q, k, v, softmax_scale, causal)
    return out, lse


def _flash_attn_backward(dout, q, k, v, out, lse, softmax_scale: float, causal: bool, dq=None, dk=None, dv=None):
    """dq / dk / dv, when given, are written in place (e.g. slices of a packed dqkv) and returned."""
    dout, q, k, v, out, lse = (maybe_contiguous(t) for t in (dout, q, k, v, out, lse))
    dq, dk, dv = flash_attn_gpu.bwd(q, k, v, out, lse, dout, softmax_scale, causal, dq, dk, dv)
    return dq, dk, dv


def _flash_attn_varlen_forward(
    q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float, causal: bool
):
    q, k, v = (maybe_contiguous(t) for t in (q, k, v))
    out, lse = flash_attn_gpu.varlen_fwd(
        q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal
    )
    return out, lse


def _flash_attn_varlen_backward(
    dout,
    q,
    k,
    v,
    out,
    lse,
    cu_seqlens_q,
    cu_seqlens_k,
    max_seqlen_q: int,
    max_seqlen_k: int,
    softmax_scale: float,
    causal: bool,
    dq=None,
    dk=None,
    dv=None,
    zero_rest: bool = False,
):
    """dq / dk / dv, when given, are written in place (rows no sequence covers are left as they are, or
    zeroed with zero_rest)."""
    dout, q, k, v, out, lse = (maybe_contiguous(t) for t in (dout, q, k, v, out, lse))
    dq, dk, dv = flash_attn_gpu.varlen_bwd(
        q, k, v, out, lse, dout, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
        dq, dk, dv, zero_rest,
    )
    return dq, dk, dv


def _flash_attn_kvcache_forward(
    q, k_cache, v_cache, k, v, cache_seqlens, cache_batch_idx, block_table, softmax_scale: float, causal: bool,
    num_splits: int, status: Optional[torch.Tensor] = None, window_size: Tuple[int, int] = (-1, -1),
    softcap: float = 0.0, cache_leftpad: Optional[torch.Tensor] = None, alibi_slopes: Optional[torch.Tensor] = None,
    rotary_cos: Optional[torch.Tensor] = None, rotary_sin: Optional[torch.Tensor] = None,
    rotary_interleaved: bool = True, lengths_checked: bool = False,
):
    tensors = (q, k_cache, v_cache, k, v, cache_seqlens, cache_batch_idx, block_table, cache_leftpad, alibi_slopes)
    q, k_cache, v_cache, k, v, cache_seqlens, cache_batch_idx, block_table, cache_leftpad, alibi_slopes = (
        maybe_contiguous(t) for t in tensors
    )
    # The 20-argument binding of flash_api.cpp:508-528; a preallocated out is
    # passed as "absent".
    out, lse = flash_attn_gpu.fwd_kvcache(
        q, k_cache, v_cache, k, v, cache_seqlens,
        rotary_cos, rotary_sin,
        cache_batch_idx,
        cache_leftpad,
        block_table,
        alibi_slopes,
        None,                  # out
        softmax_scale, causal,
        int(window_size[0]), int(window_size[1]),
        float(softcap),
        bool(rotary_interleaved),
        num_splits,
        status,                # device-side input checks instead of host reads, when given
        lengths_checked,       # cache_seqlens already read and checked against the capacity
    )
    return out, lse


# ---------------------------------------------------------------------------
# Autograd functions (interface.py:172-445).


class FlashAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, softmax_scale, causal, is_grad_enabled):
        softmax_scale = _default_scale(q, softmax_scale)
        out, lse = _flash_attn_forward(q, k, v, softmax_scale, causal)
        if is_grad_enabled and (q.requires_grad or k.requires_grad or v.requires_grad):
            ctx.save_for_backward(q, k, v, out, lse)
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = _flash_attn_backward(dout, q, k, v, out, lse, ctx.softmax_scale, ctx.causal)
        return dq, dk, dv, None, None, None


# Packed inputs: the kernels take row and head strides, so q / k / v are
# passed as views of the packed tensor (no copies, unlike the reference's
# interface.py:208-212, 244-247), and the backward writes the gradient slices
# straight into one packed gradient (no torch.stack, interface.py:226-231).


def _unpack(packed: torch.Tensor, dim: int, n: int):
    return tuple(packed.select(dim=dim, index=i) for i in range(n))


def _packed_grad(packed, dim: int, zero: bool):
    """A gradient for a packed input (shape, dtype, device) and its slices along dim."""
    shape, dtype, device = packed
    g = (torch.zeros if zero else torch.empty)(shape, dtype=dtype, device=device)
    return g, tuple(g.select(dim=dim, index=i) for i in range(shape[dim]))


class FlashAttnQKVPackedFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, softmax_scale, causal, is_grad_enabled):
        q, k, v = _unpack(qkv, 2, 3)
        softmax_scale = _default_scale(q, softmax_scale)
        out, lse = _flash_attn_forward(q, k, v, softmax_scale, causal)
        if is_grad_enabled and qkv.requires_grad:
            ctx.save_for_backward(q, k, v, out, lse)
            ctx.packed = (qkv.shape, qkv.dtype, qkv.device)
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dqkv, (dq, dk, dv) = _packed_grad(ctx.packed, 2, False)
        _flash_attn_backward(dout, q, k, v, out, lse, ctx.softmax_scale, ctx.causal, dq, dk, dv)
        return dqkv, None, None, None


class FlashAttnKVPackedFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, kv, softmax_scale, causal, is_grad_enabled):
        k, v = _unpack(kv, 2, 2)
        softmax_scale = _default_scale(q, softmax_scale)
        out, lse = _flash_attn_forward(q, k, v, softmax_scale, causal)
        if is_grad_enabled and (q.requires_grad or kv.requires_grad):
            ctx.save_for_backward(q, k, v, out, lse)
            ctx.packed = (kv.shape, kv.dtype, kv.device)
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dkv, (dk, dv) = _packed_grad(ctx.packed, 2, False)
        dq, _, _ = _flash_attn_backward(dout, q, k, v, out, lse, ctx.softmax_scale, ctx.causal, None, dk, dv)
        return dq, dkv, None, None, None


class FlashAttnVarlenFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
                is_grad_enabled):
        softmax_scale = _default_scale(q, softmax_scale)
        out, lse = _flash_attn_varlen_forward(
            q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal
        )
        if is_grad_enabled and (q.requires_grad or k.requires_grad or v.requires_grad):
            ctx.save_for_backward(q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k)
            ctx.max_seqlen_q, ctx.max_seqlen_k = max_seqlen_q, max_seqlen_k
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k = ctx.saved_tensors
        dq, dk, dv = _flash_attn_varlen_backward(
            dout, q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k, ctx.max_seqlen_q, ctx.max_seqlen_k,
            ctx.softmax_scale, ctx.causal,
        )
        return dq, dk, dv, None, None, None, None, None, None, None


class FlashAttnVarlenQKVPackedFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, cu_seqlens, max_seqlen, softmax_scale, causal, is_grad_enabled):
        q, k, v = _unpack(qkv, 1, 3)
        softmax_scale = _default_scale(q, softmax_scale)
        out, lse = _flash_attn_varlen_forward(
            q, k, v, cu_seqlens, cu_seqlens, max_seqlen, max_seqlen, softmax_scale, causal
        )
        if is_grad_enabled and qkv.requires_grad:
            ctx.save_for_backward(q, k, v, out, lse, cu_seqlens)
            ctx.packed = (qkv.shape, qkv.dtype, qkv.device)
            ctx.max_seqlen = max_seqlen
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, cu_seqlens = ctx.saved_tensors
        dqkv, (dq, dk, dv) = _packed_grad(ctx.packed, 1, False)
        _flash_attn_varlen_backward(
            dout, q, k, v, out, lse, cu_seqlens, cu_seqlens, ctx.max_seqlen, ctx.max_seqlen,
            ctx.softmax_scale, ctx.causal, dq, dk, dv, zero_rest=True,
        )
        return dqkv, None, None, None, None, None


class FlashAttnVarlenKVPackedFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, kv, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
                is_grad_enabled):
        k, v = _unpack(kv, 1, 2)
        softmax_scale = _default_scale(q, softmax_scale)
        out, lse = _flash_attn_varlen_forward(
            q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal
        )
        if is_grad_enabled and (q.requires_grad or kv.requires_grad):
            ctx.save_for_backward(q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k)
            ctx.packed = (kv.shape, kv.dtype, kv.device)
            ctx.max_seqlen_q, ctx.max_seqlen_k = max_seqlen_q, max_seqlen_k
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k = ctx.saved_tensors
        dkv, (dk, dv) = _packed_grad(ctx.packed, 1, False)
        dq, _, _ = _flash_attn_varlen_backward(
            dout, q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k, ctx.max_seqlen_q, ctx.max_seqlen_k,
            ctx.softmax_scale, ctx.causal, None, dk, dv, zero_rest=True,
        )
        return dq, dkv, None, None, None, None, None, None, None


# ---------------------------------------------------------------------------
# Public functions (interface.py:448-614).


def flash_attn_func(q, k, v, softmax_scale: Optional[float] = None, causal: bool = False) -> torch.Tensor:
    """q (batch, seqlen_q, nheads, headdim); k, v (batch, seqlen_k, nheads_k, headdim).
    Returns out (batch, seqlen_q, nheads, headdim)."""
    return FlashAttnFunc.apply(q, k, v, softmax_scale, causal, torch.is_grad_enabled())


def flash_attn_qkvpacked_func(qkv, softmax_scale: Optional[float] = None, causal: bool = False) -> torch.Tensor:
    """qkv (batch, seqlen, 3, nheads, headdim).  Returns out (batch, seqlen, nheads, headdim)."""
    return FlashAttnQKVPackedFunc.apply(qkv, softmax_scale, causal, torch.is_grad_enabled())


def flash_attn_kvpacked_func(q, kv, softmax_scale: Optional[float] = None, causal: bool = False) -> torch.Tensor:
    """q (batch, seqlen_q, nheads, headdim); kv (batch, seqlen_k, 2, nheads_k, headdim)."""
    return FlashAttnKVPackedFunc.apply(q, kv, softmax_scale, causal, torch.is_grad_enabled())


def flash_attn_varlen_func(
    q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q: int, max_seqlen_k: int,
    softmax_scale: Optional[float] = None, causal: bool = False,
) -> torch.Tensor:
    """q (total_q, nheads, headdim); k, v (total_k, nheads_k, headdim); cu_seqlens_* int32
    (batch_size + 1,).  Returns out (total_q, nheads, headdim)."""
    return FlashAttnVarlenFunc.apply(
        q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
        torch.is_grad_enabled(),
    )


def flash_attn_varlen_qkvpacked_func(
    qkv, cu_seqlens, max_seqlen: int, softmax_scale: Optional[float] = None, causal: bool = False
) -> torch.Tensor:
    """qkv (total, 3, nheads, headdim); cu_seqlens int32 (batch_size + 1,)."""
    return FlashAttnVarlenQKVPackedFunc.apply(
        qkv, cu_seqlens, max_seqlen, softmax_scale, causal, torch.is_grad_enabled()
    )


def flash_attn_varlen_kvpacked_func(
    q, kv, cu_seqlens_q, cu_seqlens_k, max_seqlen_q: int, max_seqlen_k: int,
    softmax_scale: Optional[float] = None, causal: bool = False,
) -> torch.Tensor:
    """q (total_q, nheads, headdim); kv (total_k, 2, nheads_k, headdim)."""
    return FlashAttnVarlenKVPackedFunc.apply(
        q, kv, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
        torch.is_grad_enabled(),
    )


# ---------------------------------------------------------------------------
# KV cache (interface.py:617-922).


def _validate_unsupported_kvcache_args(rotary_cos, rotary_sin, cache_leftpad, window_size, softcap, alibi_slopes):
    # interface.py:617-634 rejects all five; here they are supported with
    # upstream FlashAttention's semantics, so only their types are checked.
    for name, t in (("rotary_cos", rotary_cos), ("rotary_sin", rotary_sin)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or t.dim() != 2):
            raise TypeError(f"{name} must be a 2-D torch.float16 tensor (seqlen_ro, rotary_dim / 2)")
    if len(tuple(window_size)) != 2 or not all(isinstance(w, int) for w in window_size):
        raise TypeError("window_size must be a pair of ints")
    if not math.isfinite(softcap):
        raise ValueError("softcap must be finite")
    if cache_leftpad is not None and (not isinstance(cache_leftpad, torch.Tensor) or cache_leftpad.dtype != torch.int32):
        raise TypeError("cache_leftpad must be a torch.int32 tensor")
    if alibi_slopes is not None and (not isinstance(alibi_slopes, torch.Tensor) or alibi_slopes.dtype != torch.float32):
        raise TypeError("alibi_slopes must be a torch.float32 tensor")


def _validate_supported_head_dim(head_dim: int) -> None:
    if head_dim not in (64, 128):
        raise ValueError("Turing FlashAttention supports head_dim 64 or 128")


def _cache_capacity(k_cache: torch.Tensor, block_table: Optional[torch.Tensor]) -> int:
    return k_cache.shape[1] if block_table is None else block_table.shape[1] * k_cache.shape[1]


# Status words of the synchronisation-free KV-cache mode, one int32 per device.
_KV_STATUS = {}

# Bits of a status word and the errors the synchronous checks raise for them
# (interface.py:855-857 for the capacity, flash_api.cpp:634-641 for the rows).
_KV_STATUS_ERRORS = (
    (1, ValueError, "cache capacity is insufficient for the requested append length"),
    (2, RuntimeError, "cache_batch_idx entries must be within cache batch bounds"),
    (4, RuntimeError, "block_table entries in use must be pages of the cache"),
    (8, RuntimeError, "the cache has fewer free pages than the call needs"),
    (16, ValueError, "a list of pages or rows holds one that is out of range, taken or named twice"),
)


def _raise_kv_status(bits: int) -> None:
    for bit, exc, msg in _KV_STATUS_ERRORS:
        if bits & bit:
            raise exc(msg)


def _kv_status(device: torch.device) -> torch.Tensor:
    index = torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    st = _KV_STATUS.get(index)
    if st is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(
                "flash_attn_with_kvcache(validate=False) needs its status word allocated before graph capture: "
                "call flash_attn_kvcache_check() once on this device first"
            )
        st = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
        _KV_STATUS[index] = st
    return st


def flash_attn_kvcache_check(device: Optional[Union[torch.device, int]] = None) -> None:
    """Report what earlier flash_attn_with_kvcache(validate=False) calls on a
    device found wrong, then clear it.  Entries of a block_table that are in use
    and name no page of the cache, and negative lengths beside a block_table, are
    reported here whatever validate was.

    Such calls read neither cache_seqlens nor cache_batch_idx on the host; the
    kernels check them instead.  A sequence that would overflow its cache, or
    whose cache_batch_idx is outside the cache, is left unchanged in the cache
    and gets O = 0 (LSE 0); this function then raises the error the default
    (validate=True) call raises at once: ValueError for the capacity,
    RuntimeError for the cache row.  The calls on the pages of a cache and
    flash_diff_attn_with_kvcache report here as well.  It reads the device (a synchronisation),
    so call it outside captured graphs, for instance after each replay or
    every few steps.  It also allocates the device's status word, which must
    exist before a validate=False call is captured.
    """
    st = _kv_status(torch.device("cuda", device) if isinstance(device, int) else (device or torch.device("cuda")))
    bits = int(st.item())
    if bits:
        st.zero_()
        _raise_kv_status(bits)


def flash_attn_with_kvcache(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    rotary_cos: Optional[torch.Tensor] = None,
    rotary_sin: Optional[torch.Tensor] = None,
    cache_seqlens: Optional[Union[torch.Tensor, int]] = None,
    cache_batch_idx: Optional[torch.Tensor] = None,
    cache_leftpad: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    window_size: Tuple[int, int] = (-1, -1),
    softcap: float = 0.0,
    rotary_interleaved: bool = True,
    alibi_slopes: Optional[torch.Tensor] = None,
    num_splits: int = 0,
    return_softmax_lse: bool = False,
    validate: bool = True,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """KV-cache attention for inference (signature of upstream FlashAttention).

    Supports contiguous caches (optionally remapped by cache_batch_idx), paged
    caches via block_table, in-place append of k/v at cache_seqlens and split-KV
    (num_splits, 0 = heuristic).  Beyond the reference (which rejects them),
    rotary embeddings, window_size, softcap, alibi_slopes and cache_leftpad work
    with upstream FlashAttention's semantics: query i, at key position
    p = i + L - seqlen_q, sees keys [p - left, p + right] (-1: unbounded; causal
    caps the right side at p); softcap > 0 replaces each scaled score x by
    softcap * tanh(x / softcap); ALiBi (fp32 slopes [nheads] or [batch, nheads])
    adds -slope * |p - j| to the score of key j; keys before cache_leftpad[b]
    (int32 [batch]) do not exist.  With rotary_cos / rotary_sin (fp16
    [seqlen_ro, rotary_dim / 2]; k and v required), the first rotary_dim channels
    of new key t are rotated at position cache_seqlens[b] + t before the append,
    and q's at cache_seqlens[b] + i when causal or windowed, else at
    cache_seqlens[b]; rotary_interleaved pairs channels (2j, 2j + 1), otherwise
    (j, j + rotary_dim / 2).

    validate (after the reference's arguments): True checks the cache capacity
    and cache_batch_idx on the host, raising at once as the reference does (a
    device read each, so no graph capture).  False skips those reads: the kernels
    check every sequence themselves (an out-of-range one is neither appended to
    nor attended over) and record the error for flash_attn_kvcache_check(),
    so a decode step can be captured in a HIP graph.

    The entries of block_table are checked by the kernels in both modes (reading
    the table on the host would be a second wait): one that is in use and names
    no page of the cache, such as the -1 that flash_attn_kvcache_alloc leaves
    when the pages run out, is not appended to, page 0 is read in its place, and
    flash_attn_kvcache_check() raises the error.
    """
    # Validation order of interface.py:807-867.
    _validate_unsupported_kvcache_args(rotary_cos, rotary_sin, cache_leftpad, window_size, softcap, alibi_slopes)
    if (k is None) != (v is None):
        raise ValueError("k and v must either both be provided or both be None")
    _validate_supported_head_dim(q.shape[-1])
    batch = q.shape[0]
    if cache_seqlens is None:
        if k is not None:
            raise ValueError("cache_seqlens is required when appending k and v")
        cache_seqlens = _cache_capacity(k_cache, block_table)
    host_length = None  # the longest length, where the host knows it
    if isinstance(cache_seqlens, int):
        host_length = cache_seqlens
        cache_seqlens = torch.full((batch,), cache_seqlens, dtype=torch.int32, device=k_cache.device)
    elif not isinstance(cache_seqlens, torch.Tensor):
        raise TypeError("cache_seqlens must be an int or a torch.Tensor")
    elif cache_seqlens.dtype != torch.int32:
        raise TypeError("cache_seqlens must be a torch.int32 tensor")
    if cache_seqlens.dim() != 1 or cache_seqlens.numel() != batch:
        raise ValueError("cache_seqlens must have shape [batch_size]")
    if block_table is not None:
        if not isinstance(block_table, torch.Tensor):
            raise TypeError("block_table must be a torch.Tensor")
        if block_table.dtype != torch.int32:
            raise TypeError("block_table must be a torch.int32 tensor")
        if block_table.dim() != 2 or block_table.shape[0] != batch:
            raise ValueError("block_table must have shape [batch_size, max_num_blocks_per_seq]")
        if cache_batch_idx is not None:
            raise NotImplementedError("Paged KV cache does not support cache_batch_idx")
        if k_cache.shape[1] % 256 != 0:
            raise ValueError("Paged KV cache block size must be divisible by 256")
    if cache_batch_idx is not None:
        if not isinstance(cache_batch_idx, torch.Tensor):
            raise TypeError("cache_batch_idx must be a torch.Tensor")
        if cache_batch_idx.dtype != torch.int32:
            raise TypeError("cache_batch_idx must be a torch.int32 tensor")
        if cache_batch_idx.dim() != 1 or cache_batch_idx.numel() != batch:
            raise ValueError("cache_batch_idx must have shape [batch_size]")
    if num_splits < 0:
        raise ValueError("num_splits must be non-negative")
    seqlen_new = 0
    if k is not None and v is not None:
        if k.shape[0] != batch or v.shape[0] != batch:
            raise ValueError("k and v batch size must match q")
        if k.shape[1] != v.shape[1]:
            raise ValueError("k and v sequence length must match")
        seqlen_new = k.shape[1]
    if validate:
        # The one device read of the call (a copy without a reduction kernel
        # before it): 52 -> 34 us a decode step on one sequence of 1500 tokens
        # against reading the maximum here and again in the extension.
        if cache_seqlens.numel() == 0:
            max_cache_usage = 0
        else:
            max_cache_usage = int(cache_seqlens.cpu().max()) if host_length is None else host_length
        if max_cache_usage + seqlen_new > _cache_capacity(k_cache, block_table):
            raise ValueError("cache capacity is insufficient for the requested append length")
    if not (q.is_cuda and k_cache.is_cuda and v_cache.is_cuda):
        raise RuntimeError("q, k_cache, v_cache must be CUDA tensors")
    if q.dtype != torch.float16 or k_cache.dtype != torch.float16 or v_cache.dtype != torch.float16:
        raise RuntimeError("q, k_cache, v_cache must be float16 tensors")
    if k is not None and v is not None:
        if not (k.is_cuda and v.is_cuda):
            raise RuntimeError("k and v must be CUDA tensors")
        if k.dtype != torch.float16 or v.dtype != torch.float16:
            raise RuntimeError("k and v must be float16 tensors")
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** (-0.5)
    status = None
    if not validate:
        status = _kv_status(q.device)
    elif block_table is not None and not (q.device.index not in _KV_STATUS and torch.cuda.is_current_stream_capturing()):
        status = _kv_status(q.device)  # for the table's entries
    out, lse = _flash_attn_kvcache_forward(
        q, k_cache, v_cache, k, v, cache_seqlens, cache_batch_idx, block_table, softmax_scale, causal, num_splits,
        status, tuple(window_size), softcap, cache_leftpad, alibi_slopes, rotary_cos, rotary_sin, rotary_interleaved,
        lengths_checked=validate,
    )
    return (out, lse) if return_softmax_lse else out


# ---------------------------------------------------------------------------
# Differential attention (no counterpart in the reference).


class FlashDiffAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, softmax_scale, causal, is_grad_enabled):
        # (Before the copies of strided channels, which require no gradient here.)
        save = is_grad_enabled and any(t.requires_grad for t in (q, k, v, lam))
        q, k, v = (maybe_contiguous(t) for t in (q, k, v))
        out, o2, lse = flash_attn_gpu.diff_fwd(q, k, v, lam, softmax_scale, causal, save)
        if save:
            ctx.save_for_backward(q, k, v, lam, out, o2, lse)
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, lam, out, o2, lse = ctx.saved_tensors
        dq, dk, dv, dlam = flash_attn_gpu.diff_bwd(
            q, k, v, lam, out, o2, lse, maybe_contiguous(dout), ctx.softmax_scale, ctx.causal, ctx.needs_input_grad[3]
        )
        return dq, dk, dv, dlam, None, None, None


class FlashDiffAttnVarlenFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
                is_grad_enabled):
        # (Before the copies of strided channels, which require no gradient here.)
        save = is_grad_enabled and any(t.requires_grad for t in (q, k, v, lam))
        q, k, v = (maybe_contiguous(t) for t in (q, k, v))
        out, o2, lse = flash_attn_gpu.diff_varlen_fwd(
            q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal, save
        )
        if save:
            ctx.save_for_backward(q, k, v, lam, out, o2, lse, cu_seqlens_q, cu_seqlens_k)
            ctx.max_seqlen_q, ctx.max_seqlen_k = max_seqlen_q, max_seqlen_k
            ctx.softmax_scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, lam, out, o2, lse, cu_seqlens_q, cu_seqlens_k = ctx.saved_tensors
        dq, dk, dv, dlam = flash_attn_gpu.diff_varlen_bwd(
            q, k, v, lam, out, o2, lse, maybe_contiguous(dout), cu_seqlens_q, cu_seqlens_k, ctx.max_seqlen_q,
            ctx.max_seqlen_k, ctx.softmax_scale, ctx.causal, ctx.needs_input_grad[3],
        )
        return dq, dk, dv, dlam, None, None, None, None, None, None, None


def _check_diff_args(q, lam, softmax_scale):
    _validate_supported_head_dim(q.shape[-1])
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("differential attention needs float16 or bfloat16 tensors")
    if not isinstance(lam, torch.Tensor) or lam.dtype != torch.float32:
        raise TypeError("lam must be a torch.float32 tensor")
    # One map's channels are half of the head's.
    return (q.shape[-1] // 2) ** (-0.5) if softmax_scale is None else softmax_scale


def flash_diff_attn_func(q, k, v, lam, softmax_scale: Optional[float] = None, causal: bool = False) -> torch.Tensor:
    """Differential attention, (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v.

    q (batch, seqlen_q, nheads, headdim); k, v (batch, seqlen_k, nheads_k, headdim), fp16 or bf16.  The first
    headdim / 2 channels of q and k are the first map's, the others the second's; headdim is 64 or 128 and
    softmax_scale defaults to (headdim / 2) ** -0.5.  lam is fp32: a scalar tensor, (nheads,), or one value for each
    query and head, (batch, seqlen_q, nheads).  causal, grouped heads and rows without a visible key are as in
    flash_attn_func.  Returns out (batch, seqlen_q, nheads, headdim); q, k, v and lam get gradients.

    A backward pass is captured into a graph with torch.autograd.grad, or when no eager graph of the same leaves is
    alive: torch ties the accumulation into a leaf's grad to the stream of its first live graph."""
    softmax_scale = _check_diff_args(q, lam, softmax_scale)
    return FlashDiffAttnFunc.apply(q, k, v, lam, softmax_scale, causal, torch.is_grad_enabled())


def flash_diff_attn_varlen_func(
    q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q: int, max_seqlen_k: int,
    softmax_scale: Optional[float] = None, causal: bool = False,
) -> torch.Tensor:
    """flash_diff_attn_func on packed sequences: q (total_q, nheads, headdim); k, v (total_k, nheads_k, headdim);
    cu_seqlens_* int32 (batch_size + 1,); lam a scalar, (nheads,) or (total_q, nheads).  Rows that no sequence covers
    are 0 in out and in the gradients."""
    softmax_scale = _check_diff_args(q, lam, softmax_scale)
    return FlashDiffAttnVarlenFunc.apply(
        q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
        torch.is_grad_enabled(),
    )


def flash_diff_attn_with_kvcache(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    lam: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    cache_seqlens: Optional[Union[torch.Tensor, int]] = None,
    cache_batch_idx: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    num_splits: int = 0,
    return_softmax_lse: bool = False,
    validate: bool = True,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Differential attention with a KV cache, for inference.

    The caches, k, v, cache_seqlens, cache_batch_idx and block_table are those of flash_attn_with_kvcache (fp16 or
    bf16; both maps' keys are the halves of a key's channels, so the two functions take the same caches; pages are a
    multiple of 64 tokens here); lam is a scalar, (nheads,) or (batch, seqlen_q, nheads).  num_splits > 0 cuts the
    cache's capacity into that many pieces (calls of few query rows), and a row's bits then do not depend on the batch.
    return_softmax_lse adds the log-sum-exp of both maps, fp32 (2, batch, nheads, seqlen_q).  A q without rows
    (seqlen_q 0) appends alone.

    validate as there: True checks lengths, rows and pages on the host; False leaves that to the kernels, which
    record what is wrong for flash_attn_kvcache_check(): a sequence with a bad length or row is neither appended to
    nor attended over, a page outside the cache is not written and page 0 is read in its place."""
    softmax_scale = _check_diff_args(q, lam, softmax_scale)
    if (k is None) != (v is None):
        raise ValueError("k and v must either both be provided or both be None")
    batch = q.shape[0]
    capacity = _cache_capacity(k_cache, block_table)
    if cache_seqlens is None:
        if k is not None:
            raise ValueError("cache_seqlens is required when appending k and v")
        cache_seqlens = capacity
    if isinstance(cache_seqlens, int):
        cache_seqlens = torch.full((batch,), cache_seqlens, dtype=torch.int32, device=k_cache.device)
    elif not isinstance(cache_seqlens, torch.Tensor):
        raise TypeError("cache_seqlens must be an int or a torch.Tensor")
    for name, t, shape in (("cache_seqlens", cache_seqlens, (batch,)), ("cache_batch_idx", cache_batch_idx, (batch,)),
                           ("block_table", block_table, (batch, None))):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"{name} must be a torch.int32 tensor")
        if t.dim() != len(shape) or t.shape[0] != batch:
            raise ValueError(f"{name} must have batch_size rows")
    if block_table is not None and cache_batch_idx is not None:
        raise NotImplementedError("Paged KV cache does not support cache_batch_idx")
    if num_splits < 0:
        raise ValueError("num_splits must be non-negative")
    if validate and batch > 0:
        lens = cache_seqlens.cpu().long()
        used = lens + (0 if k is None else k.shape[1])
        if int(lens.min()) < 0 or int(used.max()) > capacity:
            raise ValueError("cache capacity is insufficient for the requested append length")
        if cache_batch_idx is not None:
            rows = cache_batch_idx.cpu()
            if int(rows.min()) < 0 or int(rows.max()) >= k_cache.shape[0]:
                raise RuntimeError("cache_batch_idx entries must be within cache batch bounds")
        if block_table is not None and block_table.shape[1] > 0:
            pages = block_table.cpu()
            needed = torch.arange(pages.shape[1]) * k_cache.shape[1] < used[:, None]
            if bool((needed & ((pages < 0) | (pages >= k_cache.shape[0]))).any()):
                raise RuntimeError("block_table entries in use must be pages of the cache")
    status = None if validate or not q.is_cuda else _kv_status(q.device)
    q, k, v, cache_seqlens, cache_batch_idx, block_table = (
        maybe_contiguous(t) for t in (q, k, v, cache_seqlens, cache_batch_idx, block_table)
    )
    out, lse = flash_attn_gpu.diff_fwd_kvcache(
        q, k_cache, v_cache, lam, k, v, cache_seqlens, cache_batch_idx, block_table, softmax_scale, causal, num_splits,
        status,
    )
    return (out, lse) if return_softmax_lse else out


# ---------------------------------------------------------------------------
# The pages of a paged KV cache (no counterpart in the reference).
#
# The state is four tensors of the caller's: the pools k_cache and v_cache [num_blocks, page_block_size, nheads_k,
# headdim], block_table int32 [rows, max_num_blocks_per_seq] (-1: no page), cache_seqlens int32 [rows] and page_refs
# int32 [num_blocks], the number of table entries that name each page (0: free).  A new cache has a table of -1 and
# zeros elsewhere.  All calls work in place on the device, on the current stream, with no host read when validate is
# False.  validate=True reads what the kernels found wrong (a synchronisation) and raises it; False leaves it for
# flash_attn_kvcache_check().  Either way a call that gives out pages changes nothing when something is wrong.


def _kv_pages_call(fn, device, validate, *args):
    status = torch.zeros(1, dtype=torch.int32, device=device) if validate else _kv_status(device)
    fn(*args, status)
    if validate:
        _raise_kv_status(int(status.item()))


def _check_pages(block_table=None, cache_seqlens=None, page_refs=None, **lists) -> None:
    for name, t in (("block_table", block_table), ("cache_seqlens", cache_seqlens), ("page_refs", page_refs),
                    *lists.items()):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"{name} must be a torch.int32 tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")


def _check_whole(what: str, *pools) -> None:
    """Pools of codes are half of a cache in 8 bits: a call that plans its copies itself would leave their scales behind."""
    for c in pools:
        if isinstance(c, torch.Tensor) and c.dtype in (torch.float8_e4m3fn, torch.int8):
            raise NotImplementedError(
                f"{what} would leave the scales of a cache in 8 bits behind; use flash_attn_kvcache_copy_pages for codes and "
                "scales (pools of bytes without scales: .view(torch.uint8))")


def flash_attn_kvcache_alloc(block_table, cache_seqlens, page_refs, seqlen_new: Union[int, torch.Tensor],
                             page_block_size: int, validate: bool = True) -> None:
    """Give every row the pages that its next seqlen_new tokens (an int, or int32 [rows], 0 for none) need and its
    table lacks: the lowest free pages first, in the order of the rows."""
    _check_pages(block_table, cache_seqlens, page_refs)
    per_row = seqlen_new if isinstance(seqlen_new, torch.Tensor) else None
    if per_row is not None:
        _check_pages(seqlen_new=per_row)
    elif seqlen_new < 0:
        raise ValueError("seqlen_new must be non-negative")
    if page_block_size <= 0:
        raise ValueError("page_block_size must be positive")
    _kv_pages_call(flash_attn_gpu.kvpages_alloc, block_table.device, validate, block_table, cache_seqlens, page_refs,
                   0 if per_row is not None else seqlen_new, per_row, page_block_size)


def flash_attn_kvcache_copy_pages(k_cache, v_cache, src: torch.Tensor, dst: torch.Tensor, validate: bool = True) -> None:
    """Copy page src[i] of both pools to page dst[i], all pairs at once.  A page that one pair writes may be in no
    other pair; such pairs, and those out of range, are not copied and reported."""
    _check_pages(src=src, dst=dst)
    _kv_pages_call(flash_attn_gpu.kvpages_copy, src.device, validate, k_cache, v_cache, src, dst)


def flash_attn_kvcache_fork(k_cache, v_cache, block_table, cache_seqlens, page_refs, parents: torch.Tensor,
                            children: torch.Tensor, validate: bool = True) -> None:
    """Make row children[i] (empty, in the list once, no parent itself) a fork of row parents[i]: it shares the
    parent's full pages, and where the parent's last page is partly filled it gets a free page (lowest first, in the
    list's order) with a copy of that page's tokens; the rest of that page is left as it was.  Not for the codes of a cache
    in 8 bits, whose scales would stay behind."""
    _check_whole("flash_attn_kvcache_fork", k_cache, v_cache)
    _check_pages(block_table, cache_seqlens, page_refs, parents=parents, children=children)
    _kv_pages_call(flash_attn_gpu.kvpages_fork, block_table.device, validate, k_cache, v_cache, block_table,
                   cache_seqlens, page_refs, parents, children)


def flash_attn_kvcache_free(block_table, cache_seqlens, page_refs, rows: torch.Tensor, validate: bool = True) -> None:
    """Empty the rows: each of their pages loses a reference (and is free at 0), their table entries become -1 and
    their lengths 0.  Empty rows, and a row named twice, are nothing special; a row out of range is reported."""
    _check_pages(block_table, cache_seqlens, page_refs, rows=rows)
    _kv_pages_call(flash_attn_gpu.kvpages_free, block_table.device, validate, block_table, cache_seqlens, page_refs,
                   rows)


def flash_attn_kvcache_compact(k_cache, v_cache, block_table, page_refs) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the pages in use to the front of the pools: with n of them, the k-th free page below n takes the contents
    of the k-th used page from n on.  Returns the table and the counts afterwards (new tensors) and n (int32 [1]).
    The moved pages stay as they were in their old places, so the old table stays right for work that is already
    queued, until those pages are given out again.  Not for the codes of a cache in 8 bits, whose scales would stay behind."""
    _check_whole("flash_attn_kvcache_compact", k_cache, v_cache)
    _check_pages(block_table, page_refs=page_refs)
    return flash_attn_gpu.kvpages_compact(k_cache, v_cache, block_table, page_refs)


# ---------------------------------------------------------------------------
# Rotary positions (no counterpart in the reference).


def flash_attn_rotary_tables(
    seqlen: int, rotary_dim: int, base: float = 10000.0, factor: float = 1.0, original_seqlen: Optional[int] = None,
    low_turns: float = 1.0, high_turns: float = 32.0, attention_factor: float = 1.0, offset: int = 0,
    dtype: torch.dtype = torch.float32, device: Union[torch.device, str, int, None] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin (seqlen, rotary_dim / 2) of the angles (offset + i) * f_j, f_j = base ** (-2 j / rotary_dim), computed
    in 64 bits and rounded once to dtype (float32, float16 or bfloat16); rotary_dim is a multiple of 16.  Positions lie
    within 2 ** 26 of 0, where 64 bits leave the angles right to half a step of float32.

    For contexts longer than those of the training by a factor: f_j / factor, or, with original_seqlen (the training's
    length), by the turns t that a pair makes in it: f_j for t >= high_turns, f_j / factor for t <= low_turns, and
    f_j (keep + (1 - keep) / factor), keep = (t - low_turns) / (high_turns - low_turns), in between.  attention_factor
    multiplies both tables, so that scores of rotated q and k grow by its square.

    flash_attn_rotary_func takes them in any of the types, flash_attn_with_kvcache in float16."""
    if rotary_dim <= 0 or rotary_dim % 16 != 0 or rotary_dim > 256:
        raise ValueError("rotary_dim must be a multiple of 16 up to 256")
    if seqlen < 0:
        raise ValueError("seqlen must be non-negative")
    if abs(offset) > 2 ** 26 or offset + max(seqlen, 1) - 1 > 2 ** 26:
        raise ValueError("positions must be within 2 ** 26 of 0")
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError("dtype must be torch.float32, torch.float16 or torch.bfloat16")
    if not all(math.isfinite(x) for x in (base, factor, attention_factor)) or base <= 0 or factor <= 0:
        raise ValueError("base and factor must be positive and finite, attention_factor finite")
    if original_seqlen is not None and (original_seqlen <= 0 or not high_turns > low_turns):
        raise ValueError("original_seqlen must be positive and high_turns larger than low_turns")
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise RuntimeError("rotary tables are made on a CUDA device")
    cos, sin = (torch.empty((seqlen, rotary_dim // 2), dtype=dtype, device=device) for _ in range(2))
    flash_attn_gpu.rotary_tables(cos, sin, offset, base, factor, original_seqlen or 0.0, low_turns, high_turns,
                                 attention_factor)
    return cos, sin


class FlashAttnRotaryFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, *rest):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*(x for x in rest if isinstance(x, torch.Tensor)))
        ctx.rest = tuple(None if isinstance(x, torch.Tensor) else (x,) for x in rest)
        return tuple(flash_attn_gpu.rotary(maybe_contiguous(q), maybe_contiguous(k), *rest))

    @staticmethod
    def backward(ctx, dq, dk):
        tensors = iter(ctx.saved_tensors)
        rest = tuple(next(tensors) if x is None else x[0] for x in ctx.rest)
        back = (*rest[:-1], not rest[-1])
        # (A gradient of k alone is rotated as q.)
        x, y = (dk, None) if dq is None else (dq, dk)
        if x is not None:
            if torch.is_grad_enabled():  # create_graph: the gradient is a rotation, too, with a gradient of its own
                x, y = FlashAttnRotaryFunc.apply(x, y, *back)
            else:
                x, y = flash_attn_gpu.rotary(maybe_contiguous(x), maybe_contiguous(y), *back)
        return ((None, x) if dq is None else (x, y)) + (None,) * len(rest)


def flash_attn_rotary_func(
    q, k, rotary_cos, rotary_sin, rotary_interleaved: bool = True, positions: Optional[torch.Tensor] = None,
    seqlen_offsets: Union[int, torch.Tensor] = 0, cu_seqlens: Optional[torch.Tensor] = None,
):
    """Rotate the first rotary_dim channels of q and k by their positions, as flash_attn_with_kvcache does.

    q (batch, seqlen, nheads, headdim) and k (batch, seqlen, nheads_k, headdim), fp16 or bf16, headdim 64 or 128; with
    cu_seqlens (int32 (batch_size + 1,)) packed: (total, nheads, headdim), and rows that no sequence covers become 0.
    k may be None.  rotary_cos and rotary_sin (rows, rotary_dim / 2) are float32, float16 or bfloat16 (as
    flash_attn_rotary_tables makes them); pairs are channels (2j, 2j + 1) if rotary_interleaved, else (j, j + rotary_dim / 2).

    Row i of a sequence is at position seqlen_offsets + i (an int, or int32 (batch_size,): the tokens before it), or, with
    positions (int32, (batch, seqlen) or (total,)), where they say.  A row whose position the tables do not have becomes
    NaN in the rotated channels.

    Returns q and k rotated, new tensors (q alone where k is None); q and k get gradients of any order, the tables none."""
    for name, t in (("rotary_cos", rotary_cos), ("rotary_sin", rotary_sin)):
        if not isinstance(t, torch.Tensor) or t.dim() != 2:
            raise TypeError(f"{name} must be a 2-D tensor (rows, rotary_dim / 2)")
    for name, t in (("positions", positions), ("cu_seqlens", cu_seqlens)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32):
            raise TypeError(f"{name} must be a torch.int32 tensor")
    offsets, offset = None, seqlen_offsets
    if isinstance(seqlen_offsets, torch.Tensor):
        offsets, offset = seqlen_offsets, 0
        if offsets.dtype != torch.int32:
            raise TypeError("seqlen_offsets must be an int or a torch.int32 tensor")
    elif not isinstance(seqlen_offsets, int):
        raise TypeError("seqlen_offsets must be an int or a torch.int32 tensor")
    rest = (maybe_contiguous(rotary_cos), maybe_contiguous(rotary_sin), rotary_interleaved, positions,
            maybe_contiguous(offsets), offset, maybe_contiguous(cu_seqlens), False)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)
                                    or rotary_cos.requires_grad or rotary_sin.requires_grad):
        if rotary_cos.requires_grad or rotary_sin.requires_grad:
            raise RuntimeError("rotary_cos and rotary_sin get no gradient")
        q, k = FlashAttnRotaryFunc.apply(q, k, *rest)
    else:
        q, k = flash_attn_gpu.rotary(maybe_contiguous(q), maybe_contiguous(k), *rest)
    return q if k is None else (q, k)


# ---------------------------------------------------------------------------
# A KV cache in 8 bits (no counterpart in the reference).
#
# The caches are those of flash_attn_with_kvcache with codes of one byte: k_cache and v_cache [num_blocks, page_block_size,
# nheads_k, headdim] with a block_table, or [rows, capacity, nheads_k, headdim], torch.float8_e4m3fn or torch.int8, and
# k_scale and v_scale fp32 [num_blocks or rows, page_block_size or capacity / block, nheads_k]: a value is its code times
# the scale of its block of tokens and head.  block (32, 64, 128 or 256 tokens) follows from the shapes.  New caches need no
# clearing.  The appends make scales powers of two: the smallest s >= 2 ** -126 with max|x| <= most * s (most is 448 for
# e4m3, 127 for int8), or the old one where the block holds earlier tokens and that is larger; codes are x / s, rounded to
# nearest even, and earlier tokens' codes are rounded again where a scale grows.  A NaN or an infinity among a block's new
# values makes its scale NaN.  The readers take any finite codes and scales that are not negative; a scale that is NaN or
# infinite makes NaN those rows of attention that see its block.


def _q8_places(batch, k_cache, lens, seqlen_new, cache_batch_idx, block_table, validate):
    """What is wrong with lengths (int32 [batch] tokens before the new ones), rows and pages; validate reads them."""
    for name, t, dim in (("cache_batch_idx", cache_batch_idx, 1), ("block_table", block_table, 2)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"{name} must be a torch.int32 tensor")
        if t.dim() != dim or t.shape[0] != batch:
            raise ValueError(f"{name} must have batch_size rows")
    if block_table is not None and cache_batch_idx is not None:
        raise NotImplementedError("Paged KV cache does not support cache_batch_idx")
    if not validate or batch == 0:
        return
    capacity, before = _cache_capacity(k_cache, block_table), lens.cpu().long()
    used = before + (seqlen_new.cpu().long() if isinstance(seqlen_new, torch.Tensor) else seqlen_new)
    if int(before.min()) < 0 or int(used.max()) > capacity or int((used - before).min()) < 0:
        raise ValueError("cache capacity is insufficient for the requested append length")
    if cache_batch_idx is not None:
        rows = cache_batch_idx.cpu()
        if int(rows.min()) < 0 or int(rows.max()) >= k_cache.shape[0]:
            raise RuntimeError("cache_batch_idx entries must be within cache batch bounds")
    if block_table is not None and block_table.shape[1] > 0:
        pages = block_table.cpu()
        needed = torch.arange(pages.shape[1]) * k_cache.shape[1] < used[:, None]
        if bool((needed & ((pages < 0) | (pages >= k_cache.shape[0]))).any()):
            raise RuntimeError("block_table entries in use must be pages of the cache")


def _q8_lengths(cache_seqlens, batch):
    if not isinstance(cache_seqlens, torch.Tensor) or cache_seqlens.dtype != torch.int32:
        raise TypeError("cache_seqlens must be a torch.int32 tensor")
    if cache_seqlens.dim() != 1 or cache_seqlens.shape[0] != batch:
        raise ValueError("cache_seqlens must have batch_size rows")


def flash_attn_kvcache_append_q8(
    k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
    v_scale: torch.Tensor, cache_seqlens: torch.Tensor, cache_batch_idx: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None, seqlens_new: Optional[torch.Tensor] = None, validate: bool = True,
) -> None:
    """Quantise k and v (batch, seqlen_new, nheads_k, headdim; fp16 or bf16) into a cache in 8 bits at cache_seqlens
    (int32 (batch,), which the caller advances).  seqlens_new (int32 (batch,)): new tokens of each sequence of a padded
    batch, the rows of k and v behind them are not looked at; None: all of them.  No two sequences of a call may append to one
    block of tokens.

    validate as in flash_diff_attn_with_kvcache: True checks lengths, rows and pages on the host; False leaves that to the
    kernels, which append nothing where something is wrong and record it for flash_attn_kvcache_check()."""
    batch = k.shape[0]
    _q8_lengths(cache_seqlens, batch)
    if seqlens_new is not None:
        if not isinstance(seqlens_new, torch.Tensor) or seqlens_new.dtype != torch.int32:
            raise TypeError("seqlens_new must be a torch.int32 tensor")
        if seqlens_new.dim() != 1 or seqlens_new.shape[0] != batch:
            raise ValueError("seqlens_new must have batch_size rows")
        if validate and batch > 0 and int(seqlens_new.max()) > k.shape[1]:
            raise ValueError("seqlens_new must not be larger than the sequence length of k and v")
    _q8_places(batch, k_cache, cache_seqlens, k.shape[1] if seqlens_new is None else seqlens_new, cache_batch_idx,
               block_table, validate)
    status = None if validate or not k.is_cuda else _kv_status(k.device)
    flash_attn_gpu.kv8_append(
        maybe_contiguous(k), maybe_contiguous(v), k_cache, v_cache, k_scale, v_scale, maybe_contiguous(cache_seqlens),
        maybe_contiguous(cache_batch_idx), maybe_contiguous(block_table), maybe_contiguous(seqlens_new), status,
    )


def flash_attn_kvcache_read_q8(
    k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, cu_seqlens_k: torch.Tensor,
    total_k: int, cache_batch_idx: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None,
    dtype: torch.dtype = torch.float16, validate: bool = True,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first tokens of every sequence of a cache in 8 bits, packed for flash_attn_varlen_func: k and v (total_k,
    nheads_k, headdim) of dtype (float16 or bfloat16), cu_seqlens_k[b + 1] - cu_seqlens_k[b] tokens of sequence b in rows
    cu_seqlens_k[b] and on.  Values are rounded once (those of float16 may overflow).  Rows that no sequence covers are 0.

    validate as in flash_attn_kvcache_append_q8; with False, a sequence that is longer than the cache's capacity is 0."""
    if not isinstance(cu_seqlens_k, torch.Tensor) or cu_seqlens_k.dtype != torch.int32:
        raise TypeError("cu_seqlens_k must be a torch.int32 tensor")
    if cu_seqlens_k.dim() != 1 or cu_seqlens_k.shape[0] < 1:
        raise ValueError("cu_seqlens_k must have batch_size + 1 elements")
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("dtype must be torch.float16 or torch.bfloat16")
    if total_k < 0:
        raise ValueError("total_k must be non-negative")
    batch = cu_seqlens_k.shape[0] - 1
    if validate:
        cu = cu_seqlens_k.cpu()
        if int(cu[0]) < 0 or int(cu[-1]) > total_k or bool((cu[1:] < cu[:-1]).any()):
            raise ValueError("cu_seqlens_k must not decrease and end at total_k at most")
        _q8_places(batch, k_cache, torch.zeros_like(cu[1:]), cu[1:] - cu[:-1], cache_batch_idx, block_table, True)
    else:
        _q8_places(batch, k_cache, None, 0, cache_batch_idx, block_table, False)
    status = None if validate or not k_cache.is_cuda else _kv_status(k_cache.device)
    return flash_attn_gpu.kv8_read(
        k_cache, v_cache, k_scale, v_scale, maybe_contiguous(cu_seqlens_k), total_k, maybe_contiguous(cache_batch_idx),
        maybe_contiguous(block_table), dtype == torch.bfloat16, status,
    )


def flash_attn_with_kvcache_q8(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    cache_seqlens: Optional[Union[torch.Tensor, int]] = None,
    cache_batch_idx: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    window_size: Tuple[int, int] = (-1, -1),
    num_splits: int = 0,
    return_softmax_lse: bool = False,
    validate: bool = True,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """flash_attn_with_kvcache over a cache in 8 bits, for inference: k and v are quantised into it as by
    flash_attn_kvcache_append_q8, then q (batch, seqlen_q, nheads, headdim; fp16 or bf16, headdim 64 or 128) attends over
    cache_seqlens + seqlen_new keys.  Masks, window_size, grouped heads and rows without a visible key (0, LSE 0) as there.

    The keys are cut into pieces on the device by the lengths of the whole batch; num_splits > 0 cuts the cache's capacity
    into that many instead, and a row's bits then do not depend on the batch.  return_softmax_lse adds the log-sum-exp,
    fp32 (batch, nheads, seqlen_q).  Calls with few query rows a KV head (nheads / nheads_k * seqlen_q) keep 16 bits of the
    probabilities in the product with v, calls with many 11, as flash_attn_func does: many are 64 where num_splits is given,
    else from 32 on by the work that the cache's capacity allows.  A q without rows (seqlen_q 0) appends alone.  For rotary positions rotate q and k by
    flash_attn_rotary_func(..., seqlen_offsets=cache_seqlens) first.

    validate as in flash_attn_kvcache_append_q8; with False a call can be captured in a graph, a sequence with a bad length
    or row is neither appended to nor attended over, a page outside the cache is not written and page 0 is read in its place."""
    _validate_supported_head_dim(q.shape[-1])
    if (k is None) != (v is None):
        raise ValueError("k and v must either both be provided or both be None")
    if len(tuple(window_size)) != 2 or not all(isinstance(w, int) for w in window_size):
        raise TypeError("window_size must be a pair of ints")
    batch = q.shape[0]
    if cache_seqlens is None:
        if k is not None:
            raise ValueError("cache_seqlens is required when appending k and v")
        cache_seqlens = _cache_capacity(k_cache, block_table)
    if isinstance(cache_seqlens, int):
        cache_seqlens = torch.full((batch,), cache_seqlens, dtype=torch.int32, device=k_cache.device)
    _q8_lengths(cache_seqlens, batch)
    if num_splits < 0:
        raise ValueError("num_splits must be non-negative")
    _q8_places(batch, k_cache, cache_seqlens, 0 if k is None else k.shape[1], cache_batch_idx, block_table, validate)
    status = None if validate or not q.is_cuda else _kv_status(q.device)
    out, lse = flash_attn_gpu.kv8_fwd_kvcache(
        maybe_contiguous(q), k_cache, v_cache, k_scale, v_scale, maybe_contiguous(k), maybe_contiguous(v),
        maybe_contiguous(cache_seqlens), maybe_contiguous(cache_batch_idx), maybe_contiguous(block_table),
        _default_scale(q, softmax_scale), causal, max(window_size[0], -1), max(window_size[1], -1), num_splits, status,
    )
    return (out, lse) if return_softmax_lse else out
