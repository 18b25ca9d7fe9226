"""Causal softmax attention on MI355X: whole prompts, a paged cache, single tokens.

The token mixer of the decoder's full-attention layers (omegalax/models/qwen3_5/attention.py:115-119
between its projections, norms, rotary embedding and output gate), beside the gated delta rule of
``omegalax_amd.deltanet`` and in the same manner: packed sequences by ``cu_seqlens``, autograd, a
cache that the decode step updates in place.  Tokens are bf16, ``[B, T, heads, D]``; query head h
reads key head ``h // (Hq // Hkv)``.

The cache is a pool of pages ``k_pages``, ``v_pages`` [pages, page_size, Hkv, D] bf16 (D 64, 128 or
256, page_size a multiple of 16), a ``block_table`` [N, width] int32 that names the pages of each
sequence in order, and ``lengths`` [N] int32, the tokens each sequence held before the call.  The
caller advances ``lengths``; a negative one marks a sequence that takes no part.  Serving a turn is
``kv_pages_write`` and then ``attention_prefill_paged`` with the same lengths; each further token is
one ``attention_decode_step``.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .deltanet import _cu_seqlens, _no_tangents, _ptr, _stream, _workspace

__all__ = ["attention_prefill", "attention_prefill_bwd", "attention_prefill_paged",
           "attention_decode_step", "kv_pages_write"]


_BF16 = torch.bfloat16


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name, *dims):
    """A workspace size, which depends on the arguments alone."""
    return getattr(_lib.lib(), name)(*dims)


def _call(dev, name, *args):
    """An entry point on ``dev``'s current stream, with ``dev`` the current device."""
    if torch.cuda.current_device() == dev.index:
        return _lib.call(name, *args, _stream(dev))
    with torch.cuda.device(dev):
        return _lib.call(name, *args, _stream(dev))


def _device(*ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("omegalax_amd kernels need GPU tensors (got a CPU tensor)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    return dev


def _tokens(name, t, dims):
    """A bf16 tensor of token rows [..., heads, D] whose heads lie side by side, with any token
    stride the kernels take (columns of one projection); another layout is copied."""
    shape = t.shape
    if len(shape) != dims or t.dtype is not _BF16:
        raise ValueError(f"{name} must be bf16 with {dims} dimensions (got {t.dtype}, {tuple(shape)})")
    H, D = shape[-2:]
    if t.is_contiguous():
        return (t if t.data_ptr() % 16 == 0 else t.clone()), H * D
    st = t.stride()
    # stride of a dimension of one is of no consequence
    ld = st[-3] if shape[-3] > 1 else H * D
    if dims == 4 and shape[1] == 1 and shape[0] > 1:
        ld = st[0]
    ok = (D == 1 or st[-1] == 1) and (H == 1 or st[-2] == D) and H * D <= ld <= 1 << 22
    if dims == 4 and shape[0] > 1:
        ok = ok and st[0] == shape[1] * ld
    if not (ok and ld % 8 == 0 and t.data_ptr() % 16 == 0):
        t, ld = t.contiguous(), H * D
        if t.data_ptr() % 16 != 0:
            t = t.clone()
    return t, ld


def _dense(name, t, shape):
    if tuple(t.shape) != tuple(shape) or t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bf16 {tuple(shape)} (got {t.dtype}, {tuple(t.shape)})")
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _scale(scale, D):
    return float(D ** -0.5) if scale is None else float(scale)


def _qkv(q, k, v, cu_seqlens, dims=4):
    dev = _device(q, k, v)
    (q, q_ld), (k, k_ld), (v, v_ld) = _tokens("q", q, dims), _tokens("k", k, dims), _tokens("v", v, dims)
    if k.shape != v.shape or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"shape mismatch: q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    N = q.shape[0]
    if cu_seqlens is not None:
        cu_seqlens, N = _cu_seqlens(cu_seqlens, q.shape[0], q.shape[1], dev)
    return dev, q, k, v, q_ld, k_ld, v_ld, cu_seqlens, N


def _prefill_fwd(q, k, v, cu_seqlens, scale, with_lse, with_rest):
    dev, q, k, v, q_ld, k_ld, v_ld, cu, N = _qkv(q, k, v, cu_seqlens)
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    o = torch.empty((B, T, Hq, D), dtype=torch.bfloat16, device=dev)
    lse = torch.empty((B, T, Hq), dtype=torch.float32, device=dev) if with_lse else None
    rest = torch.empty_like(o) if with_rest else None
    ws_bytes = _workspace_bytes("omx_gdn_attn_fwd_workspace_size", T, Hq, Hkv, 0 if cu is None else N)
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_attn_fwd", _ptr(q), _ptr(k), _ptr(v), q_ld, k_ld, v_ld, _ptr(cu), N, _ptr(o),
          _ptr(lse), _ptr(rest), B, T, Hq, Hkv, D, _scale(scale, D), _ptr(ws), ws_bytes)
    return o, lse, rest


def attention_prefill_bwd(q, k, v, o, lse, do, *, o_rest=None, cu_seqlens=None, scale=None):
    """Gradients (dq, dk, dv) of ``attention_prefill`` for the cotangent ``do`` of its output.

    ``o`` and ``lse`` are what the forward returned with ``output_lse=True``.  ``o_rest``, what
    the rounding of o left (bf16, as o), makes dq and dk about 6% more exact; autograd keeps it.
    The gradients are dense bf16 tensors of the inputs' shapes; those of a key head are summed
    over its query heads.  A value of a sequence that is not finite may reach all of its gradients.
    """
    _no_tangents("attention_prefill_bwd", q, k, v, o, lse, do, o_rest)
    dev, q, k, v, q_ld, k_ld, v_ld, cu, N = _qkv(q, k, v, cu_seqlens)
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    _device(q, o, lse, do, o_rest)
    o, do = _dense("o", o, q.shape), _dense("do", do.to(torch.bfloat16), q.shape)
    if tuple(lse.shape) != (B, T, Hq) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be fp32 {(B, T, Hq)} (got {lse.dtype}, {tuple(lse.shape)})")
    lse = lse.contiguous()
    if o_rest is not None:
        o_rest = _dense("o_rest", o_rest, q.shape)
    dq = torch.empty((B, T, Hq, D), dtype=torch.bfloat16, device=dev)
    dk = torch.empty((B, T, Hkv, D), dtype=torch.bfloat16, device=dev)
    dv = torch.empty_like(dk)
    ws_bytes = _workspace_bytes("omx_gdn_attn_bwd_workspace_size", B, T, Hq, Hkv, D, 0 if cu is None else N)
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_attn_bwd", _ptr(q), _ptr(k), _ptr(v), q_ld, k_ld, v_ld, _ptr(cu), N, _ptr(o),
          _ptr(lse), _ptr(o_rest), _ptr(do), _ptr(dq), _ptr(dk), _ptr(dv), B, T, Hq, Hkv, D, _scale(scale, D),
          _ptr(ws), ws_bytes)
    return dq, dk, dv


class _AttentionPrefill(torch.autograd.Function):
    """Autograd node of the prompt attention: forward omx_gdn_attn_fwd, backward omx_gdn_attn_bwd
    from the saved output and logarithms (no score is kept)."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale):
        o, lse, rest = _prefill_fwd(q, k, v, cu_seqlens, scale, True, True)
        ctx.save_for_backward(q, k, v, o, lse, rest, cu_seqlens)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _dlse):
        if do is None:
            return None, None, None, None, None
        q, k, v, o, lse, rest, cu_seqlens = ctx.saved_tensors
        dq, dk, dv = attention_prefill_bwd(q, k, v, o, lse, do, o_rest=rest, cu_seqlens=cu_seqlens,
                                           scale=ctx.scale)
        return dq, dk, dv, None, None


def attention_prefill(q, k, v, *, cu_seqlens=None, scale=None, output_lse=False):
    """Causal softmax attention of whole prompts.

    q [B,T,Hq,D], k and v [B,T,Hkv,D] bf16 (D a multiple of 8 up to 256; up to 32 query heads per
    key head; views into one projection are read in place).  ``cu_seqlens`` (int32 [N+1], B == 1)
    packs N sequences, as in ``gdn_prefill``.  ``scale`` defaults to D ** -0.5.  Returns o
    [B,T,Hq,D] bf16, or (o, lse) with the fp32 logarithms [B,T,Hq] of the softmax sums.  When
    gradients are enabled and an input requires them, the call is recorded for autograd (once, and
    not through lse); forward-mode derivatives are refused.  A row sees no key after it, not even one
    that is not finite.
    """
    _no_tangents("attention_prefill", q, k, v)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        o, lse = _AttentionPrefill.apply(q, k, v, cu_seqlens, scale)
    else:
        o, lse, _ = _prefill_fwd(q, k, v, cu_seqlens, scale, output_lse, False)
    return (o, lse) if output_lse else o


def _cache(dev, k_pages, v_pages, block_table, lengths, N, Hkv, D):
    """Checks of the cache's tensors, which are used where they lie."""
    for t in (k_pages, v_pages, block_table, lengths):
        if t.device != dev:
            _device(t)
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    shape = k_pages.shape
    if v_pages.shape != shape or len(shape) != 4 or shape[2] != Hkv or shape[3] != D:
        raise ValueError(f"k_pages and v_pages must both be [pages, page_size, {Hkv}, {D}] "
                         f"(got {tuple(shape)}, {tuple(v_pages.shape)})")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.dtype is not _BF16 or not t.is_contiguous():
            raise ValueError(f"{name} must be bf16 and contiguous (got {t.dtype})")
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.shape[0] != N:
        raise ValueError(f"block_table must be int32 [{N}, width] (got {block_table.dtype}, "
                         f"{tuple(block_table.shape)})")
    if lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.shape[0] != N:
        raise ValueError(f"lengths must be int32 [{N}] (got {lengths.dtype}, {tuple(lengths.shape)})")
    return block_table.contiguous(), lengths.contiguous(), shape[0], shape[1]


def _no_grad_only(name, *ts):
    for t in ts:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name}: gradients through the cache are not supported")
    _no_tangents(name, *ts)


def kv_pages_write(k, v, k_pages, v_pages, block_table, lengths, *, cu_seqlens=None):
    """Appends new tokens' keys and values to a paged cache, in place.

    k, v [B,T,Hkv,D] bf16, N = B sequences of T tokens or N packed by ``cu_seqlens`` (B == 1).
    Token i of sequence n goes to position ``lengths[n] + i``; a position without a page is
    left out.  A page that is written to must stand once in all of ``block_table``.
    """
    _no_grad_only("kv_pages_write", k, v, k_pages, v_pages)
    dev = _device(k, v)
    (k, k_ld), (v, v_ld) = _tokens("k", k, 4), _tokens("v", v, 4)
    if k.shape != v.shape:
        raise ValueError(f"shape mismatch: k{tuple(k.shape)} v{tuple(v.shape)}")
    B, T, Hkv, D = k.shape
    cu, N = (None, B) if cu_seqlens is None else _cu_seqlens(cu_seqlens, B, T, dev)
    table, lengths, pages, page = _cache(dev, k_pages, v_pages, block_table, lengths, N, Hkv, D)
    ws_bytes = _workspace_bytes("omx_gdn_kv_write_workspace_size", T, 0 if cu is None else N)
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_kv_write", _ptr(k), _ptr(v), k_ld, v_ld, _ptr(cu), N, _ptr(k_pages), _ptr(v_pages),
          pages, page, _ptr(table), table.shape[1], _ptr(lengths), B, T, Hkv, D, _ptr(ws), ws_bytes)


def attention_prefill_paged(q, k_pages, v_pages, block_table, lengths, *, cu_seqlens=None, scale=None):
    """Attention of new tokens over a paged cache that already holds their keys and values.

    q [B,T,Hq,D] bf16, N = B sequences of T new tokens or N packed by ``cu_seqlens`` (B == 1).
    Query i of sequence n attends positions 0 .. ``lengths[n] + i``.  Returns o [B,T,Hq,D] bf16,
    zeros for a query that no key is left for.
    """
    _no_grad_only("attention_prefill_paged", q, k_pages, v_pages)
    dev = _device(q)
    q, q_ld = _tokens("q", q, 4)
    B, T, Hq, D = q.shape
    N = B
    if cu_seqlens is not None:
        cu_seqlens, N = _cu_seqlens(cu_seqlens, B, T, dev)
    Hkv = k_pages.shape[2] if k_pages.dim() == 4 else 0
    table, lengths, pages, page = _cache(dev, k_pages, v_pages, block_table, lengths, N, Hkv, D)
    o = torch.empty((B, T, Hq, D), dtype=torch.bfloat16, device=dev)
    ws_bytes = _workspace_bytes("omx_gdn_attn_paged_workspace_size", B, T, Hq, Hkv, D, N, int(cu_seqlens is not None),
                                                            page, table.shape[1])
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_attn_paged", _ptr(q), q_ld, _ptr(cu_seqlens), N, _ptr(k_pages), _ptr(v_pages), pages,
          page, _ptr(table), table.shape[1], _ptr(lengths), _ptr(o), B, T, Hq, Hkv, D, _scale(scale, D),
          _ptr(ws), ws_bytes)
    return o


def attention_decode_step(q, k, v, k_pages, v_pages, block_table, lengths, *, scale=None):
    """One new token per sequence: writes its key and value to the cache in place and attends.

    q [B,Hq,D], k and v [B,Hkv,D] bf16.  The token goes to position ``lengths[b]`` and attends
    positions 0 .. ``lengths[b]``.  Returns out [B,Hq,D] bf16.
    """
    _no_grad_only("attention_decode_step", q, k, v, k_pages, v_pages)
    dev, q, k, v, q_ld, k_ld, v_ld, _, B = _qkv(q, k, v, None, dims=3)
    Hq, D = q.shape[1:]
    Hkv = k.shape[1]
    table, lengths, pages, page = _cache(dev, k_pages, v_pages, block_table, lengths, B, Hkv, D)
    out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=dev)
    ws_bytes = _workspace_bytes("omx_gdn_attn_decode_workspace_size", B, Hq, Hkv, D, page, table.shape[1])
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_attn_decode_step", _ptr(q), _ptr(k), _ptr(v), q_ld, k_ld, v_ld, _ptr(k_pages),
          _ptr(v_pages), pages, page, _ptr(table), table.shape[1], _ptr(lengths), _ptr(out), B, Hq, Hkv, D,
          _scale(scale, D), _ptr(ws), ws_bytes)
    return out
