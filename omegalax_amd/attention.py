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

A cache in 8 bits has pages of float8_e4m3fn, and ``k_exps``, ``v_exps`` int8 [pages, page_size / 16,
Hkv]: the exponent e of each block of 16 tokens of a head, whose numbers c stand for c 2^e.  A ``window``
lets a query see that many last positions, its own among them, and the first ``sinks``; what none will see
again needs no page.
"""
from __future__ import annotations

import functools
import operator

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .deltanet import _cu_seqlens, _no_tangents, _ptr, _stream, _workspace

__all__ = ["attention_prefill", "attention_prefill_bwd", "attention_prefill_paged",
           "attention_decode_step", "kv_pages_assign", "kv_pages_release", "kv_pages_write"]


_BF16 = torch.bfloat16
_MOST = (1 << 31) - 1


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


def _sight(window, sinks):
    """(window, sinks) as whole numbers, or None for all keys.  The kernels count in 32 bits."""
    if window is None:
        if sinks:
            raise ValueError("sinks are the keys that stay visible behind a window: give one")
        return None
    window, sinks = operator.index(window), operator.index(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks not negative (got {window}, {sinks})")
    return min(window, _MOST), min(sinks, _MOST)


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


def _prefill_fwd(q, k, v, cu_seqlens, scale, sight, with_lse, with_rest):
    dev, q, k, v, q_ld, k_ld, v_ld, cu, N = _qkv(q, k, v, cu_seqlens)
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    o = torch.empty((B, T, Hq, D), dtype=torch.bfloat16, device=dev)
    lse = torch.empty((B, T, Hq), dtype=torch.float32, device=dev) if with_lse else None
    rest = torch.empty_like(o) if with_rest else None
    ws_bytes = _workspace_bytes("omx_gdn_attn_fwd_workspace_size", T, Hq, Hkv, 0 if cu is None else N)
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_attn_window_fwd" if sight else "omx_gdn_attn_fwd", _ptr(q), _ptr(k), _ptr(v), q_ld, k_ld,
          v_ld, _ptr(cu), N, _ptr(o), _ptr(lse), _ptr(rest), B, T, Hq, Hkv, D, _scale(scale, D), *(sight or ()),
          _ptr(ws), ws_bytes)
    return o, lse, rest


def attention_prefill_bwd(q, k, v, o, lse, do, *, o_rest=None, cu_seqlens=None, scale=None, window=None, sinks=0):
    """Gradients (dq, dk, dv) of ``attention_prefill`` for the cotangent ``do`` of its output.

    ``window`` and ``sinks`` are the forward's.  ``o`` and ``lse`` are what the forward returned with ``output_lse=True``.  ``o_rest``, what
    the rounding of o left (bf16, as o), makes dq and dk about 6% more exact; autograd keeps it.
    The gradients are dense bf16 tensors of the inputs' shapes; those of a key head are summed
    over its query heads.  A value of a sequence that is not finite may reach all of its gradients.
    """
    _no_tangents("attention_prefill_bwd", q, k, v, o, lse, do, o_rest)
    sight = _sight(window, sinks)
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
    name = "omx_gdn_attn_window_bwd" if sight else "omx_gdn_attn_bwd"
    ws_bytes = _workspace_bytes(name + "_workspace_size", B, T, Hq, Hkv, D, 0 if cu is None else N, *(sight or ()))
    ws = _workspace(ws_bytes, dev)
    _call(dev, name, _ptr(q), _ptr(k), _ptr(v), q_ld, k_ld, v_ld, _ptr(cu), N, _ptr(o), _ptr(lse), _ptr(o_rest),
          _ptr(do), _ptr(dq), _ptr(dk), _ptr(dv), B, T, Hq, Hkv, D, _scale(scale, D), *(sight or ()), _ptr(ws),
          ws_bytes)
    return dq, dk, dv


class _AttentionPrefill(torch.autograd.Function):
    """Autograd node of the prompt attention: forward omx_gdn_attn_fwd, backward omx_gdn_attn_bwd
    from the saved output and logarithms (no score is kept)."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale, sight):
        o, lse, rest = _prefill_fwd(q, k, v, cu_seqlens, scale, sight, True, True)
        ctx.save_for_backward(q, k, v, o, lse, rest, cu_seqlens)
        ctx.scale = scale
        ctx.window, ctx.sinks = sight or (None, 0)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _dlse):
        if do is None:
            return None, None, None, None, None, None
        q, k, v, o, lse, rest, cu_seqlens = ctx.saved_tensors
        dq, dk, dv = attention_prefill_bwd(q, k, v, o, lse, do, o_rest=rest, cu_seqlens=cu_seqlens,
                                           scale=ctx.scale, window=ctx.window, sinks=ctx.sinks)
        return dq, dk, dv, None, None, None


def attention_prefill(q, k, v, *, cu_seqlens=None, scale=None, output_lse=False, window=None, sinks=0):
    """Causal softmax attention of whole prompts.

    q [B,T,Hq,D], k and v [B,T,Hkv,D] bf16 (D a multiple of 8 up to 256; up to 32 query heads per
    key head; views into one projection are read in place).  ``cu_seqlens`` (int32 [N+1], B == 1)
    packs N sequences, as in ``gdn_prefill``.  With a ``window`` a query sees that many last keys, its
    own among them, and the first ``sinks`` of its sequence, which stay visible.  ``scale`` defaults to D ** -0.5.  Returns o
    [B,T,Hq,D] bf16, or (o, lse) with the fp32 logarithms [B,T,Hq] of the softmax sums.  When
    gradients are enabled and an input requires them, the call is recorded for autograd (once, and
    not through lse); forward-mode derivatives are refused.  A row sees no key after it, nor one behind
    its window, not even one that is not finite.
    """
    _no_tangents("attention_prefill", q, k, v)
    sight = _sight(window, sinks)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        o, lse = _AttentionPrefill.apply(q, k, v, cu_seqlens, scale, sight)
    else:
        o, lse, _ = _prefill_fwd(q, k, v, cu_seqlens, scale, sight, output_lse, False)
    return (o, lse) if output_lse else o


def _cache(dev, k_pages, v_pages, block_table, lengths, N, Hkv, D, k_exps=None, v_exps=None):
    """Checks of the cache's tensors, which are used where they lie."""
    dtype = _BF16
    if k_exps is not None or v_exps is not None:
        if k_exps is None or v_exps is None:
            raise ValueError("k_exps and v_exps go together")
        dtype = torch.float8_e4m3fn
        blocks = (k_pages.shape[0], k_pages.shape[1] // 16, Hkv) if k_pages.dim() == 4 else None
        for name, t in (("k_exps", k_exps), ("v_exps", v_exps)):
            if t.dtype is not torch.int8 or tuple(t.shape) != blocks or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"{name} must be int8 {blocks}, contiguous and on {dev} (got {t.dtype}, "
                                 f"{tuple(t.shape)} on {t.device})")
    for t in (k_pages, v_pages, block_table, lengths):
        if t.device != dev:
            _device(t)
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    shape = k_pages.shape
    if v_pages.shape != shape or len(shape) != 4 or shape[2] != Hkv or shape[3] != D:
        raise ValueError(f"k_pages and v_pages must both be [pages, page_size, {Hkv}, {D}] "
                         f"(got {tuple(shape)}, {tuple(v_pages.shape)})")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.dtype is not dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be {'bf16' if dtype is _BF16 else 'float8_e4m3fn'} and contiguous "
                             f"(got {t.dtype}{', without exponents' if t.dtype is torch.float8_e4m3fn else ''})")
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.shape[0] != N:
        raise ValueError(f"block_table must be int32 [{N}, width] (got {block_table.dtype}, "
                         f"{tuple(block_table.shape)})")
    if lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.shape[0] != N:
        raise ValueError(f"lengths must be int32 [{N}] (got {lengths.dtype}, {tuple(lengths.shape)})")
    return block_table.contiguous(), lengths.contiguous(), shape[0], shape[1]


def _variant(call, k_exps, v_exps, sight):
    """(the entry point, its workspace size's, its exponents' pointers, its window and sinks) of a call over a cache."""
    if k_exps is None and sight is None:
        return *_PLAIN[call], (), ()
    return *_WINDOW[call], (_ptr(k_exps), _ptr(v_exps)), sight or (0, 0)


_PLAIN = {"paged": ("omx_gdn_attn_paged", "omx_gdn_attn_paged_workspace_size"),
          "decode": ("omx_gdn_attn_decode_step", "omx_gdn_attn_decode_workspace_size")}
_WINDOW = {"paged": ("omx_gdn_attn_paged_window", "omx_gdn_attn_paged_window_workspace_size"),
           "decode": ("omx_gdn_attn_decode_window", "omx_gdn_attn_decode_window_workspace_size")}


def _no_grad_only(name, *ts):
    for t in ts:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name}: gradients through the cache are not supported")
    _no_tangents(name, *ts)


def kv_pages_write(k, v, k_pages, v_pages, block_table, lengths, *, cu_seqlens=None, k_exps=None, v_exps=None):
    """Appends new tokens' keys and values to a paged cache, in place.

    k, v [B,T,Hkv,D] bf16, N = B sequences of T tokens or N packed by ``cu_seqlens`` (B == 1).
    Token i of sequence n goes to position ``lengths[n] + i``; a position without a page is
    left out.  A page that is written to must stand once in all of ``block_table``.  With ``k_exps``
    and ``v_exps`` the cache is one in 8 bits, and a block's older tokens are rounded again when a new
    one is larger than its exponent allows for, which shorter ``lengths`` do not undo; rows from ``cu_seqlens[N]`` on are then left out.
    """
    _no_grad_only("kv_pages_write", k, v, k_pages, v_pages)
    dev = _device(k, v)
    (k, k_ld), (v, v_ld) = _tokens("k", k, 4), _tokens("v", v, 4)
    if k.shape != v.shape:
        raise ValueError(f"shape mismatch: k{tuple(k.shape)} v{tuple(v.shape)}")
    B, T, Hkv, D = k.shape
    cu, N = (None, B) if cu_seqlens is None else _cu_seqlens(cu_seqlens, B, T, dev)
    table, lengths, pages, page = _cache(dev, k_pages, v_pages, block_table, lengths, N, Hkv, D, k_exps, v_exps)
    ws_bytes = _workspace_bytes("omx_gdn_kv_write_workspace_size", T, 0 if cu is None else N)
    ws = _workspace(ws_bytes, dev)
    name, exps = ("omx_gdn_kv_write", ()) if k_exps is None else ("omx_gdn_kv_write8", (_ptr(k_exps), _ptr(v_exps)))
    _call(dev, name, _ptr(k), _ptr(v), k_ld, v_ld, _ptr(cu), N, _ptr(k_pages), _ptr(v_pages), *exps, pages, page,
          _ptr(table), table.shape[1], _ptr(lengths), B, T, Hkv, D, _ptr(ws), ws_bytes)


def attention_prefill_paged(q, k_pages, v_pages, block_table, lengths, *, cu_seqlens=None, scale=None, k_exps=None,
                            v_exps=None, window=None, sinks=0):
    """Attention of new tokens over a paged cache that already holds their keys and values.

    q [B,T,Hq,D] bf16, N = B sequences of T new tokens or N packed by ``cu_seqlens`` (B == 1).
    Query i of sequence n attends positions 0 .. ``lengths[n] + i``, with a ``window`` that many last
    ones and the first ``sinks``.  Returns o [B,T,Hq,D] bf16, zeros for a query that no key is left for.
    """
    _no_grad_only("attention_prefill_paged", q, k_pages, v_pages)
    sight = _sight(window, sinks)
    dev = _device(q)
    q, q_ld = _tokens("q", q, 4)
    B, T, Hq, D = q.shape
    N = B
    if cu_seqlens is not None:
        cu_seqlens, N = _cu_seqlens(cu_seqlens, B, T, dev)
    Hkv = k_pages.shape[2] if k_pages.dim() == 4 else 0
    table, lengths, pages, page = _cache(dev, k_pages, v_pages, block_table, lengths, N, Hkv, D, k_exps, v_exps)
    o = torch.empty((B, T, Hq, D), dtype=torch.bfloat16, device=dev)
    name, size, exps, sight = _variant("paged", k_exps, v_exps, sight)
    ws_bytes = _workspace_bytes(size, B, T, Hq, Hkv, D, N, int(cu_seqlens is not None), page, table.shape[1], *sight)
    ws = _workspace(ws_bytes, dev)
    _call(dev, name, _ptr(q), q_ld, _ptr(cu_seqlens), N, _ptr(k_pages), _ptr(v_pages), *exps, pages, page,
          _ptr(table), table.shape[1], _ptr(lengths), _ptr(o), B, T, Hq, Hkv, D, _scale(scale, D), *sight, _ptr(ws),
          ws_bytes)
    return o


def attention_decode_step(q, k, v, k_pages, v_pages, block_table, lengths, *, scale=None, k_exps=None, v_exps=None,
                          window=None, sinks=0):
    """One new token per sequence: writes its key and value to the cache in place and attends.

    q [B,Hq,D], k and v [B,Hkv,D] bf16.  The token goes to position ``lengths[b]`` and attends
    positions 0 .. ``lengths[b]``, with a ``window`` that many last ones and the first ``sinks``.  Of a
    cache in 8 bits it attends itself as the cache holds it.  Returns out [B,Hq,D] bf16.
    """
    _no_grad_only("attention_decode_step", q, k, v, k_pages, v_pages)
    sight = _sight(window, sinks)
    dev, q, k, v, q_ld, k_ld, v_ld, _, B = _qkv(q, k, v, None, dims=3)
    Hq, D = q.shape[1:]
    Hkv = k.shape[1]
    table, lengths, pages, page = _cache(dev, k_pages, v_pages, block_table, lengths, B, Hkv, D, k_exps, v_exps)
    out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=dev)
    name, size, exps, sight = _variant("decode", k_exps, v_exps, sight)
    ws_bytes = _workspace_bytes(size, B, Hq, Hkv, D, page, table.shape[1], *sight)
    ws = _workspace(ws_bytes, dev)
    _call(dev, name, _ptr(q), _ptr(k), _ptr(v), q_ld, k_ld, v_ld, _ptr(k_pages), _ptr(v_pages), *exps, pages, page,
          _ptr(table), table.shape[1], _ptr(lengths), _ptr(out), B, Hq, Hkv, D, _scale(scale, D), *sight, _ptr(ws),
          ws_bytes)
    return out


def _pages(block_table, lengths, free_pages, free_count):
    """Checks of what deals pages; the table and the stack are changed where they lie."""
    dev = _device(block_table, lengths, free_pages, free_count)
    rows, shape = lengths.shape, block_table.shape
    N = rows[0] if len(rows) == 1 else -1
    known = (("block_table", block_table, len(shape) == 2 and shape[0] == N, "[N, width]"),
             ("lengths", lengths, N >= 0, "[N]"), ("free_pages", free_pages, len(free_pages.shape) == 1, "[pages]"),
             ("free_count", free_count, free_count.shape == (1,), "[1]"))
    for name, t, ok, want in known:
        if t.dtype is not torch.int32 or not ok:
            raise ValueError(f"{name} must be int32 {want} (got {t.dtype}, {tuple(t.shape)})")
        if t is not lengths and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    return dev, N, lengths.contiguous()


def kv_pages_assign(block_table, lengths, new_tokens, free_pages, free_count, *, page_size, tokens):
    """Gives new tokens their pages, on the GPU and in place; what the appends and attention of a step take.

    ``new_tokens`` int32 [N]: how many more tokens each sequence gets behind its ``lengths[n]``.  Entries
    of ``block_table`` that they need and that name no page take one from the stack of free pages,
    ``free_pages`` int32 [pages] with the first ``free_count`` (int32 [1]) of them free, in order; others
    keep theirs.  ``tokens``: the most that there is room for, all sequences together.  Returns
    (cu_seqlens int32 [N + 1], positions int32 [tokens], slots int64 [tokens], missing int32 [1]): the packed
    tokens' offsets, their positions in their sequences, page * page_size + row of each (-1 past the last,
    and where there is no page), and how many pages the stack was short of.  A batch padded to ``tokens`` rows
    takes a last row of the table with a length of -1, as its rows behind the last token count as the last
    sequence's.
    """
    dev, N, lengths = _pages(block_table, lengths, free_pages, free_count)
    _device(block_table, new_tokens)
    if new_tokens.dtype is not torch.int32 or tuple(new_tokens.shape) != (N,):
        raise ValueError(f"new_tokens must be int32 [{N}] (got {new_tokens.dtype}, {tuple(new_tokens.shape)})")
    new_tokens = new_tokens.contiguous()
    T = operator.index(tokens)
    if T < 0:
        raise ValueError(f"tokens must not be negative (got {T})")
    cu, positions, missing = lengths.new_empty(N + 1), lengths.new_empty(T), lengths.new_empty(1)
    slots = lengths.new_empty(T, dtype=torch.int64)
    ws_bytes = _workspace_bytes("omx_gdn_pages_assign_workspace_size", N)
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_pages_assign", _ptr(block_table), N, block_table.shape[1], _ptr(lengths), _ptr(new_tokens),
          _ptr(free_pages), _ptr(free_count), free_pages.shape[0], operator.index(page_size), T, _ptr(cu),
          _ptr(positions), _ptr(slots), _ptr(missing), _ptr(ws), ws_bytes)
    return cu, positions, slots, missing


def kv_pages_release(block_table, lengths, free_pages, free_count, *, page_size, window=None, sinks=0):
    """Returns pages to the stack that ``kv_pages_assign`` takes them from, on the GPU and in place.

    Those wholly past the ``lengths[n]`` tokens that a sequence keeps (0: it has ended, all of them; negative:
    none), and with a ``window`` those whose positions its next token no longer sees, but for the first
    ``sinks``.  Their entries become -1.  A page that two rows share is to go back from one of them only.
    """
    dev, N, lengths = _pages(block_table, lengths, free_pages, free_count)
    window, sinks = _sight(window, sinks) or (0, 0)
    ws_bytes = _workspace_bytes("omx_gdn_pages_release_workspace_size", N, block_table.shape[1])
    ws = _workspace(ws_bytes, dev)
    _call(dev, "omx_gdn_pages_release", _ptr(block_table), N, block_table.shape[1], _ptr(lengths), _ptr(free_pages),
          _ptr(free_count), free_pages.shape[0], operator.index(page_size), window, sinks, _ptr(ws), ws_bytes)
