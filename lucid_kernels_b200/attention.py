"""Attention around the LUCID solve: sliding-window attention for prefill and training, the paged key/value cache, and
the single-token forms that read it.

``window_attention`` is softmax attention restricted to the last ``window`` positions with the first ``sinks`` positions
always visible (``window=None``: plain causal attention, e.g. on V' with ``scale=k_scale / sqrt(d)``), with its backward.
``paged_append`` writes new tokens' keys and values into a paged cache and applies the position rotation on the way;
``paged_window_attention`` is one decoding step of a window (or plain causal) layer over it; ``paged_lucid_attention`` is
one decoding step of a LUCID layer: the next row of the solve, and the attention on V'.

As with the solve: head dimension 128, fp16 or bf16, launched on torch's current stream of the tensors' device without
a host synchronisation, capturable into CUDA graphs; scratch memory comes from torch's allocator per call (calls on
different streams and captured graphs share none).  ``check=True`` (or ``LUCID_B200_CHECK=1``) synchronises and raises
``LucidKernelError`` if a kernel reported an error - a wait that ran out, a position whose page does not exist.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _cabi
from .cute.forward_sub_interface import _CHECK_DEFAULT

__all__ = ["window_attention", "LUCIDWindowAttention", "paged_append", "paged_window_attention", "paged_lucid_attention",
           "_window_attention_fwd", "_window_attention_bwd"]

_D = 128


def _usable(t: torch.Tensor) -> torch.Tensor:
    """The kernels read 16-byte pieces of rows whose last dimension is contiguous; a tensor expanded along a dimension is
    materialised, like one with other strides."""
    bad = t.stride(-1) != 1 or t.data_ptr() % 16 or any(n > 1 and (s % 8 or s == 0) for s, n in zip(t.stride()[:-1], t.shape[:-1]))
    return t.clone(memory_format=torch.contiguous_format) if bad else t


def _strides(t: torch.Tensor):
    """Element strides of all but the last dimension (of a dimension of extent 1: any valid one)."""
    st = [s if n > 1 else _D for s, n in zip(t.stride()[:-1], t.shape[:-1])]
    return (ctypes.c_int64 * len(st))(*st)


def _finish(check: Optional[bool], stream: int, what: str) -> None:
    if _CHECK_DEFAULT if check is None else check:
        _cabi.raise_on_attention_error(stream, what)


def _scale(scale: Optional[float]) -> float:
    scale = 1.0 / math.sqrt(_D) if scale is None else float(scale)
    assert 0.0 < scale < 1e18, "scale must be positive and finite"
    return scale


def _int32_vector(t: torch.Tensor, n: int, like: torch.Tensor, name: str) -> torch.Tensor:
    assert t.dtype == torch.int32 and t.shape == (n,), f"{name} must be an int32 tensor of shape ({n},)"
    assert t.device == like.device, f"{name} must be on {like.device}"
    return t.contiguous()


def _window(window: Optional[int], sinks: int):
    """(window or -1, sinks) as the C entry points take them."""
    sinks = int(sinks)
    assert sinks >= 0, "sinks must be a non-negative number of positions"
    if window is None:
        return -1, 0
    window = int(window)
    assert window >= 0, "window must be None or a non-negative number of positions"
    return min(window, 1 << 30), min(sinks, 1 << 30)


def _check_qkv(q, k, v, others, lengths, sinks):
    assert q.dim() == 4 and k.dim() == 4, "q and k must be (batch, seqlen, heads, head_dim)"
    B, Nq, Hq, D = q.shape
    _, Nk, Hkv, _ = k.shape
    assert D == _D, f"this build supports head_dim == {_D}, got {D}"
    assert k.shape == (B, Nk, Hkv, D) and v.shape == k.shape, "k and v must share their shape, and q's batch and head_dim"
    assert Hkv > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of key heads ({Hkv})"
    assert Nq <= Nk, f"more queries ({Nq}) than keys ({Nk})"
    assert all(t.shape == q.shape for t in others), "out and its gradient must have q's shape"
    assert q.dtype in (torch.float16, torch.bfloat16), "inputs must be float16 or bfloat16"
    assert all(t.dtype == q.dtype for t in (k, v, *others)), "all tensors must have the same dtype"
    assert q.is_cuda and all(t.device == q.device for t in (k, v, *others)), "inputs must be on one CUDA device"
    assert sinks <= 128, f"at most 128 first positions stay visible, got {sinks}"
    if lengths is not None:
        lengths = _int32_vector(lengths, B, q, "lengths")
    return lengths


def _window_attention_fwd(q, k, v, window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None,
                          lengths: Optional[torch.Tensor] = None, *, check: Optional[bool] = None):
    """(out, lse): see ``window_attention``; ``lse`` (B, Hq, Nq) fp32, -inf for a query that sees nothing."""
    w, s = _window(window, sinks)
    lengths = _check_qkv(q, k, v, (), lengths, s)
    scale = _scale(scale)
    q, k, v = (_usable(t.detach()) for t in (q, k, v))
    B, Nq, Hq, D = q.shape
    Nk, Hkv = k.shape[1:3]
    out = torch.empty((B, Nq, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, Hq, Nq), dtype=torch.float32, device=q.device)
    if out.numel() == 0:
        return out, lse
    lib = _cabi.load()
    with torch.cuda.device(q.device):
        stream = torch.cuda.current_stream().cuda_stream
        rc = lib.lucid_window_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                                       _strides(q), _strides(k), _strides(v), _strides(out), B, Nq, Nk, Hq, Hkv, D,
                                       _cabi.dtype_code(q.dtype), w, s, scale,
                                       None if lengths is None else lengths.data_ptr(), stream)
        _cabi.check_rc(rc, "lucid_window_attn_fwd")
        _finish(check, stream, "_window_attention_fwd")
    return out, lse


def _window_attention_bwd(q, k, v, out, lse, dout, window: Optional[int] = None, sinks: int = 0,
                          scale: Optional[float] = None, lengths: Optional[torch.Tensor] = None, *, need_dq: bool = True,
                          need_dkv: bool = True, check: Optional[bool] = None):
    """(dq, dk, dv) from the forward's ``out`` and ``lse``; None for what is not needed."""
    w, s = _window(window, sinks)
    lengths = _check_qkv(q, k, v, (out, dout), lengths, s)
    scale = _scale(scale)
    q, k, v, out, dout = (_usable(t.detach()) for t in (q, k, v, out, dout))
    B, Nq, Hq, D = q.shape
    Nk, Hkv = k.shape[1:3]
    assert lse.shape == (B, Hq, Nq) and lse.dtype == torch.float32 and lse.device == q.device, "lse must be the forward's"
    lse = lse.contiguous()
    dq = torch.empty((B, Nq, Hq, D), dtype=q.dtype, device=q.device) if need_dq else None
    dk = torch.empty((B, Nk, Hkv, D), dtype=q.dtype, device=q.device) if need_dkv else None
    dv = torch.empty_like(dk) if need_dkv else None
    if q.numel() == 0:
        return dq, dk if dk is None else dk.zero_(), dv if dv is None else dv.zero_()
    lib = _cabi.load()
    with torch.cuda.device(q.device):
        stream = torch.cuda.current_stream().cuda_stream
        nbytes = lib.lucid_window_attn_bwd_workspace_bytes(B, Nq, Nk, Hq, Hkv, w, s)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        sq, sk, sv = _strides(q), _strides(k), _strides(v)
        rc = lib.lucid_window_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                                       None if dq is None else dq.data_ptr(), None if dk is None else dk.data_ptr(),
                                       None if dv is None else dv.data_ptr(), sq, sk, sv, _strides(out), _strides(dout),
                                       sq if dq is None else _strides(dq), sk if dk is None else _strides(dk),
                                       sv if dv is None else _strides(dv), B, Nq, Nk, Hq, Hkv, D,
                                       _cabi.dtype_code(q.dtype), w, s, scale,
                                       None if lengths is None else lengths.data_ptr(), ws.data_ptr(), nbytes, stream)
        _cabi.check_rc(rc, "lucid_window_attn_bwd")
        _finish(check, stream, "_window_attention_bwd")
    return dq, dk, dv


class LUCIDWindowAttention(torch.autograd.Function):
    """``out = LUCIDWindowAttention.apply(q, k, v, window, sinks, scale, lengths)``, all in BSHD layout."""

    @staticmethod
    def forward(ctx, q, k, v, window=None, sinks=0, scale=None, lengths=None):
        out, lse = _window_attention_fwd(q, k, v, window, sinks, scale, lengths)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.args = (window, sinks, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv = _window_attention_bwd(q, k, v, out, lse, dout, *ctx.args, lengths, need_dq=need[0],
                                           need_dkv=need[1] or need[2])
        return dq, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                     scale: Optional[float] = None, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over the last ``window`` positions (the query's own among them) and the first ``sinks``.

    q (B, Nq, Hq, 128); k, v (B, Nk, Hkv, 128); Hq a multiple of Hkv, Nq <= Nk, any sizes and strides.  The queries are the
    last Nq positions: query i sits at ``p = i + Nk - Nq`` and sees key j when ``j <= p and (j > p - window or j < sinks)``.
    ``window=None``: every key up to p.  ``sinks`` <= 128.  ``scale``: of the scores, 128 ** -0.5 by default.  ``lengths``
    (int32, (B,), on the device): positions from ``lengths[b]`` on are padding, neither keys nor queries, whatever they
    hold; their outputs and gradients are 0.  So are a query's that sees nothing.

    Differentiable in q, k and v (once); gradients come out the same on every run.  In a training step recorded into a CUDA
    graph, record forward and backward together and, as torch asks for every operator, keep no eager graph of the same
    leaves alive while recording."""
    return LUCIDWindowAttention.apply(q, k, v, window, sinks, scale, lengths)


# ---------------------------------------------------------------------------------------------------------------------
# paged cache
# ---------------------------------------------------------------------------------------------------------------------
def _check_cache(k_cache, v_cache, block_table, B: int, tensors):
    assert k_cache.dim() == 4 and k_cache.shape[3] == _D, f"caches must be (pages, page_size, heads, {_D})"
    assert v_cache.shape == k_cache.shape, "k_cache and v_cache must share their shape"
    pages, page, Hkv, _ = k_cache.shape
    assert k_cache.dtype in (torch.float16, torch.bfloat16), "caches must be float16 or bfloat16"
    assert v_cache.dtype == k_cache.dtype and all(t.dtype == k_cache.dtype for t in tensors), "all tensors must have the caches' dtype"
    assert k_cache.is_cuda and all(t.device == k_cache.device for t in (v_cache, block_table, *tensors)), \
        "caches, block table and inputs must be on one CUDA device"
    assert pages > 0 and 0 < page <= 65536 and page & (page - 1) == 0, f"page_size must be a power of two up to 65536, got {page}"
    for t in (k_cache, v_cache):
        # written in place: no copy can stand in for it
        assert t.stride(3) == 1 and t.data_ptr() % 16 == 0 and \
            all(n == 1 or (s % 8 == 0 and s > 0) for s, n in zip(t.stride()[:3], t.shape[:3])), \
            "caches must have a contiguous last dimension, a 16-byte aligned base and strides that are multiples of 8"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B and block_table.shape[1] > 0, \
        f"block_table must be an int32 tensor of shape ({B}, pages per sequence)"
    assert block_table.shape[1] * page <= 1 << 30, "block_table covers more than 2 ** 30 positions"
    if torch.is_grad_enabled():
        assert not any(t.requires_grad for t in (k_cache, v_cache, *tensors)), "the cache operators have no backward: use torch.no_grad()"
    if block_table.stride(1) != 1 or (B > 1 and block_table.stride(0) < block_table.shape[1]):
        block_table = block_table.contiguous()
    c = _cabi.PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), _strides(k_cache), _strides(v_cache), block_table.data_ptr(),
                         block_table.stride(0), block_table.shape[1], pages, page)
    return c, block_table


def paged_append(k: torch.Tensor, v: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_table: torch.Tensor, cache_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                 q: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False, *,
                 check: Optional[bool] = None) -> Optional[torch.Tensor]:
    """Append new tokens to a paged cache, rotating keys (and ``q``) by their position on the way.

    k, v (T, Hkv, 128): the tokens of all sequences one after another, sequence b's from ``cu_seqlens[b]`` to
    ``cu_seqlens[b + 1]`` (int32, (B + 1,)); without ``cu_seqlens`` one token per sequence, T == B.  Token i of sequence b goes
    to position ``cache_lens[b] + i`` (cache_lens int32, (B,), not changed), which is row ``position % page_size`` of page
    ``block_table[b, position // page_size]`` of the pools (pages, page_size, Hkv, 128).  ``v=None`` writes keys only.

    ``inv_freq`` (fp32, r / 2 values, r a multiple of 16 up to 128): the first r elements of every key head are rotated by
    ``position * inv_freq``, in pairs (i, i + r / 2), or (2i, 2i + 1) if ``interleaved``; the angle is formed in 64 bits.  q
    (T, Hq, 128) is rotated likewise and returned as a new tensor.  Tokens behind ``cu_seqlens[-1]`` are padding: nothing is
    written for them, their rows of the returned queries are 0.  A position without a page is skipped and reported."""
    tensors = [t for t in (k, v, q) if t is not None]
    assert k.dim() == 3 and k.shape[2] == _D, f"k must be (tokens, heads, {_D})"
    T, Hkv, _ = k.shape
    B = cache_lens.shape[0] if cache_lens.dim() == 1 else -1
    c, block_table = _check_cache(k_cache, v_cache, block_table, B, tensors)
    assert Hkv == k_cache.shape[2] and (v is None or v.shape == k.shape), "k and v must be (tokens, the caches' heads, head_dim)"
    assert q is None or (q.dim() == 3 and q.shape[0] == T and q.shape[2] == _D), "q must be (tokens, query heads, head_dim)"
    assert q is None or inv_freq is not None, "q is only rotated: it needs inv_freq"
    cache_lens = _int32_vector(cache_lens, B, k, "cache_lens")
    if cu_seqlens is not None:
        cu_seqlens = _int32_vector(cu_seqlens, B + 1, k, "cu_seqlens")
    else:
        assert T == B, f"without cu_seqlens there is one token per sequence, got {T} for {B}"
    rot = 0
    if inv_freq is not None:
        assert inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.device == k.device, "inv_freq must be an fp32 vector on the device"
        rot = 2 * inv_freq.numel()
        assert 0 < rot <= _D and rot % 16 == 0, f"inv_freq must rotate a multiple of 16 elements up to {_D}, got {rot}"
        inv_freq = inv_freq.contiguous()
    k, v, q = (None if t is None else _usable(t.detach()) for t in (k, v, q))
    q_out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if T == 0 or B == 0:
        return q_out if q_out is None else q_out.zero_()
    lib = _cabi.load()
    ptr = lambda t: None if t is None else t.data_ptr()
    with torch.cuda.device(k.device):
        stream = torch.cuda.current_stream().cuda_stream
        st = _strides(k)
        rc = lib.lucid_paged_append(ptr(k), ptr(v), ptr(q), ptr(q_out), st, st if v is None else _strides(v),
                                    st if q is None else _strides(q), ctypes.byref(c), ptr(cache_lens), ptr(cu_seqlens),
                                    ptr(inv_freq), B, T, 0 if q is None else q.shape[1], Hkv, _D, rot, int(interleaved),
                                    _cabi.dtype_code(k.dtype), stream)
        _cabi.check_rc(rc, "lucid_paged_append")
        torch.autograd.graph.increment_version([k_cache] if v is None else [k_cache, v_cache])
        _finish(check, stream, "paged_append")
    return q_out


def _check_step(q, k_cache, v_cache, block_table, seq_lens, more=()):
    assert q.dim() == 3 and q.shape[2] == _D, f"q must be (batch, query heads, {_D})"
    B, Hq, _ = q.shape
    c, block_table = _check_cache(k_cache, v_cache, block_table, B, (q, *more))
    Hkv = k_cache.shape[2]
    assert Hkv > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of key heads ({Hkv})"
    assert B <= 65535, "at most 65535 sequences in a call"
    return c, block_table, _int32_vector(seq_lens, B, q, "seq_lens"), torch.empty((B, Hq, _D), dtype=q.dtype, device=q.device)


def paged_window_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                           seq_lens: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                           scale: Optional[float] = None, *, check: Optional[bool] = None) -> torch.Tensor:
    """One decoding step of ``window_attention`` over a paged cache: q (B, Hq, 128) is the query of position
    ``seq_lens[b] - 1`` (int32, (B,); its key has been appended), which sees the last ``window`` positions and the first
    ``sinks``.  Returns (B, Hq, 128); 0 where ``seq_lens[b]`` is 0."""
    w, s = _window(window, sinks)
    c, block_table, seq_lens, out = _check_step(q, k_cache, v_cache, block_table, seq_lens)
    scale = _scale(scale)
    q = _usable(q.detach())
    B, Hq, D = q.shape
    if out.numel() == 0:
        return out
    lib = _cabi.load()
    with torch.cuda.device(q.device):
        stream = torch.cuda.current_stream().cuda_stream
        nbytes = lib.lucid_paged_attn_workspace_bytes(B, Hq, k_cache.shape[2], c.page_rows, c.table_width, w, s, 0)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        rc = lib.lucid_paged_window_attn(q.data_ptr(), out.data_ptr(), _strides(q), ctypes.byref(c), seq_lens.data_ptr(), B, Hq,
                                         k_cache.shape[2], D, _cabi.dtype_code(q.dtype), w, s, scale, ws.data_ptr(), nbytes, stream)
        _cabi.check_rc(rc, "lucid_paged_window_attn")
        _finish(check, stream, "paged_window_attention")
    return out


def paged_lucid_attention(q: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          block_table: torch.Tensor, seq_lens: torch.Tensor, k_scale: float = 1.0,
                          scale: Optional[float] = None, *, check: Optional[bool] = None) -> torch.Tensor:
    """One decoding step of a LUCID layer: the solve's row n = ``seq_lens[b] - 1`` and the attention on V'.

    The caches hold the keys of positions 0 .. n (append them with ``v=None``) and V' of positions 0 .. n - 1 (of the prompt,
    from ``_forward_sub_fwd``; later ones from this call).  v (B, Hkv, 128) is the new token's value.  With
    ``t_j = k_scale ** 2 * k_n . k_j``, ``v'_n = exp(-t_n) v_n - sum_{j < n} exp(t_j - t_n) v'_j`` is written to position n of
    v_cache, and softmax attention with scores ``scale * q . k_j`` over j <= n of V' is returned, (B, Hq, 128).  At most 15
    query heads per key head.  ``seq_lens[b] = 0``: the row of the result is 0 and nothing is written."""
    c, block_table, seq_lens, out = _check_step(q, k_cache, v_cache, block_table, seq_lens, (v,))
    scale = _scale(scale)
    assert 0.0 < float(k_scale) < 1e18, "k_scale must be positive and finite"
    B, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    assert v.shape == (B, Hkv, D), f"v must be ({B}, {Hkv}, {D})"
    assert Hq // Hkv <= 15, f"at most 15 query heads per key head, got {Hq // Hkv}"
    q, v = _usable(q.detach()), _usable(v.detach())
    if out.numel() == 0:
        return out
    lib = _cabi.load()
    with torch.cuda.device(q.device):
        stream = torch.cuda.current_stream().cuda_stream
        nbytes = lib.lucid_paged_attn_workspace_bytes(B, Hq, Hkv, c.page_rows, c.table_width, -1, 0, 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        rc = lib.lucid_paged_lucid_attn(q.data_ptr(), v.data_ptr(), out.data_ptr(), _strides(q), _strides(v), ctypes.byref(c),
                                        seq_lens.data_ptr(), B, Hq, Hkv, D, _cabi.dtype_code(q.dtype), float(k_scale), scale,
                                        ws.data_ptr(), nbytes, stream)
        _cabi.check_rc(rc, "lucid_paged_lucid_attn")
        torch.autograd.graph.increment_version([v_cache])
        _finish(check, stream, "paged_lucid_attention")
    return out
