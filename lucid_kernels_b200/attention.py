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

The checks of a call depend on shapes, strides, types and options only, and so does the descriptor the C entry point
takes: both are done once per combination and kept (``_plans``); a decoding step on the device takes a few microseconds,
less than the checks do.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _cabi
from .cute.forward_sub_interface import _CHECK_DEFAULT

__all__ = ["window_attention", "LUCIDWindowAttention", "paged_append", "paged_window_attention", "paged_lucid_attention",
           "_window_attention_fwd", "_window_attention_bwd"]

_D = 128
_DTYPES = (torch.float16, torch.bfloat16)
_raw_stream = torch._C._cuda_getCurrentRawStream
_device_now = torch._C._cuda_getDevice
_grad_enabled = torch.is_grad_enabled
_empty, _empty_like, _uint8 = torch.empty, torch.empty_like, torch.uint8
_increment_version = torch.autograd.graph.increment_version


def _new_like(t: torch.Tensor) -> torch.Tensor:
    return _empty_like(t) if t.is_contiguous() else _empty_like(t, memory_format=torch.contiguous_format)


def _refuse_tangents(name: str, *tensors) -> None:
    """The kernels see values only: a forward-mode tangent (whose tensor need not require a gradient) would be lost."""
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


class _Plan:
    """What a call's shapes, strides, types and options determine."""
    __slots__ = ("desc", "ref", "device", "copy", "empty", "workspace", "rest", "out_shape", "lse_shape")

    def __init__(self, desc, device: int, copy: bool, empty: bool):
        self.desc, self.ref = desc, ctypes.byref(desc)
        self.device = device
        self.copy = copy          # some tensor's strides have no tensor map: work on contiguous copies
        self.empty = empty        # nothing to launch


_plans: dict = {}
_MAX_PLANS = 4096


def _keep(key, plan: _Plan) -> _Plan:
    if len(_plans) >= _MAX_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _good_strides(t: torch.Tensor) -> bool:
    """The kernels read 16-byte pieces of rows whose last dimension is contiguous; a tensor expanded along a dimension is
    materialised, like one with other strides."""
    return t.stride(-1) == 1 and all(n <= 1 or (s % 8 == 0 and s > 0) for s, n in zip(t.stride()[:-1], t.shape[:-1]))


def _usable(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None or (_good_strides(t) and t.data_ptr() % 16 == 0):
        return t
    return t.detach().clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """Element strides of all but the last dimension (of a dimension of extent 1: any valid one)."""
    st = [s if n > 1 else _D for s, n in zip(t.stride()[:-1], t.shape[:-1])]
    return (ctypes.c_int64 * len(st))(*st)


def _contiguous_strides(*shape):
    st = [_D]
    for n in shape[:0:-1]:
        st.insert(0, st[0] * n)
    return (ctypes.c_int64 * len(st))(*st)




def _scale(scale: Optional[float]) -> float:
    scale = 1.0 / math.sqrt(_D) if scale is None else float(scale)
    assert 0.0 < scale < 1e18, "scale must be positive and finite"
    return scale


def _check_vector(t: torch.Tensor, n: int, device, name: str) -> None:
    assert t.dtype == torch.int32 and t.shape == (n,), f"{name} must be an int32 tensor of shape ({n},)"
    assert t.device == device, f"{name} must be on {device}"


def _window(window: Optional[int], sinks: int):
    """(window or -1, sinks) as the C entry points take them."""
    sinks = int(sinks)
    assert sinks >= 0, "sinks must be a non-negative number of positions"
    if window is None:
        return -1, 0
    window = int(window)
    assert window >= 0, "window must be None or a non-negative number of positions"
    return min(window, 1 << 30), min(sinks, 1 << 30)


def _plain_options(window, sinks, scale):
    """Options as hashable numbers (a tensor's hash is its identity)."""
    return (window if window is None or type(window) is int else int(window), sinks if type(sinks) is int else int(sinks),
            scale if scale is None or type(scale) is float else float(scale))


# ---------------------------------------------------------------------------------------------------------------------
# window attention
# ---------------------------------------------------------------------------------------------------------------------
def _window_plan(key, q, k, v, out, dout, window, sinks, scale, lengths) -> _Plan:
    """Checks a forward (out, dout None) or backward call and describes it."""
    w, s = _window(window, sinks)
    assert q.dim() == 4 and k.dim() == 4, "q and k must be (batch, seqlen, heads, head_dim)"
    B, Nq, Hq, D = q.shape
    _, Nk, Hkv, _ = k.shape
    others = [t for t in (out, dout) if t is not None]
    assert D == _D, f"this build supports head_dim == {_D}, got {D}"
    assert k.shape == (B, Nk, Hkv, D) and v.shape == k.shape, "k and v must share their shape, and q's batch and head_dim"
    assert Hkv > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of key heads ({Hkv})"
    assert Nq <= Nk, f"more queries ({Nq}) than keys ({Nk})"
    assert all(t.shape == q.shape for t in others), "out and its gradient must have q's shape"
    assert q.dtype in _DTYPES, "inputs must be float16 or bfloat16"
    assert all(t.dtype == q.dtype for t in (k, v, *others)), "all tensors must have the same dtype"
    assert q.is_cuda and all(t.device == q.device for t in (k, v, *others)), "inputs must be on one CUDA device"
    assert s <= 128, f"at most 128 first positions stay visible, got {s}"
    copy = not all(_good_strides(t) for t in (q, k, v, *others))
    if lengths is not None:
        _check_vector(lengths, B, q.device, "lengths")
        copy = copy or not lengths.is_contiguous()
    desc = _cabi.WindowAttnDesc(B, Nq, Nk, Hq, Hkv, D, _cabi.dtype_code(q.dtype), w, s, _scale(scale))
    like_q, like_k = _contiguous_strides(B, Nq, Hq), _contiguous_strides(B, Nk, Hkv)
    desc.q_strides, desc.k_strides, desc.v_strides = _strides(q), _strides(k), _strides(v)
    desc.out_strides = like_q if out is None else _strides(out)
    desc.dout_strides = like_q if dout is None else _strides(dout)
    desc.dq_strides, desc.dk_strides, desc.dv_strides = like_q, like_k, like_k
    plan = _Plan(desc, q.get_device(), copy, q.numel() == 0)
    plan.out_shape, plan.lse_shape = (B, Nq, Hq, D), (B, Hq, Nq)
    plan.workspace = plan.rest = 0
    if not plan.empty:
        plan.rest = _cabi.load().lucid_window_attn_rest_bytes(plan.ref)
        if dout is not None:
            plan.workspace = _cabi.load().lucid_window_attn_bwd_workspace_bytes(plan.ref)
    return _keep(key, plan)


def _window_attention_fwd(q, k, v, window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None,
                          lengths: Optional[torch.Tensor] = None, *, training: bool = True, check: Optional[bool] = None):
    """(out, lse, rest): see ``window_attention``; ``lse`` (B, Hq, Nq) fp32, -inf for a query that sees nothing; ``rest``, what
    the rounding of ``out`` took off, opaque.  Both are for the backward and None unless ``training``."""
    window, sinks, scale = _plain_options(window, sinks, scale)
    key = ("window", q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(),
           v.dtype, v.get_device(), window, sinks, scale,
           None if lengths is None else (lengths.shape, lengths.stride(), lengths.dtype, lengths.get_device()))
    plan = _plans.get(key)
    if plan is None:
        plan = _window_plan(key, q, k, v, None, None, window, sinks, scale, lengths)
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if plan.copy or (qp | kp | vp) & 15:
        return _window_attention_fwd(_usable(q), _usable(k), _usable(v), window, sinks, scale,
                                     None if lengths is None else lengths.contiguous(), training=training, check=check)
    if _device_now() != plan.device:
        with torch.cuda.device(plan.device):
            return _window_attention_fwd(q, k, v, window, sinks, scale, lengths, training=training, check=check)
    out = _new_like(q)
    lse = rest = None
    if training:
        lse = _empty(plan.lse_shape, dtype=torch.float32, device=q.device)
        rest = _empty(plan.rest, dtype=_uint8, device=q.device)
    if plan.empty:
        return out, lse, rest
    stream = _raw_stream(plan.device)
    rc = _cabi.load().lucid_window_attn_fwd(plan.ref, qp, kp, vp, out.data_ptr(), None if rest is None else rest.data_ptr(),
                                            None if lse is None else lse.data_ptr(),
                                            None if lengths is None else lengths.data_ptr(), stream)
    if rc:
        _cabi.check_rc(rc, "lucid_window_attn_fwd")
    if check or (check is None and _CHECK_DEFAULT):
        _cabi.raise_on_attention_error(stream, "_window_attention_fwd")
    return out, lse, rest


def _window_attention_bwd(q, k, v, out, lse, rest, dout, window: Optional[int] = None, sinks: int = 0,
                          scale: Optional[float] = None, lengths: Optional[torch.Tensor] = None, *, need_dq: bool = True,
                          need_dkv: bool = True, check: Optional[bool] = None):
    """(dq, dk, dv) from the forward's ``out``, ``lse`` and ``rest`` (None: a less accurate delta); None for what is not needed."""
    window, sinks, scale = _plain_options(window, sinks, scale)
    key = ("window bwd", q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(),
           v.dtype, v.get_device(), out.shape, out.stride(), out.dtype, out.get_device(), dout.shape, dout.stride(), dout.dtype,
           dout.get_device(), window, sinks, scale,
           None if lengths is None else (lengths.shape, lengths.stride(), lengths.dtype, lengths.get_device()))
    plan = _plans.get(key)
    if plan is None:
        plan = _window_plan(key, q, k, v, out, dout, window, sinks, scale, lengths)
    qp, kp, vp, op, gp = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr()
    if plan.copy or (qp | kp | vp | op | gp) & 15:
        return _window_attention_bwd(*(_usable(t) for t in (q, k, v, out)), lse, rest, _usable(dout), window, sinks, scale,
                                     None if lengths is None else lengths.contiguous(), need_dq=need_dq, need_dkv=need_dkv, check=check)
    assert lse.shape == plan.lse_shape and lse.dtype == torch.float32 and lse.device == q.device and lse.is_contiguous(), \
        "lse must be the forward's"
    assert rest is None or (rest.numel() == plan.rest and rest.dtype == _uint8 and rest.device == q.device and rest.is_contiguous()), \
        "rest must be the forward's"
    if _device_now() != plan.device:
        with torch.cuda.device(plan.device):
            return _window_attention_bwd(q, k, v, out, lse, rest, dout, window, sinks, scale, lengths, need_dq=need_dq, need_dkv=need_dkv,
                                         check=check)
    dq = _new_like(q) if need_dq else None
    dk, dv = (_new_like(t) if need_dkv else None for t in (k, v))
    if plan.empty:
        return dq, dk if dk is None else dk.zero_(), dv if dv is None else dv.zero_()
    ws = _empty(plan.workspace, dtype=_uint8, device=q.device)
    stream = _raw_stream(plan.device)
    rc = _cabi.load().lucid_window_attn_bwd(plan.ref, qp, kp, vp, op, None if rest is None else rest.data_ptr(), lse.data_ptr(), gp, None if dq is None else dq.data_ptr(),
                                            None if dk is None else dk.data_ptr(), None if dv is None else dv.data_ptr(),
                                            None if lengths is None else lengths.data_ptr(), ws.data_ptr(), plan.workspace, stream)
    if rc:
        _cabi.check_rc(rc, "lucid_window_attn_bwd")
    if check or (check is None and _CHECK_DEFAULT):
        _cabi.raise_on_attention_error(stream, "_window_attention_bwd")
    return dq, dk, dv


class LUCIDWindowAttention(torch.autograd.Function):
    """``out = LUCIDWindowAttention.apply(q, k, v, window, sinks, scale, lengths)``, all in BSHD layout."""

    @staticmethod
    def forward(ctx, q, k, v, window=None, sinks=0, scale=None, lengths=None):
        out, lse, rest = _window_attention_fwd(q, k, v, window, sinks, scale, lengths)
        ctx.save_for_backward(q, k, v, out, lse, rest, lengths)
        ctx.args = (window, sinks, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, rest, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv = _window_attention_bwd(q, k, v, out, lse, rest, dout, *ctx.args, lengths, need_dq=need[0],
                                           need_dkv=need[1] or need[2])
        return dq, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                     scale: Optional[float] = None, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over the last ``window`` positions (the query's own among them) and the first ``sinks``.

    q (B, Nq, Hq, 128); k, v (B, Nk, Hkv, 128); Hq a multiple of Hkv, Nq <= Nk, any sizes and strides.  The queries are the
    last Nq positions: query i sits at ``p = i + Nk - Nq`` and sees key j when ``j <= p and (j > p - window or j < sinks)``.
    ``window=None``: every key up to p.  ``sinks`` <= 128.  ``scale``: of the scores, 128 ** -0.5 by default.  ``lengths``
    (int32, (B,), on the device): positions from ``lengths[b]`` on are padding, neither keys nor queries, whatever they
    hold; their outputs and gradients are 0.  So are a query's that sees nothing.  Values at positions inside a sequence
    must be finite.

    For the backward a call keeps, besides its inputs and the result, a second tensor of the result's size (what the result's
    rounding took off; Nq above 128 counts in whole blocks of 128) and 4 bytes per query and head.

    In fp16 the gradient of a score, weight * (dout.v - dout.out), is rounded where it stands: below 2^-14 it loses bits and above
    65504 it overflows, as fp16 training does elsewhere - scale the loss accordingly.  bf16 has fp32's range.

    Differentiable in q, k and v (once, in reverse mode; forward-mode tangents are refused); gradients come out the same on every run.  In a training step recorded into a CUDA
    graph, record forward and backward together and, as torch asks for every operator, keep no eager graph of the same
    leaves alive while recording."""
    _refuse_tangents("window_attention", q, k, v)
    if _grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return LUCIDWindowAttention.apply(q, k, v, window, sinks, scale, lengths)
    return _window_attention_fwd(q, k, v, window, sinks, scale, lengths, training=False)[0]


# ---------------------------------------------------------------------------------------------------------------------
# paged cache
# ---------------------------------------------------------------------------------------------------------------------
def _cache_desc(k_cache, v_cache, block_table, B: int, tensors):
    """(descriptor, whether the block table has to be copied)"""
    assert k_cache.dim() == 4 and k_cache.shape[3] == _D, f"caches must be (pages, page_size, heads, {_D})"
    assert v_cache.shape == k_cache.shape, "k_cache and v_cache must share their shape"
    pages, page, Hkv, _ = k_cache.shape
    assert k_cache.dtype in _DTYPES, "caches must be float16 or bfloat16"
    assert v_cache.dtype == k_cache.dtype and all(t.dtype == k_cache.dtype for t in tensors), "all tensors must have the caches' dtype"
    assert k_cache.is_cuda and all(t.device == k_cache.device for t in (v_cache, block_table, *tensors)), \
        "caches, block table and inputs must be on one CUDA device"
    assert pages > 0 and 0 < page <= 65536 and page & (page - 1) == 0, f"page_size must be a power of two up to 65536, got {page}"
    # (written in place: no copy can stand in for it)
    assert _good_strides(k_cache) and _good_strides(v_cache), \
        "caches must have a contiguous last dimension and strides that are multiples of 8"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B and block_table.shape[1] > 0, \
        f"block_table must be an int32 tensor of shape ({B}, pages per sequence)"
    width = block_table.shape[1]
    assert width * page <= 1 << 30, "block_table covers more than 2 ** 30 positions"
    copy = (width > 1 and block_table.stride(1) != 1) or (B > 1 and block_table.stride(0) < width)
    return _cabi.PagedCacheDesc(pages, page, width, width if B == 1 else block_table.stride(0), _strides(k_cache), _strides(v_cache)), copy


_NO_BACKWARD = "the cache operators have no backward: use torch.no_grad()"


def _cache_pointers(k_cache, v_cache):
    kc, vc = k_cache.data_ptr(), v_cache.data_ptr()
    assert (kc | vc) & 15 == 0, "caches must be 16-byte aligned"
    return kc, vc


def _append_plan(key, k, v, k_cache, v_cache, block_table, cache_lens, cu_seqlens, q, inv_freq, interleaved) -> _Plan:
    assert k.dim() == 3 and k.shape[2] == _D, f"k must be (tokens, heads, {_D})"
    T, Hkv, _ = k.shape
    assert cache_lens.dim() == 1, "cache_lens must be an int32 tensor of shape (batch,)"
    B = cache_lens.shape[0]
    cache, copy = _cache_desc(k_cache, v_cache, block_table, B, [t for t in (k, v, q) if t is not None])
    assert Hkv == k_cache.shape[2] and (v is None or v.shape == k.shape), "k and v must be (tokens, the caches' heads, head_dim)"
    assert q is None or (q.dim() == 3 and q.shape[0] == T and q.shape[2] == _D), "q must be (tokens, query heads, head_dim)"
    assert q is None or inv_freq is not None, "q is only rotated: it needs inv_freq"
    _check_vector(cache_lens, B, k.device, "cache_lens")
    copy = copy or not cache_lens.is_contiguous()
    if cu_seqlens is not None:
        _check_vector(cu_seqlens, B + 1, k.device, "cu_seqlens")
        copy = copy or not cu_seqlens.is_contiguous()
    else:
        assert T == B, f"without cu_seqlens there is one token per sequence, got {T} for {B}"
    rot = 0
    if inv_freq is not None:
        assert inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.device == k.device, "inv_freq must be an fp32 vector on the device"
        rot = 2 * inv_freq.numel()
        assert 0 < rot <= _D and rot % 16 == 0, f"inv_freq must rotate a multiple of 16 elements up to {_D}, got {rot}"
        copy = copy or not inv_freq.is_contiguous()
    copy = copy or not all(_good_strides(t) for t in (k, v, q) if t is not None)
    desc = _cabi.PagedAppendDesc(cache, B, T, 0 if q is None else q.shape[1], Hkv, _D, rot, int(interleaved), _cabi.dtype_code(k.dtype),
                                 _strides(k), _strides(k if v is None else v), _strides(k if q is None else q))
    return _keep(key, _Plan(desc, k.get_device(), copy, T == 0 or B == 0))


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
    _refuse_tangents("paged_append", k, v, q, k_cache, v_cache, inv_freq)
    key = ("append", k.shape, k.stride(), k.dtype, k.get_device(), None if v is None else (v.shape, v.stride(), v.dtype, v.get_device()),
           None if q is None else (q.shape, q.stride(), q.dtype, q.get_device()), k_cache.shape, k_cache.stride(), k_cache.dtype,
           k_cache.get_device(), v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.get_device(), block_table.shape,
           block_table.stride(), block_table.dtype, block_table.get_device(), cache_lens.shape, cache_lens.stride(), cache_lens.dtype,
           cache_lens.get_device(),
           None if cu_seqlens is None else (cu_seqlens.shape, cu_seqlens.stride(), cu_seqlens.dtype, cu_seqlens.get_device()),
           None if inv_freq is None else (inv_freq.shape, inv_freq.stride(), inv_freq.dtype, inv_freq.get_device()), bool(interleaved))
    plan = _plans.get(key)
    if plan is None:
        plan = _append_plan(key, k, v, k_cache, v_cache, block_table, cache_lens, cu_seqlens, q, inv_freq, interleaved)
    if _grad_enabled():
        assert not (k.requires_grad or (v is not None and v.requires_grad) or (q is not None and q.requires_grad) or
                    k_cache.requires_grad or v_cache.requires_grad or (inv_freq is not None and inv_freq.requires_grad)), _NO_BACKWARD
    kp, vp, qp = k.data_ptr(), None if v is None else v.data_ptr(), None if q is None else q.data_ptr()
    if plan.copy or (kp | (vp or 0) | (qp or 0)) & 15:
        own = lambda t: None if t is None else t.contiguous()
        return paged_append(_usable(k), _usable(v), k_cache, v_cache, own(block_table), own(cache_lens), own(cu_seqlens), _usable(q),
                            own(inv_freq), interleaved, check=check)
    kc, vc = _cache_pointers(k_cache, v_cache)
    if _device_now() != plan.device:
        with torch.cuda.device(plan.device):
            return paged_append(k, v, k_cache, v_cache, block_table, cache_lens, cu_seqlens, q, inv_freq, interleaved, check=check)
    q_out = None if q is None else _new_like(q)
    if plan.empty:
        return q_out if q_out is None else q_out.zero_()
    stream = _raw_stream(plan.device)
    rc = _cabi.load().lucid_paged_append(plan.ref, kp, vp, qp, None if q_out is None else q_out.data_ptr(), kc, vc, block_table.data_ptr(),
                                         cache_lens.data_ptr(), None if cu_seqlens is None else cu_seqlens.data_ptr(),
                                         None if inv_freq is None else inv_freq.data_ptr(), stream)
    if rc:
        _cabi.check_rc(rc, "lucid_paged_append")
    _increment_version([k_cache] if v is None else [k_cache, v_cache])
    if check or (check is None and _CHECK_DEFAULT):
        _cabi.raise_on_attention_error(stream, "paged_append")
    return q_out


def _step_plan(key, q, v, k_cache, v_cache, block_table, seq_lens, window, sinks, scale, k_scale) -> _Plan:
    """Checks a decoding step (``v`` and ``k_scale``: of a LUCID layer) and describes it."""
    w, s = _window(window, sinks)
    assert q.dim() == 3 and q.shape[2] == _D, f"q must be (batch, query heads, {_D})"
    B, Hq, _ = q.shape
    cache, copy = _cache_desc(k_cache, v_cache, block_table, B, [t for t in (q, v) if t is not None])
    Hkv = k_cache.shape[2]
    assert Hkv > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of key heads ({Hkv})"
    assert B <= 65535, "at most 65535 sequences in a call"
    _check_vector(seq_lens, B, q.device, "seq_lens")
    copy = copy or not seq_lens.is_contiguous() or not _good_strides(q)
    scale = _scale(scale)
    if v is not None:
        assert 0.0 < k_scale < 1e18, "k_scale must be positive and finite"
        assert v.shape == (B, Hkv, _D), f"v must be ({B}, {Hkv}, {_D})"
        assert Hq > 0, "a LUCID step needs query heads"       # (nothing would be launched, and the new row not written)
        assert Hq // Hkv <= 15, f"at most 15 query heads per key head, got {Hq // Hkv}"
        copy = copy or not _good_strides(v)
    desc = _cabi.PagedAttnDesc(cache, B, Hq, Hkv, _D, _cabi.dtype_code(q.dtype), w, s, scale, k_scale, _strides(q),
                               _strides(q if v is None else v))
    plan = _Plan(desc, q.get_device(), copy, q.numel() == 0)
    plan.workspace = 0 if plan.empty else _cabi.load().lucid_paged_attn_workspace_bytes(plan.ref, 0 if v is None else 1)
    return _keep(key, plan)


def paged_window_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                           seq_lens: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                           scale: Optional[float] = None, *, check: Optional[bool] = None) -> torch.Tensor:
    """One decoding step of ``window_attention`` over a paged cache: q (B, Hq, 128) is the query of position
    ``seq_lens[b] - 1`` (int32, (B,); its key has been appended), which sees the last ``window`` positions and the first
    ``sinks``.  Returns (B, Hq, 128); 0 where ``seq_lens[b]`` is 0."""
    _refuse_tangents("paged_window_attention", q, k_cache, v_cache)
    window, sinks, scale = _plain_options(window, sinks, scale)
    key = ("step", q.shape, q.stride(), q.dtype, q.get_device(), k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.get_device(),
           v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.get_device(), block_table.shape, block_table.stride(), block_table.dtype,
           block_table.get_device(), seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.get_device(), window, sinks, scale)
    plan = _plans.get(key)
    if plan is None:
        plan = _step_plan(key, q, None, k_cache, v_cache, block_table, seq_lens, window, sinks, scale, 1.0)
    if _grad_enabled():
        assert not (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad), _NO_BACKWARD
    qp = q.data_ptr()
    if plan.copy or qp & 15:
        return paged_window_attention(_usable(q), k_cache, v_cache, block_table.contiguous(), seq_lens.contiguous(), window, sinks, scale,
                                      check=check)
    kc, vc = _cache_pointers(k_cache, v_cache)
    if _device_now() != plan.device:
        with torch.cuda.device(plan.device):
            return paged_window_attention(q, k_cache, v_cache, block_table, seq_lens, window, sinks, scale, check=check)
    out = _new_like(q)
    if plan.empty:
        return out
    ws = _empty(plan.workspace, dtype=_uint8, device=q.device) if plan.workspace else None
    stream = _raw_stream(plan.device)
    rc = _cabi.load().lucid_paged_window_attn(plan.ref, qp, out.data_ptr(), kc, vc, block_table.data_ptr(), seq_lens.data_ptr(),
                                              None if ws is None else ws.data_ptr(), plan.workspace, stream)
    if rc:
        _cabi.check_rc(rc, "lucid_paged_window_attn")
    if check or (check is None and _CHECK_DEFAULT):
        _cabi.raise_on_attention_error(stream, "paged_window_attention")
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
    _refuse_tangents("paged_lucid_attention", q, v, k_cache, v_cache)
    _, _, scale = _plain_options(None, 0, scale)
    if type(k_scale) is not float:
        k_scale = float(k_scale)
    key = ("lucid step", q.shape, q.stride(), q.dtype, q.get_device(), v.shape, v.stride(), v.dtype, v.get_device(), k_cache.shape,
           k_cache.stride(), k_cache.dtype, k_cache.get_device(), v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.get_device(),
           block_table.shape, block_table.stride(), block_table.dtype, block_table.get_device(), seq_lens.shape, seq_lens.stride(),
           seq_lens.dtype, seq_lens.get_device(), scale, k_scale)
    plan = _plans.get(key)
    if plan is None:
        plan = _step_plan(key, q, v, k_cache, v_cache, block_table, seq_lens, None, 0, scale, k_scale)
    if _grad_enabled():
        assert not (q.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad), _NO_BACKWARD
    qp, vp = q.data_ptr(), v.data_ptr()
    if plan.copy or (qp | vp) & 15:
        return paged_lucid_attention(_usable(q), _usable(v), k_cache, v_cache, block_table.contiguous(), seq_lens.contiguous(), k_scale,
                                     scale, check=check)
    kc, vc = _cache_pointers(k_cache, v_cache)
    if _device_now() != plan.device:
        with torch.cuda.device(plan.device):
            return paged_lucid_attention(q, v, k_cache, v_cache, block_table, seq_lens, k_scale, scale, check=check)
    out = _new_like(q)
    if plan.empty:
        return out
    ws = _empty(plan.workspace, dtype=_uint8, device=q.device) if plan.workspace else None
    stream = _raw_stream(plan.device)
    rc = _cabi.load().lucid_paged_lucid_attn(plan.ref, qp, vp, out.data_ptr(), kc, vc, block_table.data_ptr(), seq_lens.data_ptr(),
                                             None if ws is None else ws.data_ptr(), plan.workspace, stream)
    if rc:
        _cabi.check_rc(rc, "lucid_paged_lucid_attn")
    _increment_version([v_cache])
    if check or (check is None and _CHECK_DEFAULT):
        _cabi.raise_on_attention_error(stream, "paged_lucid_attention")
    return out
