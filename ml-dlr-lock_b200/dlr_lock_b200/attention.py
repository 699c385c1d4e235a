"""Tensor-level entry points of the attention block of a locked decoder on a paged key-value cache.

* ``paged_plan``          - one step's bookkeeping: block tables and slots, on the device.
* ``qk_norm_rope``        - norm and rotation of query and key heads, differentiable.
* ``qk_norm_rope_append`` - the same for serving: keys and values go to their slots of the cache.
* ``paged_attention``     - attention of one new token per request over its pages.
* ``rope_tables``         - the cosines and sines that the rotation takes.

A cache is a pair of (pages, kv_heads, page tokens, dim) tensors, bf16 or fp16, with pages of 2^n tokens (16 or more); slot
``s`` is token ``s % page`` of page ``s // page``.  The host framework's decode loop, which the reference leaves in charge of
attention and cache, has no counterpart of these.

Every call is asynchronous on the current stream of the tensors' device, never synchronises, and can be captured in a CUDA
graph; workspaces are taken from torch's allocator per call, so that captured graphs share none.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .ops import EPS, _stream_ptr

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
MAX_REQUESTS = 8192                     # of one plan


class PagedPlan(NamedTuple):
    """What ``paged_plan`` returns: int32 tensors on the device."""
    slots: torch.Tensor                 # (rows) slot of each row's token, -1 for rows without one
    positions: torch.Tensor             # (rows) position of each row's token in its request, 0 for rows without one
    starts: torch.Tensor                # (requests + 1) first row of each request
    lengths: torch.Tensor               # (requests) tokens held after the step
    n_free: torch.Tensor                # (1) free pages after the step


def _all_tensors(what, *tensors):
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what} takes tensors, got {type(t).__name__}")


def _on_one_device(what, *tensors):
    device = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{what} runs on CUDA tensors only (there is no CPU path)")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")
    return device


def _int32(what, name, t, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"{what}: {name} has type {t.dtype}, expected int32")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be contiguous")


def _page_size(what, page_size):
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"{what}: pages have 2^n tokens, 16 or more, not {page_size}")


def _check_cache(what, k_cache, v_cache, dtype, kv_heads, dim, multiple):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"{what}: the caches must be (pages, kv_heads, page tokens, dim) tensors of one shape")
    if not (k_cache.dtype == v_cache.dtype == dtype):
        raise TypeError(f"{what}: the caches have types {k_cache.dtype} and {v_cache.dtype}, expected {dtype}")
    if k_cache.shape[1] != kv_heads or k_cache.shape[3] != dim:
        raise ValueError(f"{what}: the caches have shape {tuple(k_cache.shape)}, expected {kv_heads} heads of {dim}")
    _page_size(what, k_cache.shape[2])
    if k_cache.shape[0] * k_cache.shape[2] > 0x7fffffff:
        raise ValueError(f"{what}: the caches have more than 2^31 - 1 slots")
    for c in (k_cache, v_cache):
        if c.numel() and (c.stride(3) != 1 or any(s % multiple for s in c.stride()[:3]) or c.data_ptr() % (2 * multiple)):
            raise ValueError(f"{what}: the caches need a contiguous last dimension and strides of a multiple of {multiple} elements")


def _heads(t: torch.Tensor, multiple: int) -> torch.Tensor:
    """t if its rows can be read where they are, else a contiguous copy."""
    if t.stride(-1) == 1 and not any(s % multiple for s in t.stride()[:-1]) and t.data_ptr() % (2 * multiple) == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


# ---- plan -------------------------------------------------------------------------------------------------------------------
def paged_plan(lengths: torch.Tensor, new_tokens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               n_free: torch.Tensor, page_size: int, *, width: Optional[int] = 1, rows: Optional[int] = None,
               finished: Optional[torch.Tensor] = None, in_place: bool = False) -> PagedPlan:
    """Give every request its new tokens: pages off the stack of free ones, block-table entries, slots and positions.

    ``lengths`` (requests) tokens held, ``new_tokens`` (requests) tokens to come, ``block_table`` (requests, columns),
    ``free_pages`` (pages) a stack of which the first ``n_free`` (1) entries are free; all int32.  ``finished`` (requests,
    bool): these requests give their pages back first and start again from no tokens.  The batch has ``width`` rows per
    request (1: a decode step), or, with ``width=None``, one request behind the other in ``rows`` rows.

    ``block_table`` and ``free_pages`` are written in place; lengths and the count of free pages come back as new tensors,
    or, with ``in_place``, in those given.  A request is refused (its length comes back as it was, its rows have slot -1)
    when the table has no columns for its tokens, when they do not fit its rows, or when it needs pages and those asked for
    up to and including it are more than there are free.
    """
    what = "paged_plan"
    _all_tensors(what, lengths, new_tokens, block_table, free_pages, n_free)
    if lengths.dim() != 1 or block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError(f"{what}: expected lengths (requests), block_table (requests, columns), free_pages (pages)")
    n = lengths.shape[0]
    if n > MAX_REQUESTS:
        raise ValueError(f"{what}: {n} requests, at most {MAX_REQUESTS} are planned at once")
    _page_size(what, page_size)
    _int32(what, "lengths", lengths, (n,))
    _int32(what, "new_tokens", new_tokens, (n,))
    _int32(what, "free_pages", free_pages, free_pages.shape)
    _int32(what, "n_free", n_free, (1,))
    if block_table.dtype != torch.int32:
        raise TypeError(f"{what}: block_table has type {block_table.dtype}, expected int32")
    if block_table.shape[0] != n or (block_table.numel() and block_table.stride(1) != 1):
        raise ValueError(f"{what}: block_table must have a row for each of the {n} requests, with contiguous entries")
    if n > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError(f"{what}: the rows of block_table overlap")
    if free_pages.shape[0] * page_size > 0x7fffffff:
        raise ValueError(f"{what}: the cache has more than 2^31 - 1 slots")
    if finished is not None and (finished.dtype not in (torch.bool, torch.uint8) or finished.shape != (n,) or not finished.is_contiguous()):
        raise ValueError(f"{what}: finished must be a contiguous bool tensor of {n} entries")
    if (width is None) == (rows is None):
        if width is None or rows != width * n:
            raise ValueError(f"{what}: give width, or width=None and rows")
    if width is not None:
        if width < 1:
            raise ValueError(f"{what}: width is at least 1")
        rows = width * n
    if rows < 0 or rows > 0x7fffffff:
        raise ValueError(f"{what}: {rows} rows")
    device = _on_one_device(what, lengths, new_tokens, block_table, free_pages, n_free, finished)
    with torch.cuda.device(device):
        # one allocation: slots, positions, starts, lengths, count
        out = torch.empty(2 * rows + 2 * n + 2, dtype=torch.int32, device=device)
        slots, positions, starts, new_lengths, count = out.split([rows, rows, n + 1, n, 1])
        if in_place:
            new_lengths, count = lengths, n_free
        step = _lib.PlanStep(lengths.data_ptr(), new_tokens.data_ptr(), finished.data_ptr() if finished is not None else None,
                             block_table.data_ptr(), block_table.stride(0), free_pages.data_ptr(), n_free.data_ptr(),
                             slots.data_ptr(), positions.data_ptr(), starts.data_ptr(), new_lengths.data_ptr(), count.data_ptr(),
                             n, block_table.shape[1], free_pages.shape[0], page_size, width or 0, rows)
        _lib.check(_lib.load().dlrb200_paged_plan(ctypes.byref(step), _stream_ptr(device.index)), "dlrb200_paged_plan")
    return PagedPlan(slots, positions, starts, new_lengths, count)


# ---- norm and rotation ------------------------------------------------------------------------------------------------------
def rope_tables(inv_freq: torch.Tensor, positions: int, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin (positions, len(inv_freq)) fp32 of position x frequency, times ``scale`` (the attention factor of the
    scaled forms); angles are formed in 64 bits.  Any scaling for long contexts is a matter of the frequencies."""
    if inv_freq.dim() != 1 or positions < 0:
        raise ValueError("rope_tables takes the frequencies as a vector and a number of positions")
    angle = torch.arange(positions, dtype=torch.float64, device=inv_freq.device)[:, None] * inv_freq.double()
    return (angle.cos() * scale).float(), (angle.sin() * scale).float()


def _check_norm_rope(what, q, k, q_weight, k_weight, cos, sin, positions):
    _all_tensors(what, q, k, cos, sin, positions)
    if q.dim() < 2 or k.dim() != q.dim() or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"{what}: expected q (..., heads, dim) and k (..., kv_heads, dim), got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype not in _TYPES or k.dtype != q.dtype:
        raise TypeError(f"{what} takes bfloat16 or float16 heads of one type, got {q.dtype} and {k.dtype}")
    dim = q.shape[-1]
    if dim % 8 or not 0 < dim <= 256 or q.shape[-2] < 1 or k.shape[-2] < 1:
        raise ValueError(f"{what}: heads of {dim} (a multiple of 8 up to 256 is supported), {q.shape[-2]} and {k.shape[-2]} of them")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"{what}: cos and sin must be float32 tensors (positions, half) of one shape")
    if not (cos.is_contiguous() and sin.is_contiguous()) or cos.data_ptr() % 16 or sin.data_ptr() % 16:
        raise ValueError(f"{what}: cos and sin must be contiguous and 16-byte aligned")
    half = cos.shape[1]
    if half % 4 or 2 * half > dim:
        raise ValueError(f"{what}: the tables turn {2 * half} of {dim} values: a multiple of 8 up to the head's size is supported")
    if cos.shape[0] > 0x7fffffff:
        raise ValueError(f"{what}: too many positions")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: positions have type {positions.dtype}, expected int32 or int64")
    if positions.shape != q.shape[:-2]:
        raise ValueError(f"{what}: positions have shape {tuple(positions.shape)}, expected {tuple(q.shape[:-2])}")
    given = [w for w in (q_weight, k_weight) if w is not None]
    for w in given:
        if w.dtype not in (q.dtype, torch.float32) or w.dtype != given[0].dtype:
            raise TypeError(f"{what}: the weights have type {w.dtype}, expected {q.dtype} or float32 for both")
        if w.shape != (dim,):
            raise ValueError(f"{what}: the weights have shape {tuple(w.shape)}, expected {(dim,)}")
    return dim, half


def _vector(w):
    """A weight as the kernels read it: contiguous from a 16-byte boundary."""
    if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0):
        return w
    return w.clone(memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _flat(t: torch.Tensor) -> torch.Tensor:
    """(..., heads, dim) as (tokens, heads, dim), where it lies if that can be."""
    return _heads(t.reshape(-1, *t.shape[-2:]) if t.dim() != 3 else t, 4)


def _strides(t):
    return t.stride(0), t.stride(1)


def _forward_args(q, k, q_weight, k_weight, cos, sin, positions, q_out, k_out, eps, interleaved, v=None, slots=None, k_cache=None, v_cache=None):
    weight = q_weight if q_weight is not None else k_weight
    kc, vc = ((*c.stride()[:3],) if c is not None else (0, 0, 0) for c in (k_cache, v_cache))
    pages, page_size = (k_cache.shape[0], k_cache.shape[2]) if k_cache is not None else (0, 0)
    return _lib.NormRopeArgs(
        q.data_ptr(), k.data_ptr(), _ptr(v), *_strides(q), *_strides(k), *(_strides(v) if v is not None else (0, 0)),
        _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), q_out.data_ptr(), _ptr(k_out),
        _ptr(slots), _ptr(k_cache), _ptr(v_cache), *kc, *vc, q.shape[0], q.shape[1], k.shape[1], q.shape[2], cos.shape[1],
        cos.shape[0], pages, page_size, _TYPES[q.dtype], int(weight is not None and weight.dtype == torch.float32),
        int(positions.dtype == torch.int64), int(interleaved), eps)


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        with torch.cuda.device(q.device):
            q3, k3 = _flat(q), _flat(k)
            qw, kw = _vector(q_weight), _vector(k_weight)
            at = positions.reshape(-1).contiguous()
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
            if at.numel():
                args = _forward_args(q3, k3, qw, kw, cos, sin, at, q_out, k_out, eps, interleaved)
                _lib.check(_lib.load().dlrb200_qk_norm_rope(ctypes.byref(args), _stream_ptr(q.get_device())), "dlrb200_qk_norm_rope")
        # without a norm the gradient does not depend on the input
        ctx.save_for_backward(q if q_weight is not None else None, k if k_weight is not None else None, q_weight, k_weight, cos, sin, positions)
        ctx.eps, ctx.interleaved, ctx.shapes = eps, interleaved, (q.shape, k.shape)
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, q_grad, k_grad):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        device, dtype = q_grad.device, q_grad.dtype
        with torch.cuda.device(device):
            lib = _lib.load()
            dq, dk = (torch.empty(s, dtype=dtype, device=device) for s in ctx.shapes)
            dqw, dkw = (None if w is None else torch.empty(w.shape, dtype=w.dtype, device=device) for w in (q_weight, k_weight))
            gq, gk = _flat(q_grad), _flat(k_grad)
            q3, k3 = (None if t is None else _flat(t) for t in (q, k))
            qw, kw = _vector(q_weight), _vector(k_weight)
            at = positions.reshape(-1).contiguous()
            weight = qw if qw is not None else kw
            dim = gq.shape[2]
            workspace, need = None, 0
            if weight is not None:
                need = lib.dlrb200_qk_norm_rope_backward_workspace_bytes(dim)
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
            none = (0, 0)
            args = _lib.NormRopeGradArgs(
                _ptr(q3), _ptr(k3), gq.data_ptr(), gk.data_ptr(), *(_strides(q3) if q3 is not None else none),
                *(_strides(k3) if k3 is not None else none), *_strides(gq), *_strides(gk), _ptr(qw), _ptr(kw), cos.data_ptr(),
                sin.data_ptr(), at.data_ptr(), dq.data_ptr(), dk.data_ptr(), _ptr(dqw), _ptr(dkw), _ptr(workspace), need,
                gq.shape[0], gq.shape[1], gk.shape[1], dim, cos.shape[1], cos.shape[0], _TYPES[dtype],
                int(weight is not None and weight.dtype == torch.float32), int(at.dtype == torch.int64), int(ctx.interleaved), ctx.eps)
            _lib.check(lib.dlrb200_qk_norm_rope_backward(ctypes.byref(args), _stream_ptr(device.index)), "dlrb200_qk_norm_rope_backward")
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *, eps: float = EPS,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q`` (..., heads, dim) and ``k`` (..., kv_heads, dim), then the rotation by position; new
    tensors.

    ``q_weight`` and ``k_weight`` (dim), in the heads' type or fp32; None leaves that norm out.  ``cos`` and ``sin``
    (positions, half) fp32, see ``rope_tables``: the first 2 * half values of a head are turned, in pairs (i, i + half), or
    (2i, 2i + 1) with ``interleaved``; the rest passes through.  ``positions`` (...) int32 or int64; one outside the tables
    makes its row NaN.  fp32 throughout, rounded once.  Differentiable (once) in q, k and the weights.
    """
    what = "qk_norm_rope"
    _check_norm_rope(what, q, k, q_weight, k_weight, cos, sin, positions)
    if cos.requires_grad or sin.requires_grad:
        raise ValueError(f"{what}: the tables have no gradient")
    _on_one_device(what, q, k, q_weight, k_weight, cos, sin, positions)
    return _NormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor],
                        k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                        slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, eps: float = EPS,
                        interleaved: bool = False, return_keys: bool = False):
    """``qk_norm_rope`` for serving: keys, and ``v`` as it is, go to ``slots`` (...) int32 of the caches; returns the queries,
    and with ``return_keys`` the keys too (what the attention over a whole prompt takes).

    Rows whose slot is outside the caches (-1) are not stored; the others must name different slots.  No gradient.
    """
    what = "qk_norm_rope_append"
    _all_tensors(what, v, slots, k_cache, v_cache)
    dim, _ = _check_norm_rope(what, q, k, q_weight, k_weight, cos, sin, positions)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must be like k, {tuple(k.shape)} {k.dtype}")
    if slots.dtype != torch.int32 or slots.shape != positions.shape:
        raise ValueError(f"{what}: slots must be int32 of shape {tuple(positions.shape)}")
    _check_cache(what, k_cache, v_cache, q.dtype, k.shape[-2], dim, 4)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, q_weight, k_weight, k_cache, v_cache)):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    device = _on_one_device(what, q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache)
    with torch.cuda.device(device):
        q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=device) if return_keys else None
        at, to = positions.reshape(-1).contiguous(), slots.reshape(-1).contiguous()
        if at.numel():
            args = _forward_args(_flat(q), _flat(k), _vector(q_weight), _vector(k_weight), cos, sin, at, q_out, k_out, float(eps),
                                 interleaved, _flat(v), to, k_cache, v_cache)
            _lib.check(_lib.load().dlrb200_qk_norm_rope(ctypes.byref(args), _stream_ptr(device.index)), "dlrb200_qk_norm_rope")
    return (q_out, k_out) if return_keys else q_out


# ---- attention --------------------------------------------------------------------------------------------------------------
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one token per request: ``q`` (requests, heads, dim) over the first ``lengths`` (requests) tokens of each
    request's pages, (requests, heads, dim); zeros where the length is 0.

    ``block_table`` (requests, columns) and ``lengths`` int32.  ``heads`` is a multiple of the caches' heads, each of which
    serves that many neighbouring query heads; dim is 64, 96, 128 or 256.  ``scale`` is 1 / sqrt(dim) unless given.  Lengths
    are read on the device: a captured call follows them.  A table entry outside the caches counts as a page of zeros and
    is never followed.  Scores, softmax and sums are fp32.  No gradient.
    """
    what = "paged_attention"
    _all_tensors(what, q, k_cache, v_cache, block_table, lengths)
    if q.dim() != 3:
        raise ValueError(f"{what}: expected q (requests, heads, dim), got {tuple(q.shape)}")
    if q.dtype not in _TYPES:
        raise TypeError(f"{what} takes bfloat16 or float16 queries, got {q.dtype}")
    n, heads, dim = q.shape
    if dim not in (64, 96, 128, 256):
        raise ValueError(f"{what}: heads of {dim}: 64, 96, 128 and 256 are supported")
    kv_heads = k_cache.shape[1] if k_cache.dim() == 4 else 0
    _check_cache(what, k_cache, v_cache, q.dtype, kv_heads, dim, 8)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{what}: {heads} query heads on {kv_heads} heads of the caches")
    _int32(what, "lengths", lengths, (n,))
    if block_table.dtype != torch.int32:
        raise TypeError(f"{what}: block_table has type {block_table.dtype}, expected int32")
    if block_table.dim() != 2 or block_table.shape[0] != n or (block_table.numel() and block_table.stride(1) != 1):
        raise ValueError(f"{what}: block_table must have a row for each of the {n} requests, with contiguous entries")
    if block_table.shape[1] * k_cache.shape[2] > 1 << 30:
        raise ValueError(f"{what}: a request of more than 2^30 tokens")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    device = _on_one_device(what, q, k_cache, v_cache, block_table, lengths)
    with torch.cuda.device(device):
        lib = _lib.load()
        out = torch.empty(n, heads, dim, dtype=q.dtype, device=device)
        if n:
            need = lib.dlrb200_paged_attention_workspace_bytes(heads, kv_heads, dim)
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
            q = _heads(q, 2)
            args = _lib.PagedAttentionArgs(
                q.data_ptr(), *_strides(q), k_cache.data_ptr(), v_cache.data_ptr(), *k_cache.stride()[:3], *v_cache.stride()[:3],
                block_table.data_ptr(), block_table.stride(0), lengths.data_ptr(), out.data_ptr(), workspace.data_ptr(), need,
                n, heads, kv_heads, dim, block_table.shape[1], k_cache.shape[0], k_cache.shape[2], _TYPES[q.dtype],
                1.0 / math.sqrt(dim) if scale is None else float(scale))
            _lib.check(lib.dlrb200_paged_attention(ctypes.byref(args), _stream_ptr(device.index)), "dlrb200_paged_attention")
    return out
