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
graph; workspaces are taken from torch's allocator per call, so that captured graphs share none.  Forward-mode tangents are
refused.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import EPS

_TYPES = (torch.bfloat16, torch.float16)
MAX_REQUESTS = 8192                     # of one plan


class PagedPlan(NamedTuple):
    """What ``paged_plan`` returns: int32 tensors on the device."""
    slots: torch.Tensor                 # (rows) slot of each row's token, -1 for rows without one
    positions: torch.Tensor             # (rows) position of each row's token in its request, 0 for rows without one
    starts: torch.Tensor                # (requests + 1) first row of each request
    lengths: torch.Tensor               # (requests) tokens held after the step
    n_free: torch.Tensor                # (1) free pages after the step


_bound = None


def _native():
    """The native side of these calls (csrc/host_attention.cpp), which takes arguments that are as the kernels read them and
    returns None for all others."""
    global _bound
    if _bound is None:
        lib, host = _lib.load(), _lib.host()
        host.bind(*(ctypes.cast(getattr(lib, "dlrb200_" + name), ctypes.c_void_p).value
                    for name in ("paged_plan", "qk_norm_rope", "qk_norm_rope_backward", "qk_norm_rope_backward_workspace_bytes",
                                 "paged_attention", "paged_attention_workspace_bytes", "strerror")))
        _bound = host
    return _bound


def _result(out, what):
    if type(out) is int:
        _lib.check(out, what)
    if out is None:
        raise RuntimeError(f"{what}: arguments that passed every check were not taken")
    return out


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


def _no_tangents(what, *tensors):
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")


def _not_negated(what, *tensors):
    for t in tensors:
        if t is not None and t.is_neg():
            raise ValueError(f"{what}: tensors that are negated lazily are not taken here")


def _int32(what, name, t, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"{what}: {name} has type {t.dtype}, expected int32")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be contiguous")


def _page_size(what, page_size):
    if type(page_size) is not int:
        raise TypeError(f"{what}: the page size must be an int, not {type(page_size).__name__}")
    if not 16 <= page_size <= 1 << 20 or page_size & (page_size - 1):
        raise ValueError(f"{what}: pages have 2^n tokens, 16 to 2^20, not {page_size}")


def _check_cache(what, k_cache, v_cache, dtype, kv_heads, dim, multiple):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"{what}: the caches must be (pages, kv_heads, page tokens, dim) tensors of one shape")
    if not (k_cache.dtype == v_cache.dtype == dtype):
        raise TypeError(f"{what}: the caches have types {k_cache.dtype} and {v_cache.dtype}, expected {dtype}")
    if k_cache.shape[1] != kv_heads or k_cache.shape[3] != dim:
        raise ValueError(f"{what}: the caches have shape {tuple(k_cache.shape)}, expected {kv_heads} heads of {dim}")
    _not_negated(what, k_cache, v_cache)
    _page_size(what, k_cache.shape[2])
    if k_cache.shape[0] * k_cache.shape[2] > 0x7fffffff:
        raise ValueError(f"{what}: the caches have more than 2^31 - 1 slots")
    for c in (k_cache, v_cache):
        strides = [s for s, n in zip(c.stride()[:3], c.shape) if n > 1]
        if c.numel() and (c.stride(3) != 1 or any(s % multiple for s in strides) or c.data_ptr() % (2 * multiple)):
            raise ValueError(f"{what}: the caches need a contiguous last dimension and strides of a multiple of {multiple} elements")


def _heads(t: torch.Tensor, multiple: int) -> torch.Tensor:
    """t if its rows can be read where they are, else a contiguous copy."""
    t = t.resolve_neg()
    one = t.dim() <= 3 or t.is_contiguous()               # the leading dimensions are a single one
    if one and t.stride(-1) == 1 and not any(s % multiple for s in t.stride()[:-1]) and t.data_ptr() % (2 * multiple) == 0:
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
    or, with ``in_place``, in those given.  A request is refused (it keeps its tokens, none if it is finished, and its rows have
    slot -1) when the table has no columns for its tokens, when they do not fit its rows, or when it needs pages and those asked for
    up to and including it are more than there are free.
    """
    out = _native().paged_plan(lengths, new_tokens, block_table, free_pages, n_free, page_size, width, rows, finished, in_place)
    if type(out) is tuple:
        return PagedPlan(*out)
    what = "paged_plan"
    _all_tensors(what, lengths, new_tokens, block_table, free_pages, n_free, *(() if finished is None else (finished,)))
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
        if type(width) is not int or width < 1:
            raise ValueError(f"{what}: width is an int, at least 1")
        rows = width * n
    if type(rows) is not int or rows < 0 or rows > 1 << 30:
        raise ValueError(f"{what}: {rows} rows, 0 to 2^30 are possible")
    _not_negated(what, lengths, new_tokens, block_table, free_pages, n_free, finished)
    device = _on_one_device(what, lengths, new_tokens, block_table, free_pages, n_free, finished)
    with torch.cuda.device(device):
        out = _native().paged_plan(lengths, new_tokens, block_table, free_pages, n_free, page_size, width, rows, finished, in_place)
    return PagedPlan(*_result(out, "dlrb200_paged_plan"))


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
    _all_tensors(what, *given)
    for w in given:
        if w.dtype not in (q.dtype, torch.float32) or w.dtype != given[0].dtype:
            raise TypeError(f"{what}: the weights have type {w.dtype}, expected {q.dtype} or float32 for both")
        if w.shape != (dim,):
            raise ValueError(f"{what}: the weights have shape {tuple(w.shape)}, expected {(dim,)}")
    return dim, half


def _vector(w):
    """A weight as the kernels read it: contiguous from a 16-byte boundary."""
    w = w if w is None else w.resolve_neg()
    if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0):
        return w
    return w.clone(memory_format=torch.contiguous_format)


def _in_shape(q, k, q_weight, k_weight, cos, sin, positions):
    """The arguments laid out as the kernels read them; gradients pass through."""
    return (_heads(q, 4), _heads(k, 4), _vector(q_weight), _vector(k_weight), cos.resolve_neg(), sin.resolve_neg(),
            positions.resolve_neg().contiguous())


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *, eps: float = EPS,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q`` (..., heads, dim) and ``k`` (..., kv_heads, dim), then the rotation by position; new
    tensors.

    ``q_weight`` and ``k_weight`` (dim), in the heads' type or fp32; None leaves that norm out.  ``cos`` and ``sin``
    (positions, half) fp32, see ``rope_tables``: the first 2 * half values of a head are turned, in pairs (i, i + half), or
    (2i, 2i + 1) with ``interleaved``; the rest passes through.  ``positions`` (...) int32 or int64; one outside the tables
    makes its row NaN.  fp32 throughout, rounded once.  Differentiable (once, in reverse mode) in q, k and
    the weights.
    """
    out = _native().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    if type(out) is tuple:
        return out
    what = "qk_norm_rope"
    _check_norm_rope(what, q, k, q_weight, k_weight, cos, sin, positions)
    if cos.requires_grad or sin.requires_grad:
        raise ValueError(f"{what}: the tables have no gradient")
    _no_tangents(what, q, k, q_weight, k_weight, cos, sin)
    device = _on_one_device(what, q, k, q_weight, k_weight, cos, sin, positions)
    with torch.cuda.device(device):
        out = _native().qk_norm_rope(*_in_shape(q, k, q_weight, k_weight, cos, sin, positions), float(eps), bool(interleaved))
    return _result(out, "dlrb200_qk_norm_rope")


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor],
                        k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                        slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, eps: float = EPS,
                        interleaved: bool = False, return_keys: bool = False):
    """``qk_norm_rope`` for serving: keys, and ``v`` as it is, go to ``slots`` (...) int32 of the caches; returns the queries,
    and with ``return_keys`` the keys too (what the attention over a whole prompt takes).

    Rows whose slot is outside the caches (-1) are not stored; the others must name different slots.  No gradient.
    """
    out = _native().qk_norm_rope_append(q, k, q_weight, k_weight, cos, sin, positions, v, slots, k_cache, v_cache, eps, interleaved,
                                        return_keys)
    if out is not None and type(out) is not int:
        return out
    what = "qk_norm_rope_append"
    _all_tensors(what, v, slots, k_cache, v_cache)
    dim, _ = _check_norm_rope(what, q, k, q_weight, k_weight, cos, sin, positions)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must be like k, {tuple(k.shape)} {k.dtype}")
    if slots.dtype != torch.int32 or slots.shape != positions.shape:
        raise ValueError(f"{what}: slots must be int32 of shape {tuple(positions.shape)}")
    _check_cache(what, k_cache, v_cache, q.dtype, k.shape[-2], dim, 4)
    if any(n > 1 and not step for c in (k_cache, v_cache) if c.numel() for n, step in zip(c.shape, c.stride())):
        raise ValueError(f"{what}: slots of the caches share memory")
    given = (q, k, v, q_weight, k_weight, cos, sin, k_cache, v_cache)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    _no_tangents(what, *given)
    device = _on_one_device(what, q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache)
    with torch.cuda.device(device):
        out = _native().qk_norm_rope_append(*_in_shape(q, k, q_weight, k_weight, cos, sin, positions), _heads(v, 4),
                                            slots.resolve_neg().contiguous(), k_cache, v_cache, float(eps), bool(interleaved),
                                            bool(return_keys))
    return _result(out, "dlrb200_qk_norm_rope")


# ---- attention --------------------------------------------------------------------------------------------------------------
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one token per request: ``q`` (requests, heads, dim) over the first ``lengths`` (requests) tokens of each
    request's pages, (requests, heads, dim); zeros where the length is 0.

    ``block_table`` (requests, columns) and ``lengths`` int32.  ``heads`` is a multiple of the caches' heads, each of which
    serves that many neighbouring query heads; dim is 64, 96, 128 or 256.  ``scale`` is 1 / sqrt(dim) unless given.  Lengths
    are read on the device: a captured call follows them.  A table entry outside the caches counts as a page of zeros and
    is never followed.  Scores, softmax and sums are fp32; the weights enter their product with the values to 16 bits at least
    (fp16: down to 2^-24 of the largest).  An infinite value of a request's token comes out infinite.  No gradient.
    """
    out = _native().paged_attention(q, k_cache, v_cache, block_table, lengths, scale)
    if out is not None and type(out) is not int:
        return out
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
    _no_tangents(what, q, k_cache, v_cache)
    device = _on_one_device(what, q, k_cache, v_cache, block_table, lengths)
    with torch.cuda.device(device):
        out = _native().paged_attention(_heads(q, 2), k_cache, v_cache, block_table.resolve_neg(), lengths.resolve_neg(),
                                        None if scale is None else float(scale))
    return _result(out, "dlrb200_paged_attention")
