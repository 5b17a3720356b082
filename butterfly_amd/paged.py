"""A paged key-value cache for the layers that keep dense attention, and its operators.

The swap replaces the attention of chosen layers; the others keep dense attention over a cache that
grows with the context (bna/integrations/qwen_mlx.py:1822-1846, qwen_torch.py:1652-1700 leave them and
their caches to the host model).  Here their keys and values live in pages of ``page_size`` rows,
``[num_pages, Hkv, page_size, d]``, which a block table assigns to the requests that are served together.
Requests have lengths of their own, and nothing on the way of a decode step needs the host:

* :func:`paged_plan` makes a step's bookkeeping from the requests' lengths: pages from and to a free
  list, the block table, each new row's slot (``page * page_size + row``) and position;
* :func:`paged_append` writes rows of keys and values into their slots;
* :func:`paged_rope_append` does so for a decoder's projection rows, with the q/k RMSNorm and RoPE at
  each row's own position on the way;
* :func:`paged_attention` lets one new token of every request attend over its pages.

:class:`PagedKVCache` holds the tensors of all layers and the bookkeeping they share.  Every call runs on
the current stream of its tensors' device, allocates only its outputs (and a workspace of its own, so
captured graphs share none), and can be captured in a HIP graph.  The operators are for inference: they refuse
tensors that require gradients (with gradients enabled) or carry tangents, and traces.
"""
from __future__ import annotations

import math
from functools import lru_cache
from operator import index
from typing import Iterable, List, NamedTuple, Optional

import torch
from torch import _C
from torch.autograd import forward_ad

from . import _native
from ._device import _GET_DEVICE, stream_of

_PLAN, _APPEND, _ROPE, _ATTN = (_native.PAGED_STRUCTS["bfly_paged_" + x].pack
                                for x in ("plan", "append", "rope_append", "attention"))
_EMPTY = torch.empty_strided     # (0.95 us a call; torch.empty, which also sorts out layouts, 1.8)
PAGE_SIZES = frozenset(1 << i for i in range(4, 11))
HEAD_DIMS = (64, 128, 256)       # of paged_rope_append and paged_attention

# state[1] after a plan that did not fit (include/butterfly_amd_paged.h)
PLAN_ERRORS = {
    1: "a request's length is negative or beyond its block table row",
    2: "a request would outgrow its block table row",
    3: "the counts sum to more than num_rows",
    4: "the free list holds too few pages",
    5: "the free list's count is outside its array",
}


class PagedPlan(NamedTuple):
    """What :func:`paged_plan` gives: the requests' new ``lengths`` [B], ``state`` [2] (free pages, error),
    ``starts`` [B + 1] (each request's first row), ``slots`` and ``positions`` [num_rows] of the new rows."""

    lengths: torch.Tensor
    state: torch.Tensor
    starts: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor


# The checks below cost a decode step's host time (these calls take 4 to 8 us on the GPU): each tests what a
# well-formed call has in as few attribute reads as it takes, and only then, case by case, what is wrong.
_GRAD = "the paged operators are for inference: call them under torch.no_grad()"


def _check_followed(*tensors: Optional[torch.Tensor]) -> None:
    """Refuses what a native call would hide itself from: a trace, or a tangent of one of ``tensors``."""
    if _C._get_tracing_state() is not None:
        raise ValueError("the paged operators cannot be traced: a trace would hold this call's result as a constant")
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(_GRAD + " and without tangents")


def _device_of(t: torch.Tensor) -> int:
    dev = t.get_device()
    if dev < 0:
        raise ValueError("butterfly_amd operators take GPU tensors (device 'cuda')")
    return dev


def _other_device() -> None:
    raise ValueError("all tensors must be GPU tensors of one device")


def _dtype_code(dtype: torch.dtype) -> int:
    if dtype is torch.bfloat16:
        return _native.DTYPE_BF16
    if dtype is torch.float32:
        return _native.DTYPE_F32
    raise ValueError(f"unsupported dtype {dtype}; expected float32 or bfloat16")


def _check_ints(t: torch.Tensor, name: str, dtype: torch.dtype, n: int) -> None:
    if t.dtype is not dtype or t.shape != (n,):
        raise ValueError(f"{name} must be a 1-D {dtype} tensor of {n}")


def _table_stride(t: torch.Tensor, b: int) -> int:
    """The block table's row stride (its width where there is one row)."""
    shape = t.shape
    if len(shape) != 2 or t.dtype is not torch.int32 or shape[0] != b:
        raise ValueError(f"block_table must be an int32 [{b}, pages] tensor")
    stride, one = t.stride()
    if one != 1 and shape[1] > 1:
        raise ValueError("block_table's rows must be contiguous")
    return stride if b > 1 else shape[1]


def _lies(t: torch.Tensor, dims: int):
    """The strides of the first ``dims`` dimensions of ``t`` where 16-byte accesses take it as it lies
    (contiguous in the last dimension, 16-byte aligned in every other), else None."""
    strides = [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)][:dims]
    es = t.element_size()
    if t.data_ptr() % 16 or t.stride(-1) != 1 or any(s * es % 16 for s in strides):
        return None
    return strides


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, dev: int, written: bool):
    """Shape and the six page, head and row strides of a pair of page tensors."""
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not dtype:
        raise ValueError("k_pages and v_pages must be [num_pages, Hkv, page_size, d] of one shape and type")
    if k_pages.get_device() != dev or v_pages.get_device() != dev:
        _other_device()
    if shape[2] not in PAGE_SIZES:
        raise ValueError(f"page_size {shape[2]} must be a power of two from 16 to 1024")
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    kd, vd = k_pages.data_ptr(), v_pages.data_ptr()
    if k3 == v3 == 1 and kd and vd \
            and not ((kd | vd) & 15 or (k0 | k1 | k2 | v0 | v1 | v2) & (7 if dtype is torch.bfloat16 else 3)) \
            and (not written or k0 and k1 and k2 and v0 and v1 and v2 and kd != vd):
        return shape, (k0, k1, k2, v0, v1, v2)
    if 0 in shape:
        raise ValueError("the pages hold nothing")
    k, v = _lies(k_pages, 3), _lies(v_pages, 3)
    if k is None or v is None:
        raise ValueError("pages must be contiguous in head_dim and 16-byte aligned in every other dimension")
    if written and (kd == vd or any(s == 0 and n > 1 for s, n in zip(k + v, tuple(shape[:3]) * 2))):
        raise ValueError("pages that are written must not overlap themselves or each other")
    return shape, (*k, *v)


def _rows(t: torch.Tensor):
    """[N, H, d] rows and their two strides, as they lie where a kernel takes them so, else of a contiguous copy."""
    s0, s1, s2 = t.stride()
    if s2 == 1 and not (t.data_ptr() & 15 or (s0 | s1) & (7 if t.dtype is torch.bfloat16 else 3)):
        return t, s0, s1
    strides = _lies(t, 2)
    if strides is None:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = t.stride()
    return t, strides[0], strides[1]


def paged_plan(block_table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor, free_pages: torch.Tensor,
               state: torch.Tensor, *, page_size: int, num_rows: int, rows_each: int = 0, in_place: bool = False) -> PagedPlan:
    """One step's bookkeeping on the device (``bfly_paged_plan``, two launches for many rows, else one).

    Request ``b`` of ``B`` holds ``lengths[b]`` tokens and its pages are ``block_table[b]`` (int32
    [B, pages]).  ``counts[b] > 0`` appends that many tokens, ``counts[b] < 0`` takes back the last
    ``-counts[b]`` (all of them at the most: the request leaves), 0 leaves it as it is.  ``free_pages`` is a
    stack of ``state[0]`` page ids: pages no longer needed go on top, the first of them topmost, then the
    pages that others need are taken from the top in request order.  All of these are int32.

    ``num_rows`` (known on the host) is how many rows the step has room for: row ``starts[b] + i`` is request
    ``b``'s ``i``-th new token, rows behind the last have slot -1 and position 0.  With ``rows_each`` every
    request has that many rows of its own instead (``num_rows = B * rows_each``, ``starts[b] = b * rows_each``):
    a batch of fixed shape in which requests may be idle, as a captured decode step needs.

    ``block_table`` and ``free_pages`` are updated; ``lengths`` and ``state`` too with ``in_place``, else the
    new ones are in the result only.  When something does not fit (``PLAN_ERRORS``) nothing changes,
    ``state[1]`` holds the code and every slot is -1, and so for every later step until the caller clears
    it: a captured loop that ran out of pages is found out by reading the state once.

    A page belongs to one request (``paged_attention`` reads tables whose rows share pages, but a plan would
    give such a page back with each of them).
    """
    dev = _device_of(lengths)
    if not block_table.get_device() == counts.get_device() == free_pages.get_device() == state.get_device() == dev:
        _other_device()
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_plan(block_table, lengths, counts, free_pages, state, page_size=page_size, num_rows=num_rows,
                              rows_each=rows_each, in_place=in_place)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed()
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size} must be a power of two from 16 to 1024")
    if lengths.dim() != 1:
        raise ValueError("lengths must be a 1-D torch.int32 tensor")
    b, i32 = lengths.shape[0], torch.int32
    if not lengths.dtype is counts.dtype is state.dtype is free_pages.dtype is i32 or counts.shape != lengths.shape \
            or state.shape != (2,) or free_pages.dim() != 1:
        raise ValueError("lengths and counts [B], free_pages and state [2] must be 1-D torch.int32 tensors")
    stride, width = _table_stride(block_table, b), block_table.shape[1]
    if stride < width:
        raise ValueError("block_table's rows must not overlap")
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    if rows_each < 0 or rows_each and num_rows != b * rows_each:
        raise ValueError(f"num_rows must be the {b} requests' {rows_each} rows each")
    if not (lengths.is_contiguous() and counts.is_contiguous() and state.is_contiguous() and free_pages.is_contiguous()):
        if not free_pages.is_contiguous() or in_place and not (lengths.is_contiguous() and state.is_contiguous()):
            raise ValueError("tensors that are updated must be contiguous")
        lengths, counts, state = lengths.contiguous(), counts.contiguous(), state.contiguous()
    cuda = lengths.device
    # one allocation for the int32 results and the kernel's workspace, one for the rows
    if in_place:
        new_lengths, new_state = lengths, state
        starts, ws = _EMPTY((4 * b + 4,), (1,), dtype=i32, device=cuda).split_with_sizes((b + 1, 3 * b + 3))
    else:
        new_lengths, new_state, starts, ws = _EMPTY((5 * b + 6,), (1,), dtype=i32, device=cuda).split_with_sizes(
            (b, 2, b + 1, 3 * b + 3))
    slots, positions = _EMPTY((2, num_rows), (num_rows, 1), dtype=torch.int64, device=cuda).unbind(0)
    _native.call("bfly_paged_plan", _PLAN(
        block_table.data_ptr(), b, width, stride, lengths.data_ptr(), counts.data_ptr(), free_pages.data_ptr(),
        free_pages.shape[0], state.data_ptr(), page_size, num_rows, rows_each, new_lengths.data_ptr(), new_state.data_ptr(),
        starts.data_ptr(), slots.data_ptr(), positions.data_ptr(), ws.data_ptr(), 12 * (b + 1)), stream_of(dev))
    return PagedPlan(new_lengths, new_state, starts, slots, positions)


def _check_rows(k, v, shape, dtype, slots, dev):
    n = k.shape
    if len(n) != 3 or v.shape != n or n[1] != shape[1] or n[2] != shape[3]:
        raise ValueError("k and v must be [N, Hkv, d] of the pages' heads and head_dim")
    if not k.dtype is v.dtype is dtype:
        raise ValueError("rows and pages must have one type")
    if k.get_device() != dev or v.get_device() != dev:
        _other_device()
    _check_ints(slots, "slots", torch.int64, n[0])
    return n


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Rows ``k``, ``v`` [N, Hkv, d] (any strides) into their ``slots`` (int64 [N]) of the pages
    [num_pages, Hkv, page_size, d], one launch of ``bfly_paged_append``.  A row whose slot is negative or
    beyond the pages is passed over.  The slots of a call are distinct, as a plan gives them (of two rows
    with one slot it is not defined which stays), and the rows are not themselves among the slots' rows.
    float32 or bfloat16; ``d`` of whole 16-byte pieces."""
    dev = _device_of(slots)
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_append(k, v, k_pages, v_pages, slots)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise ValueError(_GRAD)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed(k, v, k_pages, v_pages)
    shape, strides = _pages(k_pages, v_pages, dev, True)
    n, hkv, d = _check_rows(k, v, shape, k_pages.dtype, slots, dev)
    code = _dtype_code(k_pages.dtype)
    if d % (4 if code == _native.DTYPE_F32 else 8):
        raise ValueError("head_dim must be whole 16-byte pieces")
    if n == 0:
        return
    (k, k0, k1), (v, v0, v1) = _rows(k), _rows(v)
    slots = slots.contiguous()
    _native.call("bfly_paged_append", _APPEND(
        k.data_ptr(), v.data_ptr(), code, n, hkv, d, k0, k1, v0, v1, slots.data_ptr(),
        k_pages.data_ptr(), v_pages.data_ptr(), shape[0], shape[2], *strides), stream_of(dev))


def paged_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      slots: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                      q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                      eps: float = 1e-6) -> torch.Tensor:
    """The projection tail of a paged layer, one launch of ``bfly_paged_rope_append``: RMSNorm of each head of
    ``q`` [N, Hq, d] and ``k`` [N, Hkv, d] with ``q_weight`` / ``k_weight`` [d] (both ``None``: no norm),
    rotate-half RoPE at each row's own position, and ``k`` and ``v`` into their ``slots``.  Returns the rotated
    ``q`` [N, Hq, d].

    ``cos`` and ``sin`` [rows, r] (float32) are whole tables, ``positions`` (int64 [N]) picks their rows;
    elements from ``r`` on are not rotated.  q, k and v may be column ranges of one fused projection.  Every
    row of q is computed; k and v rows as in :func:`paged_append`.  A position outside the tables gives NaN.
    Between the inputs and the outputs nothing is rounded to fewer than 32 bits (``bfly_qk_norm_rope``, whose
    rounding points are the modules', rounds after the norm as well).  head_dim 64, 128 or 256, ``r`` a multiple
    of 16."""
    dev = _device_of(q)
    if not slots.get_device() == positions.get_device() == cos.get_device() == sin.get_device() == dev:
        _other_device()
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_rope_append(q, k, v, k_pages, v_pages, slots, positions, cos, sin, q_weight=q_weight,
                                     k_weight=k_weight, eps=eps)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_pages.requires_grad
                                    or v_pages.requires_grad or cos.requires_grad or sin.requires_grad
                                    or q_weight is not None and q_weight.requires_grad
                                    or k_weight is not None and k_weight.requires_grad):
        raise ValueError(_GRAD)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed(q, k, v, k_pages, v_pages, cos, sin, q_weight, k_weight)
    shape, strides = _pages(k_pages, v_pages, dev, True)
    dtype = k_pages.dtype
    n, hkv, d = _check_rows(k, v, shape, dtype, slots, dev)
    sq = q.shape
    if len(sq) != 3 or sq[0] != n or sq[2] != d or q.dtype is not dtype:
        raise ValueError("q must be [N, Hq, d] rows of k's type")
    hq, code = sq[1], _dtype_code(dtype)
    if hq == 0 or hq % hkv:
        raise ValueError(f"query heads {hq} must be a multiple of kv heads {hkv}")
    _check_ints(positions, "positions", torch.int64, n)
    table = cos.shape
    if len(table) != 2 or sin.shape != table or table[0] == 0 or not cos.dtype is sin.dtype is torch.float32:
        raise ValueError("cos and sin must be float32 [rows, r] tables of one shape")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("give both norm weights or neither")
    qw = kw = 0
    if q_weight is not None:
        if q_weight.shape != (d,) or k_weight.shape != (d,) or not q_weight.dtype is k_weight.dtype is dtype:
            raise ValueError("norm weights must be [d] of the rows' type")
        if not q_weight.get_device() == k_weight.get_device() == dev:
            _other_device()
        q_weight, k_weight = _flat(q_weight), _flat(k_weight)
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
    out = _EMPTY(sq, (hq * d, d, 1), dtype=dtype, device=q.device)
    if n == 0:
        return out
    q0, q1, q2 = q.stride()
    k0, k1, k2 = k.stride()
    v0, v1, v2 = v.stride()
    if not q2 == k2 == v2 == 1 or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15 \
            or (q0 | q1 | k0 | k1 | v0 | v1) & (7 if code else 3):
        (q, q0, q1), (k, k0, k1), (v, v0, v1) = _rows(q), _rows(k), _rows(v)
    slots, positions, cos, sin = slots.contiguous(), positions.contiguous(), _flat(cos), _flat(sin)
    _native.call("bfly_paged_rope_append", _ROPE(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), code, n, hq, hkv, d, q0, q1, k0, k1, v0, v1, qw, kw, eps, cos.data_ptr(),
        sin.data_ptr(), table[0], table[1], positions.data_ptr(), slots.data_ptr(), out.data_ptr(),
        k_pages.data_ptr(), v_pages.data_ptr(), shape[0], shape[2], *strides), stream_of(dev))
    return out


def _flat(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned."""
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: Optional[float] = None, window: int = 0,
                    return_stats: bool = False):
    """One new token of every request over its pages (``bfly_paged_attention``).

    ``q`` [B, Hq, 1, d]; request ``b`` sees positions ``[max(0, lengths[b] - window), lengths[b])`` of its
    pages (``window`` 0: all of them; its own key is appended first, as the last of them), query head ``h``
    those of kv head ``h // (Hq / Hkv)``.  ``block_table`` int32 [B, pages], ``lengths`` int32 [B].  ``scale``
    defaults to ``1 / sqrt(d)``.

    Returns ``out`` [B, Hq, 1, d], with ``return_stats`` the stream ``(out, l, m)`` of
    ``swa_stream_attention``, which ``online_softmax_merge`` takes.  A request without tokens gives zeros and
    the empty stream ``(0, 0, -1e30)``; a length beyond its table row, or a page id outside the pages among
    those that are read, gives NaN for that request.  Rows of a page behind the request's last token are never
    part of the result, whatever they hold.  Sums are divided by ``l`` at the end: values whose weighted sum passes the
    largest fp32 number give infinities.  float32 or bfloat16, head_dim 64, 128 or 256."""
    dev = _device_of(q)
    if not block_table.get_device() == lengths.get_device() == dev:
        _other_device()
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_attention(q, k_pages, v_pages, block_table, lengths, scale=scale, window=window,
                                   return_stats=return_stats)
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise ValueError(_GRAD)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed(q, k_pages, v_pages)
    shape, strides = _pages(k_pages, v_pages, dev, False)
    pages, hkv, page_size, d = shape
    sq, dtype = q.shape, q.dtype
    if len(sq) != 4 or sq[2] != 1 or sq[3] != d or dtype is not k_pages.dtype:
        raise ValueError("q must be [B, Hq, 1, d] of the pages' type")
    b, hq, code = sq[0], sq[1], _dtype_code(dtype)
    if hq == 0 or hq % hkv:
        raise ValueError(f"query heads {hq} must be a multiple of kv heads {hkv}")
    stride, width = _table_stride(block_table, b), block_table.shape[1]
    _check_ints(lengths, "lengths", torch.int32, b)
    window = index(window)
    if not 0 <= window < 1 << 31:
        raise ValueError("window must be 0 (everything) or a number of tokens")
    cuda = q.device
    out = _EMPTY(sq, (hq * d, d, d, 1), dtype=dtype, device=cuda)
    l = m = ws = None
    lp = mp = 0
    if return_stats:
        l, m = _EMPTY((2, b, hq, 1, 1), (b * hq, hq, 1, 1, 1), dtype=torch.float32, device=cuda).unbind(0)
        lp, mp = l.data_ptr(), m.data_ptr()
    if b:
        q0, q1, _, q3 = q.stride()
        if q3 != 1 or q.data_ptr() & 15 or (q0 | q1) & (7 if code else 3):
            q = q.clone(memory_format=torch.contiguous_format)
            q0, q1, _, _ = q.stride()
        lengths = lengths.contiguous()
        need = _workspace_bytes(code, b, hq, hkv, d, width, page_size, window)
        if need:
            ws = _EMPTY((need,), (1,), dtype=torch.uint8, device=cuda)
        _native.call("bfly_paged_attention", _ATTN(
            q.data_ptr(), code, b, hq, hkv, d, q0, q1, k_pages.data_ptr(), v_pages.data_ptr(), pages, page_size, *strides,
            block_table.data_ptr(), width, stride, lengths.data_ptr(), window, 1.0 / math.sqrt(d) if scale is None else scale,
            out.data_ptr(), lp, mp, 0 if ws is None else ws.data_ptr(), need), stream_of(dev))
    return (out, l, m) if return_stats else out


@lru_cache(maxsize=1024)
def _workspace_bytes(*sizes: int) -> int:
    return _native.lib().bfly_paged_attention_workspace_bytes(*sizes)


def _capturing(x: torch.Tensor) -> bool:
    return x.is_cuda and torch.cuda.is_current_stream_capturing()


class PagedLayer:
    """One layer's pages of a :class:`PagedKVCache`: what an attention module takes as its ``cache``.  Between the
    cache's :meth:`PagedKVCache.begin` and the next one, its rows are the step's."""

    def __init__(self, cache: "PagedKVCache", k_pages: torch.Tensor, v_pages: torch.Tensor):
        self.cache, self.k_pages, self.v_pages = cache, k_pages, v_pages

    @property
    def plan(self) -> PagedPlan:
        if self.cache.plan is None:
            raise RuntimeError("begin() a step of the paged cache before its layers")
        return self.cache.plan

    def check_step(self, requests: int, rows_each: int) -> None:
        """``ValueError`` unless the step has ``rows_each`` rows of each of ``requests`` requests, ``RuntimeError`` where none
        has begun."""
        c, _ = self.cache, self.plan
        if c.max_requests != requests or c.rows_each != rows_each:
            has = f"{c.rows_each} rows of each" if c.rows_each else "packed rows"
            raise ValueError(f"the paged cache's step has {has} of its {c.max_requests} requests, not {rows_each} of each of "
                             f"{requests}")

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's rows of keys and values [N, Hkv, d] into their slots."""
        paged_append(k, v, self.k_pages, self.v_pages, self.plan.slots)

    def rope_append(self, q, k, v, cos, sin, *, q_weight=None, k_weight=None, eps: float = 1e-6) -> torch.Tensor:
        """The step's projection rows: :func:`paged_rope_append` at the plan's positions and slots."""
        p = self.plan
        return paged_rope_append(q, k, v, self.k_pages, self.v_pages, p.slots, p.positions, cos, sin, q_weight=q_weight,
                                 k_weight=k_weight, eps=eps)

    def attend(self, q: torch.Tensor, *, scale: Optional[float] = None, window: int = 0, return_stats: bool = False):
        """:func:`paged_attention` of one new token ``q`` [B, Hq, 1, d] of every request over its pages."""
        return paged_attention(q, self.k_pages, self.v_pages, self.cache.block_table, self.plan.lengths, scale=scale,
                               window=window, return_stats=return_stats)

    def history(self, tokens: int, request: Optional[int] = None):
        """The first ``tokens`` keys and values of every request, or of one, as dense [B, Hkv, tokens, d] tensors
        (what a prompt's further part attends to); the requests hold that many."""
        size, table = self.k_pages.shape[2], self.cache.block_table
        if request is not None:
            table = table[request:request + 1]
        ids = table[:, :-(-tokens // size)].long().clamp_(0, self.k_pages.shape[0] - 1)
        return tuple(x[ids].transpose(1, 2).flatten(2, 3)[:, :, :tokens] for x in (self.k_pages, self.v_pages))


class PagedKVCache:
    """Keys and values of ``max_requests`` requests in ``num_layers`` dense layers: pages
    ``[num_layers, num_pages, Hkv, page_size, d]`` and one block table, lengths and free list on the device,
    which all layers share (page ``p`` of a request is page ``p`` in every layer).

    ``max_tokens`` bounds a request (default: all pages).  A step is :meth:`begin` (or :meth:`begin_packed`), then
    every layer's rows and attention through ``layers[i]``; :meth:`sync` reads the state back."""

    def __init__(self, *, num_layers: int, num_pages: int, max_requests: int, num_kv_heads: int, head_dim: int,
                 page_size: int = 128, max_tokens: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device=None):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size {page_size} must be a power of two from 16 to 1024")
        if min(num_layers, num_pages, max_requests, num_kv_heads, head_dim) <= 0 or max_tokens is not None and max_tokens <= 0:
            raise ValueError("the cache's sizes must be positive")
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"unsupported dtype {dtype}; expected float32 or bfloat16")
        device = torch.device("cuda" if device is None else device)
        width = num_pages if max_tokens is None else min(num_pages, -(-max_tokens // page_size))
        self.page_size, self.max_requests, self.max_tokens = page_size, max_requests, width * page_size
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.k_pages, self.v_pages = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.layers = [PagedLayer(self, k, v) for k, v in zip(self.k_pages, self.v_pages)]
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_requests, width), -1, **i32)
        self.lengths = torch.zeros(max_requests, **i32)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)
        self.state = torch.tensor([num_pages, 0], **i32)
        self.plan: Optional[PagedPlan] = None
        self.rows_each = 0             # the step's rows of every request; 0: packed
        self._held: Optional[List[Optional[int]]] = None
        self._replayed = False         # the step was captured: replays make others of it

    @property
    def nbytes(self) -> int:
        return self.k_pages.nbytes + self.v_pages.nbytes

    def _begin(self, counts: torch.Tensor, num_rows: int, rows_each: int) -> PagedPlan:
        self.plan = paged_plan(self.block_table, self.lengths, counts, self.free_pages, self.state,
                               page_size=self.page_size, num_rows=num_rows, rows_each=rows_each, in_place=True)
        self.rows_each, self._held, self._replayed = rows_each, None, _capturing(self.lengths)
        return self.plan

    def begin(self, counts: torch.Tensor, rows_each: int = 1, *, start: Optional[int] = None) -> PagedPlan:
        """A step in which request ``b`` adds ``counts[b] <= rows_each`` tokens (int32 [B], on the device; negative:
        takes tokens back) and has ``rows_each`` rows, row ``b * rows_each + i`` its ``i``-th.  ``start``: every request
        holds that many tokens before the step, else ``ValueError`` and nothing changes (the lengths are read
        back for it)."""
        known = start is not None and self.require(start)
        plan = self._begin(counts, self.max_requests * rows_each, rows_each)
        if known:
            self._held = [int(start)] * self.max_requests
        return plan

    def begin_packed(self, counts: torch.Tensor, num_rows: int) -> PagedPlan:
        """A step whose rows follow each other, request by request: ragged prompts (for the layers' operators; an
        attention module has rows of every request, :meth:`begin`)."""
        return self._begin(counts, num_rows, 0)

    def check_heads(self, num_kv_heads: int, head_dim: int, dtype: torch.dtype) -> None:
        """``NotImplementedError`` or ``ValueError`` unless attention of such heads runs over these pages: before a
        step begins, not in the middle of a generation."""
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"attention over pages: head_dim={head_dim} unsupported {HEAD_DIMS}")
        _, _, heads, _, d = self.k_pages.shape
        if (heads, d, self.k_pages.dtype) != (num_kv_heads, head_dim, dtype):
            raise ValueError(f"a paged cache of {heads} kv heads of {d} in {self.k_pages.dtype} cannot take {num_kv_heads} of "
                             f"{head_dim} in {dtype}")

    def require(self, tokens: int, *, at_most: bool = False) -> bool:
        """``ValueError`` unless every request holds ``tokens`` tokens, or ``at_most`` as many (waits for the current
        stream).  ``False`` where an earlier step did not fit: lengths stand still then, until :meth:`sync` reports it."""
        *lengths, _, error = self._read(torch.cat([self.lengths, self.state]))
        if error:
            return False
        if any(n > tokens or n < tokens and not at_most for n in lengths):
            raise ValueError(f"the paged cache's requests hold {lengths} tokens, not {'at most ' * at_most}{tokens} each "
                             "(release() empties them)")
        return True

    def held(self) -> List[Optional[int]]:
        """How many tokens each request held before the step (``None``: one that adds none in it), for a step of
        ``rows_each`` rows.  Read back once a step (a captured one: every time, for its latest replay), which waits for
        the current stream."""
        if self._held is None or self._replayed:
            p = self.plan
            first = torch.where(p.slots >= 0, p.positions, -1).view(-1, self.rows_each)[:, 0]
            self._held = [None if n < 0 else n for n in self._read(first)]
        return self._held

    @staticmethod
    def _read(x: torch.Tensor) -> List[int]:
        if _capturing(x):
            raise RuntimeError("a paged step that needs its lengths on the host cannot be captured (steps of one token can)")
        return x.tolist()

    def release(self, requests: Iterable[int]) -> None:
        """The given requests (indices) leave: their pages go back to the free list."""
        counts = [0] * self.max_requests
        for r in requests:
            if not 0 <= r < self.max_requests:
                raise ValueError(f"request {r} is not one of {self.max_requests}")
            counts[r] = -(2 ** 31 - 1)
        self._begin(torch.tensor(counts, dtype=torch.int32, device=self.lengths.device), 0, 0)

    def sync(self) -> int:
        """Waits for the current stream; the number of free pages.  Raises ``RuntimeError`` if a step did not fit (that
        step and all after it changed nothing), and clears the error."""
        free, error = self.state.tolist()
        if error:
            self.state[1] = 0
            raise RuntimeError(f"paged cache: {PLAN_ERRORS.get(error, error)}")
        return free
