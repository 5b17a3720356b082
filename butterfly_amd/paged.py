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
captured graphs share none), and can be captured in a HIP graph.  The operators are for inference: with
gradients enabled they refuse tensors that require them.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Union

import torch

from . import _native
from ._device import on, stream_of
from .attention import _check_heads, _dtype_code, _require_cuda, _scale

PAGE_SIZES = tuple(1 << i for i in range(4, 11))

# state[1] after a plan that did not fit (include/butterfly_amd_paged.h)
PLAN_ERRORS = {
    1: "a request's length is negative or beyond its block table row",
    2: "a request would outgrow its block table row",
    3: "the counts sum to more than num_rows",
    4: "the free list holds too few pages",
    5: "the free list's count is outside its array",
}


@dataclass
class PagedPlan:
    """What :func:`paged_plan` gives: the requests' new ``lengths`` [B], ``state`` [2] (free pages, error),
    ``starts`` [B + 1] (each request's first row), ``slots`` and ``positions`` [num_rows] of the new rows."""

    lengths: torch.Tensor
    state: torch.Tensor
    starts: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor


def _no_grad(*ts: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise ValueError("the paged operators are for inference: call them under torch.no_grad()")


def _one_device(*ts: Optional[torch.Tensor]) -> torch.device:
    ts = [t for t in ts if t is not None]
    _require_cuda(*ts)
    if any(t.device != ts[0].device for t in ts):
        raise ValueError("all tensors must be on one device")
    return ts[0].device


def _check_page_size(page_size: int) -> int:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size} must be a power of two from 16 to 1024")
    return int(page_size)


def _ints(t: torch.Tensor, name: str, dtype: torch.dtype, n: Optional[int] = None) -> torch.Tensor:
    if t.dim() != 1 or t.dtype != dtype or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be a 1-D {dtype} tensor" + (f" of {n}" if n is not None else ""))
    return t


def _table(t: torch.Tensor, b: int) -> int:
    """The block table's row stride."""
    if t.dim() != 2 or t.dtype != torch.int32 or t.shape[0] != b:
        raise ValueError(f"block_table must be an int32 [{b}, pages] tensor")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError("block_table's rows must be contiguous")
    return t.stride(0) if b > 1 else max(1, t.shape[1])


def _strides(t: torch.Tensor, dims) -> List[int]:
    """Strides of ``dims``; 0 where a dimension has a single entry."""
    return [t.stride(i) if t.shape[i] > 1 else 0 for i in dims]


def _rows_fit(t: torch.Tensor, dims) -> bool:
    """Whether a kernel's 16-byte accesses take ``t`` as it lies: contiguous in its last dimension, 16-byte
    aligned in every other (``dims``)."""
    es = t.element_size()
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(s >= 0 and s * es % 16 == 0 for s in _strides(t, dims)))


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, written: bool) -> List[int]:
    """The six page, head and row strides of a pair of page tensors."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must be [num_pages, Hkv, page_size, d] of one shape and type")
    if 0 in k_pages.shape:
        raise ValueError("the pages hold nothing")
    _check_page_size(k_pages.shape[2])
    for t in (k_pages, v_pages):
        if not _rows_fit(t, (0, 1, 2)):
            raise ValueError("pages must be contiguous in head_dim and 16-byte aligned in every other dimension")
        if written and any(t.shape[i] > 1 and t.stride(i) == 0 for i in range(3)):
            raise ValueError("pages that are written must not overlap themselves")
    return _strides(k_pages, (0, 1, 2)) + _strides(v_pages, (0, 1, 2))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[N, H, d] rows that the kernels take as they lie, or a contiguous copy."""
    return t if _rows_fit(t, (0, 1)) else t.clone(memory_format=torch.contiguous_format)


def paged_plan(block_table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor, free_pages: torch.Tensor,
               state: torch.Tensor, *, page_size: int, num_rows: int, in_place: bool = False) -> PagedPlan:
    """One step's bookkeeping on the device (``bfly_paged_plan``, two launches for many rows, else one).

    Request ``b`` of ``B`` holds ``lengths[b]`` tokens and its pages are ``block_table[b]`` (int32
    [B, pages]).  ``counts[b] > 0`` appends that many tokens, ``counts[b] < 0`` takes back the last
    ``-counts[b]`` (all of them at the most: the request leaves), 0 leaves it as it is.  ``free_pages`` is a
    stack of ``state[0]`` page ids: pages no longer needed go on top, the first of them topmost, then the
    pages that others need are taken from the top in request order.  All of these are int32.

    ``num_rows`` (known on the host) is how many rows the step has room for: row ``starts[b] + i`` is request
    ``b``'s ``i``-th new token, rows behind the last have slot -1 and position 0.

    ``block_table`` and ``free_pages`` are updated; ``lengths`` and ``state`` too with ``in_place``, else the
    new ones are in the result only.  When something does not fit (``PLAN_ERRORS``) nothing changes,
    ``state[1]`` holds the code and every slot is -1, and so for every later step until the caller clears
    it: a captured loop that ran out of pages is found out by reading the state once.
    """
    dev = _one_device(block_table, lengths, counts, free_pages, state)
    page_size, num_rows = _check_page_size(page_size), int(num_rows)
    b = lengths.shape[0] if lengths.dim() == 1 else -1
    stride = _table(block_table, b)
    if b > 1 and stride < block_table.shape[1]:
        raise ValueError("block_table's rows must not overlap")
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    i32 = torch.int32
    for t, name, n in ((lengths, "lengths", b), (counts, "counts", b), (free_pages, "free_pages", None), (state, "state", 2)):
        _ints(t, name, i32, n)
    if not free_pages.is_contiguous() or in_place and not (lengths.is_contiguous() and state.is_contiguous()):
        raise ValueError("tensors that are updated must be contiguous")
    lengths, counts, state = lengths.contiguous(), counts.contiguous(), state.contiguous()
    new_lengths, new_state = (lengths, state) if in_place else (torch.empty_like(lengths), torch.empty_like(state))
    # the row starts and, behind them, the kernel's workspace
    starts = torch.empty(2, b + 1, dtype=i32, device=dev)
    rows = torch.empty(2, num_rows, dtype=torch.int64, device=dev)
    with on(dev):
        _native.call("bfly_paged_plan", block_table.data_ptr(), b, block_table.shape[1], stride, lengths.data_ptr(),
                     counts.data_ptr(), free_pages.data_ptr(), free_pages.numel(), state.data_ptr(), page_size, num_rows,
                     new_lengths.data_ptr(), new_state.data_ptr(), starts.data_ptr(), rows.data_ptr(),
                     rows.data_ptr() + 8 * num_rows, starts.data_ptr() + 4 * (b + 1), 4 * (b + 1), stream_of(dev))
    return PagedPlan(new_lengths, new_state, starts[0], rows[0], rows[1])


def _check_rows(k, v, k_pages, v_pages, slots):
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError("k and v must be [N, Hkv, d] of one shape")
    if not k.dtype == v.dtype == k_pages.dtype:
        raise ValueError("rows and pages must have one type")
    if k_pages.dim() == 4 and (k.shape[1], k.shape[2]) != (k_pages.shape[1], k_pages.shape[3]):
        raise ValueError("rows and pages must have the same heads and head_dim")
    _ints(slots, "slots", torch.int64, k.shape[0])


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Rows ``k``, ``v`` [N, Hkv, d] (any strides) into their ``slots`` (int64 [N]) of the pages
    [num_pages, Hkv, page_size, d], one launch of ``bfly_paged_append``.  A row whose slot is negative or
    beyond the pages is passed over.  The slots of a call are distinct, as a plan gives them (of two rows
    with one slot it is not defined which stays).  float32 or bfloat16; ``d`` of whole 16-byte pieces."""
    dev = _one_device(k, v, k_pages, v_pages, slots)
    _no_grad(k, v, k_pages, v_pages)
    strides = _pages(k_pages, v_pages, True)
    _check_rows(k, v, k_pages, v_pages, slots)
    n, hkv, d = k.shape
    code = _dtype_code(k)
    if d * k.element_size() % 16:
        raise ValueError("head_dim must be whole 16-byte pieces")
    if n == 0:
        return
    k, v, slots = _rows(k), _rows(v), slots.contiguous()
    with on(dev):
        _native.call("bfly_paged_append", k.data_ptr(), v.data_ptr(), code, n, hkv, d, *_strides(k, (0, 1)),
                     *_strides(v, (0, 1)), slots.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0],
                     k_pages.shape[2], *strides, stream_of(dev))


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
    dev = _one_device(q, k, v, k_pages, v_pages, slots, positions, cos, sin, q_weight, k_weight)
    _no_grad(q, k, v, k_pages, v_pages, cos, sin, q_weight, k_weight)
    strides = _pages(k_pages, v_pages, True)
    _check_rows(k, v, k_pages, v_pages, slots)
    n, hkv, d = k.shape
    if q.dim() != 3 or (q.shape[0], q.shape[2]) != (n, d) or q.dtype != k.dtype:
        raise ValueError("q must be [N, Hq, d] rows of k's type")
    hq, code = q.shape[1], _dtype_code(q)
    _check_heads(hq, hkv)
    if hq == 0:
        raise ValueError("q holds no heads")
    _ints(positions, "positions", torch.int64, n)
    if cos.dim() != 2 or cos.shape != sin.shape or not cos.dtype == sin.dtype == torch.float32 or cos.shape[0] == 0:
        raise ValueError("cos and sin must be float32 [rows, r] tables of one shape")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("give both norm weights or neither")
    if q_weight is not None and any(w.shape != (d,) or w.dtype != q.dtype for w in (q_weight, k_weight)):
        raise ValueError("norm weights must be [d] of the rows' type")
    out = torch.empty(n, hq, d, dtype=q.dtype, device=dev)
    if n == 0:
        return out
    q, k, v, slots, positions = _rows(q), _rows(k), _rows(v), slots.contiguous(), positions.contiguous()
    cos, sin, qw, kw = (t if t is None or t.is_contiguous() and t.data_ptr() % 16 == 0
                        else t.clone(memory_format=torch.contiguous_format) for t in (cos, sin, q_weight, k_weight))
    with on(dev):
        _native.call("bfly_paged_rope_append", q.data_ptr(), k.data_ptr(), v.data_ptr(), code, n, hq, hkv, d,
                     *_strides(q, (0, 1)), *_strides(k, (0, 1)), *_strides(v, (0, 1)),
                     qw.data_ptr() if qw is not None else None, kw.data_ptr() if kw is not None else None, float(eps),
                     cos.data_ptr(), sin.data_ptr(), cos.shape[0], cos.shape[1], positions.data_ptr(), slots.data_ptr(),
                     out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0], k_pages.shape[2], *strides,
                     stream_of(dev))
    return out


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
    part of the result, whatever they hold.  float32 or bfloat16, head_dim 64, 128 or 256."""
    dev = _one_device(q, k_pages, v_pages, block_table, lengths)
    _no_grad(q, k_pages, v_pages)
    strides = _pages(k_pages, v_pages, False)
    pages, hkv, page_size, d = k_pages.shape
    if q.dim() != 4 or q.shape[2] != 1 or q.shape[3] != d or q.dtype != k_pages.dtype:
        raise ValueError("q must be [B, Hq, 1, d] of the pages' type")
    b, hq, code = q.shape[0], q.shape[1], _dtype_code(q)
    _check_heads(hq, hkv)
    if hq == 0:
        raise ValueError("q holds no heads")
    stride = _table(block_table, b)
    _ints(lengths, "lengths", torch.int32, b)
    window = int(window)
    if window < 0 or window >= 1 << 31:
        raise ValueError("window must be 0 (everything) or a number of tokens")
    width = block_table.shape[1]
    out = torch.empty(b, hq, 1, d, dtype=q.dtype, device=dev)
    l = m = None
    if return_stats:
        l, m = torch.empty(2, b, hq, 1, 1, dtype=torch.float32, device=dev)
    if b:
        q, lengths = _rows(q[:, :, 0]), lengths.contiguous()
        with on(dev):
            need = _native.lib().bfly_paged_attention_workspace_bytes(b, hq, hkv, d, width, page_size, window)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            _native.call("bfly_paged_attention", q.data_ptr(), code, b, hq, hkv, d, *_strides(q, (0, 1)),
                         k_pages.data_ptr(), v_pages.data_ptr(), pages, page_size, *strides, block_table.data_ptr(), width,
                         stride, lengths.data_ptr(), window, _scale(scale, d), out.data_ptr(),
                         l.data_ptr() if l is not None else None, m.data_ptr() if m is not None else None,
                         ws.data_ptr() if ws is not None else None, need, stream_of(dev))
    return (out, l, m) if return_stats else out
