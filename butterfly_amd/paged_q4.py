"""The paged cache (:mod:`butterfly_amd.paged`) with its keys and values held in 4 bits, and its operators.

A row of a kv head is groups of 32 or 64 consecutive elements, each held as 4-bit affine codes: an element is
``code * scale + bias`` with a bf16 scale and bias for its group, the form of this package's 4-bit weights
(and of the reference's quantised caches, bna/integrations/mlx_kv_quant.py).  With groups of 64 a bf16 cache becomes 3.56
times smaller, and a decode step reads as much less.

* :func:`paged_q4_append` writes rows of keys and values into their slots;
* :func:`paged_q4_rope_append` does so for a decoder's projection rows, with the q/k RMSNorm and RoPE on the way;
* :func:`paged_q4_attention` lets one new token of every request attend over its pages;
* :func:`paged_q4_read` gives the first tokens of every request back as dense keys and values.

The bookkeeping is :func:`butterfly_amd.paged_plan`'s; ``PagedKVCache(..., quant_bits=4)`` holds such pages for all
layers.  Every call runs on the current stream of its tensors' device, allocates only its outputs (and a workspace of its
own), and can be captured in a HIP graph.  The operators are for inference: they refuse tensors that require
gradients (with gradients enabled) or carry tangents, and traces.
"""
from __future__ import annotations

import math
from functools import lru_cache
from operator import index
from typing import NamedTuple, Optional, Tuple

import torch
from torch import _C
from torch.autograd import forward_ad

from . import _native
from ._device import _GET_DEVICE, stream_of
from .paged import (_EMPTY, _GRAD, HEAD_DIMS, PAGE_SIZES, PagedLayer, _check_followed, _check_ints, _device_of, _dtype_code, _flat,
                    _other_device, _rows, _table_stride)

_APPEND, _ROPE, _READ, _ATTN = (_native.PAGED_Q4_STRUCTS["bfly_paged_q4_" + x].pack
                                for x in ("append", "rope_append", "read", "attention"))
GROUPS = (32, 64)


class Q4Pages(NamedTuple):
    """One layer's pages in 4 bits: ``k_codes`` and ``v_codes`` uint8 [num_pages, Hkv, page_size, d / 2], ``k_scales``
    and ``v_scales`` bfloat16 [num_pages, Hkv, page_size, d / group, 2] (scale, bias).

    Two codes a byte, the lower one first; the ``n``-th of 16 equal pieces of a row of codes holds the ``n``-th sixteenth
    of every group, group by group (what a lane of the attention takes of a row is part of every group)."""

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    @property
    def nbytes(self) -> int:
        return sum(t.nbytes for t in self)


def empty_q4_pages(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, *, group: int = 64,
                   layers: Tuple[int, ...] = (), device=None) -> Q4Pages:
    """Uninitialised pages (``layers``: dimensions before the pages')."""
    if head_dim not in HEAD_DIMS:
        raise NotImplementedError(f"pages in 4 bits: head_dim={head_dim} unsupported {HEAD_DIMS}")
    if group not in GROUPS:
        raise ValueError(f"group {group} must be 32 or 64")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size} must be a power of two from 16 to 1024")
    shape = (*layers, num_pages, num_kv_heads, page_size)
    device = torch.device("cuda" if device is None else device)
    codes, scales = ([torch.empty(*shape, *last, dtype=dtype, device=device) for _ in range(2)]
                     for last, dtype in (((head_dim // 2,), torch.uint8), ((head_dim // group, 2), torch.bfloat16)))
    return Q4Pages(codes[0], scales[0], codes[1], scales[1])


def _pages(pages: Q4Pages, dev: int, written: bool):
    """(num_pages, Hkv, page_size, d), and what the packed structs hold of the pages."""
    kc, ks, vc, vs = pages
    if not kc.dtype is vc.dtype is torch.uint8 or not ks.dtype is vs.dtype is torch.bfloat16:
        raise ValueError("pages must be uint8 codes and bfloat16 scales")
    if not kc.get_device() == ks.get_device() == vc.get_device() == vs.get_device() == dev:
        _other_device()
    shape, sizes = _layout(kc.shape, kc.stride(), ks.shape, ks.stride(), vc.shape, vc.stride(), vs.shape, vs.stride(), written)
    a, b, c, d = kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()
    if (a | b | c | d) & 15:
        raise ValueError("pages must be 16-byte aligned")
    if written and len({a, b, c, d}) < 4:
        raise ValueError("pages that are written must not overlap themselves or each other")
    return shape, (a, b, c, d, *sizes)


@lru_cache(maxsize=1024)
def _layout(kc, kc_strides, ks, ks_strides, vc, vc_strides, vs, vs_strides, written):
    """The checks of the pages' shapes and strides, which a decode step would repeat for every layer: (num_pages, Hkv,
    page_size, d) and (num_pages, page_size, group, strides in bytes)."""
    if len(kc) != 4 or len(ks) != 5 or vc != kc or vs != ks or ks[:3] != kc[:3] or ks[4] != 2 or ks[3] == 0:
        raise ValueError("pages must be codes [num_pages, Hkv, page_size, d / 2] and scales [num_pages, Hkv, page_size, "
                         "d / group, 2], k's and v's alike")
    num, hkv, size, half = kc
    d, groups = 2 * half, ks[3]
    group = d // groups
    if size not in PAGE_SIZES:
        raise ValueError(f"page_size {size} must be a power of two from 16 to 1024")
    if 0 in kc:
        raise ValueError("the pages hold nothing")
    if d not in HEAD_DIMS:
        raise NotImplementedError(f"pages in 4 bits: head_dim={d} unsupported {HEAD_DIMS}")
    if group not in GROUPS or group * groups != d:
        raise ValueError(f"groups of {d} / {groups} elements: must be of 32 or 64")
    out = []
    for shape, strides, last, es, unit in ((kc, kc_strides, (1,), 1, 16), (ks, ks_strides, (2, 1), 2, min(16, 4 * groups)),
                                           (vc, vc_strides, (1,), 1, 16), (vs, vs_strides, (2, 1), 2, min(16, 4 * groups))):
        # (a dimension of one element has no stride to speak of)
        own = [s * es if n > 1 else 0 for s, n in zip(strides[:3], shape)]
        if any(s != x for s, n, x in zip(strides[3:], shape[3:], last) if n > 1) or any(s % unit for s in own):
            raise ValueError("a row's codes and its scales must be contiguous, 16-byte aligned in every other dimension "
                             "(scales of less than 16 bytes a row: as long as that)")
        if written and any(s == 0 and n > 1 for s, n in zip(own, shape)):
            raise ValueError("pages that are written must not overlap themselves or each other")
        out += own
    return (num, hkv, size, d), (num, size, group, *out)


def _grad(pages: Q4Pages) -> bool:
    a, b, c, d = pages
    return a.requires_grad or b.requires_grad or c.requires_grad or d.requires_grad


def _check_rows(k, v, shape, slots, dev):
    n, dtype = k.shape, k.dtype
    if len(n) != 3 or v.shape != n or n[1] != shape[1] or n[2] != shape[3]:
        raise ValueError("k and v must be [N, Hkv, d] of the pages' heads and head_dim")
    if v.dtype is not dtype:
        raise ValueError("rows must have one type")
    if k.get_device() != dev or v.get_device() != dev:
        _other_device()
    _check_ints(slots, "slots", torch.int64, n[0])
    return n, _dtype_code(dtype)


def paged_q4_append(k: torch.Tensor, v: torch.Tensor, pages: Q4Pages, slots: torch.Tensor) -> None:
    """Rows ``k``, ``v`` [N, Hkv, d] (float32 or bfloat16, any strides) quantised into their ``slots`` (int64 [N]) of
    ``pages``, one launch of ``bfly_paged_q4_append``.

    A group's bias is the bf16 of its least element, its scale that of a 15th of its range (1e-8 at least), a code the
    nearest whole number to ``(x - bias) / scale`` (the even one of two) within 0..15, in 64-bit arithmetic.  A group
    that holds an infinity or NaN, or whose bias or scale is one in bf16, reads as NaN.  A row whose slot is negative or beyond the pages is
    passed over.  The slots of a call are distinct, as a plan gives them.  head_dim 64, 128 or 256."""
    dev = _device_of(slots)
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_q4_append(k, v, pages, slots)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or _grad(pages)):
        raise ValueError(_GRAD)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed(k, v, *pages)
    shape, packed = _pages(pages, dev, True)
    (n, hkv, d), code = _check_rows(k, v, shape, slots, dev)
    if n == 0:
        return
    (k, k0, k1), (v, v0, v1) = _rows(k), _rows(v)
    slots = slots.contiguous()
    _native.call("bfly_paged_q4_append", _APPEND(
        k.data_ptr(), v.data_ptr(), code, n, hkv, d, k0, k1, v0, v1, slots.data_ptr(), *packed), stream_of(dev))


def paged_q4_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pages: Q4Pages, slots: torch.Tensor,
                         positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                         q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                         eps: float = 1e-6) -> torch.Tensor:
    """The projection tail of a layer over pages in 4 bits, one launch of ``bfly_paged_q4_rope_append``: RMSNorm of
    each head of ``q`` [N, Hq, d] and ``k`` [N, Hkv, d] with ``q_weight`` / ``k_weight`` [d] (both ``None``: no
    norm), rotate-half RoPE at each row's own position, and ``k`` and ``v`` quantised into their ``slots`` (as
    :func:`paged_q4_append`).  Returns the rotated ``q`` [N, Hq, d].

    ``cos`` and ``sin`` [rows, r] (float32) are whole tables, ``positions`` (int64 [N]) picks their rows; elements
    from ``r`` on are not rotated.  q, k and v may be column ranges of one fused projection.  Every row of q is computed,
    in 32 bits and rounded once; k is computed in 64 bits up to its codes, which so do not depend on the order of a sum.
    (Rows that come normed and rotated in bfloat16, as a prompt's do through :func:`paged_q4_append`, have been rounded once
    before that.)  A position outside the tables gives NaN.  head_dim 64, 128 or 256, ``r`` a multiple of 16."""
    dev = _device_of(q)
    if not slots.get_device() == positions.get_device() == cos.get_device() == sin.get_device() == dev:
        _other_device()
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_q4_rope_append(q, k, v, pages, slots, positions, cos, sin, q_weight=q_weight, k_weight=k_weight,
                                        eps=eps)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or cos.requires_grad
                                    or sin.requires_grad or _grad(pages)
                                    or q_weight is not None and q_weight.requires_grad
                                    or k_weight is not None and k_weight.requires_grad):
        raise ValueError(_GRAD)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed(q, k, v, *pages, cos, sin, q_weight, k_weight)
    shape, packed = _pages(pages, dev, True)
    (n, hkv, d), code = _check_rows(k, v, shape, slots, dev)
    sq, dtype = q.shape, q.dtype
    if len(sq) != 3 or sq[0] != n or sq[2] != d or dtype is not k.dtype:
        raise ValueError("q must be [N, Hq, d] rows of k's type")
    hq = sq[1]
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
    (q, q0, q1), (k, k0, k1), (v, v0, v1) = _rows(q), _rows(k), _rows(v)
    slots, positions, cos, sin = slots.contiguous(), positions.contiguous(), _flat(cos), _flat(sin)
    _native.call("bfly_paged_q4_rope_append", _ROPE(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), code, n, hq, hkv, d, q0, q1, k0, k1, v0, v1, qw, kw, eps, cos.data_ptr(),
        sin.data_ptr(), table[0], table[1], positions.data_ptr(), slots.data_ptr(), out.data_ptr(), *packed), stream_of(dev))
    return out


def paged_q4_read(pages: Q4Pages, block_table: torch.Tensor, tokens: int, *,
                  dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``tokens`` keys and values of every request as dense [B, Hkv, tokens, d] tensors of ``dtype`` (float32:
    what the codes stand for; bfloat16: rounded once), one launch of ``bfly_paged_q4_read``.

    ``block_table`` int32 [B, pages]; ``tokens`` at most what its rows hold.  Rows whose page id is outside the pages read as
    NaN."""
    dev = _device_of(block_table)
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_q4_read(pages, block_table, tokens, dtype=dtype)
    if torch.is_grad_enabled() and _grad(pages):
        raise ValueError(_GRAD)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed(*pages)
    (_, hkv, size, d), packed = _pages(pages, dev, False)
    b, code, tokens = block_table.shape[0], _dtype_code(dtype), index(tokens)
    stride, width = _table_stride(block_table, b), block_table.shape[1]
    if not 0 <= tokens <= width * size:
        raise ValueError(f"tokens {tokens} must be at most the {width * size} of a block table row")
    k, v = (_EMPTY((b, hkv, tokens, d), (hkv * tokens * d, tokens * d, d, 1), dtype=dtype, device=block_table.device)
            for _ in range(2))
    _native.call("bfly_paged_q4_read", _READ(code, b, hkv, d, tokens, block_table.data_ptr(), width, stride, k.data_ptr(),
                                             v.data_ptr(), *packed), stream_of(dev))
    return k, v


def paged_q4_attention(q: torch.Tensor, pages: Q4Pages, block_table: torch.Tensor, lengths: torch.Tensor, *,
                       scale: Optional[float] = None, window: int = 0, return_stats: bool = False):
    """One new token of every request over its pages in 4 bits (``bfly_paged_q4_attention``):
    :func:`butterfly_amd.paged_attention` over the keys and values that the codes stand for, which are not rounded on
    the way (``q`` and the result are float32 or bfloat16, sums and softmax in 32 bits).

    ``q`` [B, Hq, 1, d]; request ``b`` sees positions ``[max(0, lengths[b] - window), lengths[b])`` of its pages
    (``window`` 0: all of them), query head ``h`` those of kv head ``h // (Hq / Hkv)``.  ``block_table`` int32 [B, pages],
    ``lengths`` int32 [B].  ``scale`` defaults to ``1 / sqrt(d)``.

    Returns ``out`` [B, Hq, 1, d], with ``return_stats`` the stream ``(out, l, m)`` of ``swa_stream_attention``.  A request
    without tokens gives zeros and the empty stream ``(0, 0, -1e30)``; a length beyond its table row, or a page id outside
    the pages among those that are read, gives NaN for that request.  An infinity or NaN in a query gives NaN for its head, a
    NaN in k's scales for its kv head's, in v's in that group.  (An infinity in a scale or bias, which rows into pages never
    leave there, gives infinities or NaN, or takes its key's weight.)  Rows of a page that the request does not see are never
    part of the result, whatever they hold.  Queries of 2^110 and more, or of 2^107 and more times the size of ``scale``, and
    scales of v of 2^80 and more, may give infinities or NaN; values whose weighted sum passes 2^124 give infinities (sums keep
    a reference while weights are at most 2^4, and are divided by ``l`` at the end)."""
    dev = _device_of(q)
    if not block_table.get_device() == lengths.get_device() == dev:
        _other_device()
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return paged_q4_attention(q, pages, block_table, lengths, scale=scale, window=window, return_stats=return_stats)
    if torch.is_grad_enabled() and (q.requires_grad or _grad(pages)):
        raise ValueError(_GRAD)
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        _check_followed(q, *pages)
    (_, hkv, size, d), packed = _pages(pages, dev, False)
    sq, dtype = q.shape, q.dtype
    if len(sq) != 4 or sq[2] != 1 or sq[3] != d:
        raise ValueError("q must be [B, Hq, 1, d] of the pages' head_dim")
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
        need = _workspace_bytes(code, b, hq, hkv, d, width, size, window)
        if need:
            ws = _EMPTY((need,), (1,), dtype=torch.uint8, device=cuda)
        _native.call("bfly_paged_q4_attention", _ATTN(
            q.data_ptr(), code, b, hq, hkv, d, q0, q1, *packed, block_table.data_ptr(), width, stride, lengths.data_ptr(),
            window, 1.0 / math.sqrt(d) if scale is None else scale, out.data_ptr(), lp, mp, 0 if ws is None else ws.data_ptr(),
            need), stream_of(dev))
    return (out, l, m) if return_stats else out


@lru_cache(maxsize=1024)
def _workspace_bytes(*sizes: int) -> int:
    return _native.lib().bfly_paged_q4_attention_workspace_bytes(*sizes)


class PagedQ4Layer(PagedLayer):
    """One layer's pages of a :class:`butterfly_amd.PagedKVCache` in 4 bits, as :class:`butterfly_amd.PagedLayer`."""

    def __init__(self, cache, pages: Q4Pages):
        super().__init__(cache, None, None)
        self.pages = pages

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's rows of keys and values [N, Hkv, d] into their slots."""
        paged_q4_append(k, v, self.pages, self.plan.slots)

    def rope_append(self, q, k, v, cos, sin, *, q_weight=None, k_weight=None, eps: float = 1e-6) -> torch.Tensor:
        """The step's projection rows: :func:`paged_q4_rope_append` at the plan's positions and slots."""
        p = self.plan
        return paged_q4_rope_append(q, k, v, self.pages, p.slots, p.positions, cos, sin, q_weight=q_weight,
                                    k_weight=k_weight, eps=eps)

    def attend(self, q: torch.Tensor, *, scale: Optional[float] = None, window: int = 0, return_stats: bool = False):
        """:func:`paged_q4_attention` of one new token ``q`` [B, Hq, 1, d] of every request over its pages."""
        return paged_q4_attention(q, self.pages, self.cache.block_table, self.plan.lengths, scale=scale, window=window,
                                  return_stats=return_stats)

    def history(self, tokens: int, request: Optional[int] = None):
        """The first ``tokens`` keys and values of every request, or of one, as dense [B, Hkv, tokens, d] tensors of
        the rows' type; the requests hold that many."""
        table = self.cache.block_table
        if request is not None:
            table = table[request:request + 1]
        return paged_q4_read(self.pages, table, tokens, dtype=self.cache.dtype)
