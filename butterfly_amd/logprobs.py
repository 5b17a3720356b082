"""Log probabilities of given tokens, with entropy and the top alternatives, from a decoder's logits.

What a decoder reports beside the tokens it picks, and what a text is scored with
(``butterfly_amd.decoder.Decoder.score``).  The reference compares its swapped models' top entries and divergence on host
arrays (scripts/quality_smoke.py); this is one pass over the logits on the device.
"""
from __future__ import annotations

from functools import lru_cache
from operator import index
from typing import NamedTuple

import torch
from torch import _C
from torch.autograd import forward_ad

from . import _native
from ._device import _GET_DEVICE, stream_of

MAX_TOP = 64
_EMPTY = torch.empty_strided


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` gives: ``logprobs`` and ``entropy`` [...] (float32), ``top_logprobs`` [..., top]
    (float32) and ``top_tokens`` [..., top] (int64), the most probable first."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """The log probabilities of ``tokens`` (int64 [...]) under the softmax of ``logits`` [..., vocab] (float32 or
    bfloat16), that softmax's entropy (nats) and its ``top`` most probable tokens, one pass of ``bfly_token_logprobs``.

    A token outside the vocabulary gives NaN (a row without a next token: -1).  Equal logits rank by the lower token, NaN
    above every number.  A logit of -inf has probability 0 (log probability -inf); a row that holds a NaN or +inf, or
    nothing but -inf, gives NaN.  Sums are held in 32 bits.  ``top`` at most 64 and at most the vocabulary; vocabularies
    below 2^30.  Rows may lie at any distance; logits that are not contiguous in the vocabulary are copied.

    Runs on the current stream of its tensors' device, allocates only its outputs and a workspace of its own, and can be
    captured in a HIP graph.  For inference: it refuses logits that require gradients (with gradients enabled) or carry
    tangents, and traces."""
    dev = logits.get_device()
    if dev < 0:
        raise ValueError("butterfly_amd operators take GPU tensors (device 'cuda')")
    if tokens.get_device() != dev:
        raise ValueError("all tensors must be GPU tensors of one device")
    if dev != _GET_DEVICE():
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, top=top)
    if torch.is_grad_enabled() and logits.requires_grad:
        raise ValueError("token_logprobs is for inference: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 or _C._get_tracing_state() is not None:
        if _C._get_tracing_state() is not None:
            raise ValueError("token_logprobs cannot be traced: a trace would hold this call's result as a constant")
        if forward_ad.unpack_dual(logits).tangent is not None:
            raise ValueError("token_logprobs is for inference: call it without tangents")
    dtype = logits.dtype
    if dtype is torch.bfloat16:
        code = _native.DTYPE_BF16
    elif dtype is torch.float32:
        code = _native.DTYPE_F32
    else:
        raise ValueError(f"unsupported dtype {dtype}; expected float32 or bfloat16")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must be [..., vocab]")
    shape, vocab, top = logits.shape[:-1], logits.shape[-1], index(top)
    if tokens.dtype is not torch.int64 or tokens.shape != shape:
        raise ValueError(f"tokens must be an int64 tensor of shape {list(shape)}")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top {top} must be 0 to {min(MAX_TOP, vocab)}")
    if logits.dim() != 2:
        logits = logits.reshape(-1, vocab)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.clone(memory_format=torch.contiguous_format)
    tokens = tokens.contiguous()
    rows, cuda = logits.shape[0], logits.device
    f32, many = torch.float32, (*shape, top)
    strides, by = (1,) if len(shape) == 1 else _strides(shape), _strides(many)
    logprobs, entropy = _EMPTY(shape, strides, dtype=f32, device=cuda), _EMPTY(shape, strides, dtype=f32, device=cuda)
    tops, ids = _EMPTY(many, by, dtype=f32, device=cuda), _EMPTY(many, by, dtype=torch.int64, device=cuda)
    if rows:
        need = _workspace_bytes(rows, vocab, top)
        ws = _EMPTY((need,), (1,), dtype=torch.uint8, device=cuda) if need else None
        _native.call("bfly_token_logprobs", logits.data_ptr(), code, rows, vocab, logits.stride(0) if rows > 1 else vocab,
                     tokens.data_ptr(), top, logprobs.data_ptr(), entropy.data_ptr(), tops.data_ptr(), ids.data_ptr(),
                     0 if ws is None else ws.data_ptr(), need, stream_of(dev))
    return TokenLogprobs(logprobs, entropy, tops, ids)


def _strides(shape):
    """Strides of a contiguous tensor."""
    out, n = [], 1
    for s in reversed(shape):
        out.append(n)
        n *= max(1, s)
    return tuple(reversed(out))


@lru_cache(maxsize=1024)
def _workspace_bytes(*sizes: int) -> int:
    return _native.lib().bfly_token_logprobs_workspace_bytes(*sizes)
