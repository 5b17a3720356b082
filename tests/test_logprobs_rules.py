"""bfly_token_logprobs' argument checks, without a GPU: every refusal comes before any launch."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd import _native

I = 4096   # stands for an aligned device pointer, never followed


def _call(**kw):
    a = dict(logits=I, dtype=1, rows=4, vocab=100, stride=100, tokens=I, top=5, lp=I, h=I, tl=I, tt=I, ws=I, ws_bytes=1 << 40)
    assert set(kw) <= set(a)
    return _native.lib().bfly_token_logprobs(*{**a, **kw}.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), b"dtype"), (dict(vocab=0), b"shape"), (dict(vocab=1 << 30), b"shape"), (dict(rows=-1), b"shape"),
    (dict(top=65), b"top"), (dict(top=-1), b"top"), (dict(vocab=4), b"top"), (dict(stride=-1), b"stride"),
    (dict(logits=None), b"null"), (dict(tokens=None), b"null"), (dict(h=None), b"null"), (dict(tl=None), b"null"),
    (dict(logits=I + 1), b"aligned"), (dict(dtype=0, logits=I + 2), b"aligned"), (dict(rows=1 << 24), b"too many"),
    (dict(vocab=100000, ws=None), b"workspace"), (dict(vocab=100000, ws_bytes=100), b"workspace"),
    (dict(vocab=100000, ws=I + 8), b"workspace"),
])
def test_refused_before_launch(kw, msg):
    assert _call(**kw) == _native.ERR_INVALID
    assert msg in _native.lib().bfly_last_error()


def test_no_rows_and_workspace():
    assert _call(rows=0, logits=None, tokens=None) == 0
    need = _native.lib().bfly_token_logprobs_workspace_bytes
    assert need(0, 100, 5) == 0 and need(4, 100, 5) == 0 and need(5000, 151936, 5) == 0
    assert 0 < need(1, 151936, 0) < need(1, 151936, 5) < need(2, 151936, 5)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        bf.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))
