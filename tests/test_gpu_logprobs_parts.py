"""GPU: ``token_logprobs`` of rows on both sides of where parts begin, against the same in 64 bits.

fp32 sums of exponentials: a thread's run one after another (at most 256 terms of its own for these rows, each rounding 2^-24 of a
partial sum of positive terms), threads, waves and parts pairwise (16 more): 2^-15 at the most, of l and so absolutely of log l; the
terms themselves are rounded to 2^-22 of themselves.  Entropy counts terms up to |x - m| <= 64 times as large in its second
sum, which cancels against log l: 2^-9 at the most."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [8191, 8193, 12000, 16383, 16384, 16385])
@pytest.mark.parametrize("rows,offset", [(1, 0), (33, 0), (7, 3)])
def test_rows_around_the_first_parts(dtype, vocab, rows, offset):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    wide = (torch.randn(rows, vocab + 5, generator=g, device="cuda") * 4).to(dtype)
    x = wide[:, offset:offset + vocab]                  # rows at any alignment
    x[0, vocab // 2:] = x[0, 0]                         # ties through every part
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    got = bf.token_logprobs(x, tokens, top=20)
    lp = x.double().log_softmax(-1)
    near = dict(rtol=2.0 ** -22, atol=2.0 ** -15)
    torch.testing.assert_close(got.logprobs.double(), lp.gather(1, tokens[:, None])[:, 0], **near)
    torch.testing.assert_close(got.entropy.double(), -(lp.exp() * lp).sum(-1), rtol=0, atol=2.0 ** -9)
    order = x.float().sort(stable=True, dim=-1, descending=True).indices[:, :20]
    assert torch.equal(got.top_tokens, order)
    torch.testing.assert_close(got.top_logprobs.double(), lp.gather(1, order), **near)
