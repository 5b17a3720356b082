"""GPU: bf16 outputs of one-token attention over long 4-bit pages, held as a whole to their rounding.

An element that is rounded to the nearest from a value x is off by ulp(x) u / 2 with u spread evenly over [-1, 1]: its
square is ulp^2 / 12 in the mean, with a variance of ulp^4 / 180 (1/80 - 1/144 of ulp^4).  Over all elements of a request the sum of
squares is S = sum ulp^2 / 12 in the mean; six deviations above it, sqrt(sum ulp^4 / 180) each, is what chance does not reach.  What
the kernel adds before that rounding is at most 2^-17 of the weights (two bf16 parts) and 2^-18 from the scores, of errors that
are independent from key to key: 2^-16 of the output's norm, as fp32 outputs are held to.  So |error| <= sqrt(S + 6 dev) + 2^-16 |out|
in the 2-norm, request by request and kv head by kv head.  (Weights of one bf16 part only would be off by 2^-9 of themselves, about twice S.)

Element by element the terms t = 31 scale + |bias| are those of the request's own keys and kv head."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf
from tests import q4_plain

from .test_gpu_paged_q4 import _gen, _i32, _pages, _table

pytestmark = pytest.mark.gpu


def _ulp(x: torch.Tensor) -> torch.Tensor:
    """The distance of bf16 numbers around x (8 bits from the leading one)."""
    return torch.exp2(torch.frexp(x)[1].double() - 8)


def _room(want):
    ulp = _ulp(want)
    return ((ulp ** 2).sum() / 12 + 6 * ((ulp ** 4).sum() / 180).sqrt()).sqrt() + 2.0 ** -16 * want.norm()


@pytest.mark.parametrize("d,group,hq,hkv,lens,page,window", [
    (128, 64, 16, 4, [9000], 128, 0),
    (256, 64, 4, 1, [30000, 100], 256, 0),
    (256, 32, 8, 2, [5000, 700], 32, 0),
    (64, 64, 34, 1, [4000] * 3, 16, 0),
    (64, 32, 8, 2, [40000, 17], 64, 0),
    (128, 32, 8, 8, [12000, 0, 7000], 128, 8001),
    (128, 64, 4, 2, [700] * 40 + [40000], 128, 0),
    (128, 64, 8, 2, [1024, 1023, 1], 16, 0),
])
@pytest.mark.parametrize("spread", [1.0, 2.0])
def test_bf16_outputs_are_as_near_as_their_rounding(d, group, hq, hkv, lens, page, window, spread):
    pages = _pages(sum(-(-n // page) for n in lens) + 1, hkv, page, d, group, spread=spread)
    table = _table(lens, page, pages.k_codes.shape[0])
    q = torch.randn(len(lens), hq, 1, d, generator=_gen(3), device="cuda").bfloat16()
    out = bf.paged_q4_attention(q, pages, table, _i32(lens), window=window)
    want = q4_plain.attention(q, *pages, table, _i32(lens), window=window)[0]
    sc = pages.v_scales.double().abs()
    terms = (31 * sc[..., 0] + sc[..., 1]).amax(-1)                   # [pages, hkv, row]
    g = hq // hkv
    for b, n in enumerate(lens):
        if n == 0:
            assert not bool(out[b].any())
            continue
        seen = slice(max(0, n - window) if window else 0, n)
        for h in range(hkv):
            t = terms[table[b, :-(-n // page)].long(), h].flatten()[seen].max()
            got, w = out[b, h * g:(h + 1) * g].double(), want[b, h * g:(h + 1) * g]
            assert bool(((got - w).abs() <= _ulp(w) / 2 + 2.0 ** -15 * t).all()), (b, h)
            # (few elements: the mean says little, six deviations still hold)
            assert (got - w).norm() <= _room(w), (b, h, (got - w).norm() / w.norm(), _room(w) / w.norm())
