"""GPU: one-token attention over 4-bit pages near the ends of fp32, against 64 bits."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf

from .test_gpu_paged_q4 import _check, _gen, _i32, _pages, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 64)])
@pytest.mark.parametrize("scale,power", [(1.0, 104), (8.0, 101), (-0.125, 104), (2.0 ** -20, 106)])
def test_large_queries_under_a_scale_that_does_not_shrink_them(dtype, d, group, scale, power):
    """The largest query times the scale up to 2^107, over keys small enough for scores of some unit's size.  (A score of 1
    is at least 2^-127 on the way, so fp32's smallest number, 2^-149, is 2^-22 of one: 24 such roundings are far inside
    the bound, 24 u of terms that sum to 50 and more.)"""
    lens = [500, 33, 200]
    pages = _pages(30, 2, 32, d, group)
    pages.k_scales.mul_(2.0 ** (-power - 3) / abs(scale))
    table = _table(lens, 32, 30)
    q = torch.randn(3, 8, 1, d, generator=_gen(1), device="cuda").clamp(-7.5, 7.5)
    q[:, 0, 0, 3] = 7.5
    q = (q * 2.0 ** power).to(dtype)
    out, l, m = bf.paged_q4_attention(q, pages, table, _i32(lens), scale=scale, return_stats=True)
    assert bool(out.isfinite().all())
    _check(out, q, pages, table, _i32(lens), (l, m), scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 64)])
def test_large_values_under_their_limits(dtype, d, group):
    """Scales of v just below 2^80, and biases whose sum over 500 keys of weight 2^4 at most stays below 2^124."""
    lens = [500, 33, 200]
    pages = _pages(30, 2, 32, d, group)
    table = _table(lens, 32, 30)
    q = torch.randn(3, 8, 1, d, generator=_gen(1), device="cuda").to(dtype)
    for scales, biases in ((80, 80), (0, 108)):
        big = bf.Q4Pages(*(t.clone() for t in pages))
        assert float(big.v_scales[..., 0].max()) < 1 and float(big.v_scales[..., 1].abs().max()) < 8
        big.v_scales[..., 0].mul_(2.0 ** scales)
        big.v_scales[..., 1].mul_(2.0 ** biases)
        out = bf.paged_q4_attention(q, big, table, _i32(lens))
        assert bool(out.isfinite().all())
        _check(out, q, big, table, _i32(lens))
