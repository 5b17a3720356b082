"""What the bound of test_gpu_paged_q4_norms.py tells apart, on the oracle alone."""
from __future__ import annotations

import torch

from .test_gpu_paged_q4_norms import _room


def test_the_bound_tells_lost_values_and_coarser_weights():
    """9000 keys and 32 rows of weights exp(2 N(0, 1)).  Rounding to bf16 is inside the bound.  Weights of one bf16 part add
    as much again as the rounding, so their norm is some 1.4 times its, and the bound's six deviations over 4096 elements are a few
    percent.  A key that has its row's root mean square weight is 1 / sqrt(9000) of the output, 1.05 %, six times the bound."""
    g = torch.Generator().manual_seed(5)
    v = torch.randn(9000, 128, generator=g).double()
    p = (torch.randn(32, 9000, generator=g).double() * 2).exp()
    l = p.sum(-1, keepdim=True)
    want = p @ v / l
    room = _room(want)
    assert (want.bfloat16().double() - want).norm() <= room
    coarse = p.bfloat16().double() @ v / l
    assert (coarse.bfloat16().double() - want).norm() > room
    rms = p.pow(2).mean(-1, keepdim=True).sqrt()
    lost = p.scatter(1, (p - rms).abs().argmin(-1, keepdim=True), 0.0) @ v / l
    assert (lost.bfloat16().double() - want).norm() > room
