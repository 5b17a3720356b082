"""GPU: scales of 4-bit pages where a 15th of a group's range lies next to a border of every rounding on its way.

A range of 15 (1 + 2^-8 + 2^-24) + 2^-49 has the 15th q = 1 + 2^-8 + 2^-24 + 2^-52 in 64 bits (the last bit is the division's:
2^-49 / 15 is more than half a step).  1 + 2^-8 + 2^-24 is a tie between two fp32 numbers, the even one of them 1 + 2^-8 a tie
between two bf16 numbers, the even one of them 1: q is above both borders, its fp32 is 1 + 2^-8 + 2^-23 and its bf16 1 + 2^-7.  Without
its last bit both would fall, to 1.  (The oracle runs on the CPU: on the GPU torch divides by a number by way of its
reciprocal, and has no last bit either.)"""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf

from . import q4_plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_scale_next_to_both_borders(d, group):
    rows, hkv, page = 3, 2, 16
    x = torch.linspace(1.0, 14.0, d, device="cuda").repeat(rows, hkv, 1)
    cos, sin = torch.ones(4, d, device="cuda"), torch.zeros(4, d, device="cuda")
    hi, lo = torch.arange(3, d, group), torch.arange(5, d, group)
    # the least element (2^25 - 1) 2^-49 as a rotation's product: 31 * 601 and 1801 2^-49
    x[..., hi] = 15 * (1 + 2.0 ** -8) + 2.0 ** -20
    x[..., lo], cos[:, lo] = 18631.0, 1801 * 2.0 ** -49
    positions = torch.arange(rows, device="cuda")
    want = q4_plain.rope(x, None, cos, sin, positions, 0.0).cpu()
    assert float(want.amax() - want.amin()) == 15 * (1 + 2.0 ** -8 + 2.0 ** -24) + 2.0 ** -49
    pages = bf.empty_q4_pages(2, hkv, page, d, group=group)
    bf.paged_q4_rope_append(x, x, x, pages, positions, positions, cos, sin)
    codes, scales = q4_plain.packed(want, group)
    assert bool((scales[..., 0] == 1 + 2.0 ** -7).all())
    assert torch.equal(pages.k_scales[0, :, :rows].transpose(0, 1).cpu(), scales)
    assert torch.equal(pages.k_codes[0, :, :rows].transpose(0, 1).cpu(), codes)
