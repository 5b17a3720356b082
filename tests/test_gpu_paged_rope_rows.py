"""GPU: paged_rope_append on both sides of the rule that gives a group of lanes one head or four of a token."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                # half a step of fp32
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, F32: U}


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv,rot,norm", [(5, 1, 0, True), (6, 2, 32, True), (7, 7, 48, False)])
def test_rope_append_on_both_sides_of_its_row_rule(dtype, d, hq, hkv, rot, norm):
    """Few rows take a head to a group of lanes, from 2^16 heads' rows on four of a token (here with borders of q, k and v
    inside a four, and fours that are not full): the same values, bit for bit, and the formula's."""
    rot, heads, page = rot or d, hq + 2 * hkv, 64
    edge = -(-(1 << 16) // heads)
    g = torch.Generator(device="cuda").manual_seed(d + heads)
    n = edge + 3
    x = torch.randn(n, heads, d, generator=g, device="cuda").to(dtype)
    ang = torch.rand(500, rot // 2, generator=g, device="cuda").repeat(1, 2) * 6
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(500, (n,), generator=g, device="cuda")
    pages = -(-n // page) + 2
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
    slots[5], slots[n - 2], slots[n - 4] = -1, pages * page, -7
    pos[9], pos[n - 1] = 500, -1
    w = [(torch.rand(d, generator=g, device="cuda") + 0.5).to(dtype) for _ in range(2)] if norm else [None, None]
    q, k, v = x.split((hq, hkv, hkv), 1)

    def run(parts):
        kp, vp = (torch.zeros(pages, hkv, page, d, dtype=dtype, device="cuda") for _ in range(2))
        out = [bf.paged_rope_append(q[i:j], k[i:j], v[i:j], kp, vp, slots[i:j], pos[i:j], cos, sin, q_weight=w[0],
                                    k_weight=w[1], eps=1e-5) for i, j in parts]
        return torch.cat(out), kp, vp

    whole = run([(0, n)])
    for parts in ([(0, edge - 1), (edge - 1, n)], [(0, edge), (edge, n)]):
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(run(parts), whole))
    out, kp, vp = whole
    live = (slots >= 0) & (slots < pages * page)
    off = (pos < 0) | (pos >= 500)
    at, row = slots[live] // page, slots[live] % page
    want = torch.zeros_like(vp)
    want[at, :, row] = v[live]
    assert torch.equal(vp, want)
    got_k = torch.full_like(k, 0)
    got_k[live] = kp[at, :, row]
    kp[at, :, row] = 0
    assert bool((kp == 0).all())                     # nothing else was written
    c, s = (t[pos.clamp(0, 499)].double()[:, None] for t in (cos, sin))
    for got, y, wt, rows in ((out, q, w[0], torch.ones_like(live)), (got_k, k, w[1], live)):
        y = y.double()
        if wt is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * wt.double()
        r = y[..., :rot]
        turned = torch.cat([-r[..., rot // 2:], r[..., :rot // 2]], -1)
        z = torch.cat([r * c + turned * s, y[..., rot:]], -1)
        size = torch.cat([(r * c).abs() + (turned * s).abs(), y[..., rot:].abs()], -1)
        bound = size * (d / 2 + 16) * U              # the mean square's sum, rsqrt, three products, a sum
        ok = (got.double() - z).abs() <= bound + HALF_STEP[dtype] * (z.abs() + bound)
        assert bool(ok[rows & ~off].all()) and bool(torch.isnan(got[rows & off]).all())
