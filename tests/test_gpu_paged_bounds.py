"""GPU: paged attention where the arithmetic leaves next to nothing to a tolerance, so that a key left out or taken twice
or weights of fewer bits show.

u = 2^-24 is half a step of fp32; scores are made of small whole numbers and powers of two, exact in fp32."""
from __future__ import annotations

import random

import pytest
import torch

import butterfly_amd as bf

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, F32: U}
NAN = float("nan")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(lens, page, seed, width=None):
    """A block table over pages in random order, and how many pages there are."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.full((len(lens), width or max(need) + 1), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.cuda(), len(order)


def _rows(pages, table, b, n):
    """Request b's first n rows [Hkv, n, d]."""
    ids = table[b, :-(-n // pages.shape[2])].long()
    return pages[ids].transpose(0, 1).flatten(1, 2)[:, :n]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [5, 16, 33])
def test_fp32_weights_have_the_precision_of_fp32(d, n):
    """V's rows are unit vectors, so output j is weight j.  A weight's own error: the argument of exp2 has two roundings of
    |s - m| log2(e), exp2 and the factor between two waves' maxima 2 u each and a product's rounding; the sum
    adds n - 1 roundings; then a quotient (5 u) and a product."""
    hq, hkv, page, b = 32, 2, 16, 8
    g = torch.Generator().manual_seed(n + d)
    table, pages = _tables([n] * b, page, n)
    k = torch.randint(-2, 3, (pages, hkv, page, d), generator=g).float().cuda()
    v = torch.full_like(k, NAN)
    for r in range(b):
        for t in range(n):
            v[table[r, t // page].long(), :, t % page] = torch.eye(d, device="cuda")[t]
    q = torch.randint(-2, 3, (b, hq, 1, d), generator=g).float().cuda()
    scale = 0.125
    o, l, m = bf.paged_attention(q, k, v, table, _i32([n] * b), scale=scale, return_stats=True)
    dense = torch.stack([_rows(k, table, r, n) for r in range(b)]).double().repeat_interleave(hq // hkv, 1)
    s = (dense @ q[:, :, 0, :, None].double())[..., 0] * scale
    top = s.amax(-1, keepdim=True)
    p = (s - top).exp()
    w = p / p.sum(-1, keepdim=True)
    own = 2 * (top - s) + 8
    total = (w * own).sum(-1, keepdim=True) + n
    assert torch.equal(m[:, :, 0].double(), top)
    assert bool(((l[:, :, 0].double() - p.sum(-1, keepdim=True)).abs() <= total * U * p.sum(-1, keepdim=True)).all())
    bound = (own + total + 8) * U * w
    assert bool(((o[:, :, 0, :n].double() - w).abs() <= bound).all())
    assert bool((o[:, :, 0, n:] == 0).all())
    if n <= 16:                                     # weights of two bf16 parts would be outside
        high = w.bfloat16().double()
        assert bool((((high + (w - high).bfloat16().double()) - w).abs() > bound).any())


CASES = [([20011], 8, 2, 64), ([70001], 16, 4, 64), ([1, 9000, 0, 3], 4, 2, 64), ([4097] * 5, 2, 1, 16), ([513, 511, 512, 1025], 5, 1, 32)]
# many requests, some of them beyond what stays one run for so many pairs of request and kv head
MANY = [(70, 8, 2), (130, 8, 4), (520, 8, 4), (300, 40, 2)]


def _many(count, longest=12000):
    r = random.Random(count)
    lens = [r.choice([0, 1, 17, 64, r.randint(1, 300)]) for _ in range(count)]
    lens[0], lens[count // 2], lens[count - 1] = longest, longest // 2 + 1, longest - 77
    return lens


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,hq,hkv,page", CASES + [(_many(b), hq, hkv, 64) for b, hq, hkv in MANY],
                         ids=[f"{len(c[0])}x{max(c[0])}" for c in CASES] + [f"many{b}" for b, _, _ in MANY])
def test_every_key_counts_once(dtype, d, lens, hq, hkv, page):
    """All scores are 0: weights are 1 and sums of whole numbers exact (below 2^24), so l is the number of keys, and an output
    their mean up to a quotient, a product and its rounding."""
    g = torch.Generator(device="cuda").manual_seed(len(lens))
    table, pages = _tables(lens, page, len(lens))
    k = torch.zeros(pages, hkv, page, d, dtype=dtype, device="cuda")
    v = torch.randint(-8, 9, k.shape, generator=g, device="cuda").to(dtype)
    q = torch.randn(len(lens), hq, 1, d, generator=g, device="cuda").to(dtype)
    for window in (0, 5000):
        o, l, m = bf.paged_attention(q, k, v, table, _i32(lens), window=window, return_stats=True)
        for b, n in enumerate(lens):
            if n < 400 and b % 16:                  # (the short ones of many: some)
                continue
            lo = max(0, n - window) if window else 0
            assert bool((l[b] == n - lo).all()) and bool((m[b] == (0 if n else -1e30)).all())
            if n:
                want = (_rows(v, table, b, n)[:, lo:].double().sum(1) / (n - lo)).repeat_interleave(hq // hkv, 0)
                assert bool(((o[b, :, 0].double() - want).abs() <= (HALF_STEP[dtype] + 8 * U) * want.abs()).all()), (b, n, window)
            else:
                assert bool((o[b] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,d,page", [(20011, 64, 64), (9001, 128, 16), (5000, 256, 1024)])
def test_a_key_on_either_side_of_every_edge_is_found(dtype, n, d, page):
    """Keys are vectors of +-1 and each query is one of them: its score is d, the others' are at most half of it, and the
    output is its value (the others add at most 16 n exp(-d / 2) < 2^-24 of the largest).  The keys asked for lie on both
    sides of every multiple of 64, so of every edge of a tile, a round and a run."""
    hkv, group, b = 2, 16, 2
    g = torch.Generator(device="cuda").manual_seed(n)
    table, pages = _tables([n], page, n)
    k = (torch.randint(0, 2, (pages, hkv, page, d), generator=g, device="cuda") * 2 - 1).to(dtype)
    v = torch.randint(-8, 9, k.shape, generator=g, device="cuda").to(dtype)
    dk, dv = _rows(k, table, 0, n), _rows(v, table, 0, n)
    asked = sorted({t for e in range(0, n + 64, 64) for t in (e - 1, e) if 0 <= t < n} | {n - 1})
    lens = _i32([n] * b)
    for at in range(0, len(asked), b * group):
        ts = torch.tensor((asked[at:at + b * group] * (b * group))[:b * group], device="cuda").view(b, 1, group)
        ts = ts.expand(b, hkv, group)
        head = torch.arange(hkv, device="cuda")[None, :, None]
        q = dk[head, ts].reshape(b, hkv * group, 1, d)
        others = (q.view(b, hkv, group, d).float() @ dk.float().transpose(1, 2)).scatter(3, ts[..., None], -float(d))
        o, l, m = bf.paged_attention(q, k, v, table.expand(b, -1), lens, scale=1.0, return_stats=True)
        want = dv[head, ts].reshape(b, hkv * group, d).double()
        rest = (others.double().amax() - d).exp().item() * n
        assert rest < 2.0 ** -9
        assert bool((m == d).all()) and bool(((l.double() - 1).abs() <= rest + n * U * rest + 2 * U).all())
        assert bool(((o[:, :, 0].double() - want).abs() <= HALF_STEP[dtype] * want.abs() + 8 * U * 8 + 17 * rest).all())
