"""GPU: the 4-bit paged cache's operators against the same in plain operations and 64 bits (tests/q4_plain.py).

Codes, scales and biases are defined by 64-bit arithmetic and have to be equal, bit for bit.  Tolerances of the
attention, with u = 2^-24 and a row's terms at most t = 31 scale + |bias| of v:
  * scores: sums of d products q c and their scales in fp32, errors of u each that add up like a random
    walk: below 2^-18 of the weights for the sizes here, twice (in the sum and in l);
  * weights: two bf16 parts are off by 2^-17 (half a step of the second one), three by 2^-25;
  * so |error| <= t (2^-17 + 2^-16) = 0.75 * 2^-15 t, rounded up to 2^-15 t, and half a step of the output's type.
A relative 2-norm of 2^-16 holds fp32 outputs to more: their errors are independent, 2^-18 at the most each.
The statistics are held to the worst case.  A score's terms, scale |q_e| (31 scale + |bias|) summed over its elements, are A
at the most (of all rows and keys), and each of its fp32 roundings is of a partial sum of them, so at most u A: some 6
for the products of a group (up to three, of 32 products each, and the bias's term), two for each of up to 8 groups, two
for the scale.  So m is off by at most delta = 24 u A, however small it is itself, and l, a sum of exp(s - m), by a
part of 2 delta and the 2^-18 of its own sum."""
from __future__ import annotations

import math

import pytest
import torch

import butterfly_amd as bf
from tests import q4_plain

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pages(num, hkv, page, d, group, seed=0, spread=1.0):
    """Pages of quantised N(0, spread) rows."""
    g = _gen(seed)
    out = []
    for _ in range(2):
        x = torch.randn(num, hkv, page, d, generator=g, device="cuda") * spread
        out += q4_plain.packed(x, group)
    return bf.Q4Pages(*out)


def _table(lens, page, pages, seed=0, width=None):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    width = max(1, -(-max(lens) // page)) if width is None else width
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        p = min(-(-max(0, n) // page), width)
        table[b, :p] = order[at:at + p]
        at += p
    return table.cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _same(a, b):
    """Equal, NaN where NaN (bf16 scales: -0 is 0)."""
    if a.dtype == torch.uint8:
        return torch.equal(a, b)
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0).float(), b.nan_to_num(7.0).float())


# --------------------------------------------------------------------------- rows into pages
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_equals_the_definition(dtype, d, group):
    g = _gen(d + group)
    for rows, hkv, page, layout in ((1, 1, 16, "rows"), (37, 3, 16, "heads"), (130, 2, 64, "fused"), (5, 4, 1024, "odd")):
        pages = _pages(-(-rows // page) + 2, hkv, page, d, group, seed=rows)
        before = bf.Q4Pages(*(t.clone() for t in pages))
        x = torch.randn(2, rows, hkv, d, generator=g, device="cuda")
        x = (x * torch.rand(d, generator=g, device="cuda") * 4 + torch.randn(2, 1, hkv, 1, generator=g, device="cuda")).to(dtype)
        k, v = x
        if layout == "heads":
            k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
        elif layout == "fused":
            k, v = torch.cat([k, v, k], 1).split(hkv, 1)[:2]
        elif layout == "odd":       # unaligned rows: a copy is made
            buf = torch.empty(2 * rows * hkv * (d + 1), dtype=dtype, device="cuda")
            odd = buf.view(2, rows, hkv, d + 1)[..., 1:]
            odd.copy_(x)
            k, v = odd
        slots = torch.randperm(pages.k_codes.shape[0] * page, generator=torch.Generator().manual_seed(1))[:rows].cuda()
        if rows > 3:
            slots[1], slots[3] = -1, pages.k_codes.shape[0] * page
        bf.paged_q4_append(k, v, pages, slots)
        want = bf.Q4Pages(*(t.clone() for t in before))
        for t, codes, scales in ((k, want.k_codes, want.k_scales), (v, want.v_codes, want.v_scales)):
            c, s = q4_plain.packed(t, group)
            for i, slot in enumerate(slots.tolist()):
                if 0 <= slot < pages.k_codes.shape[0] * page:
                    codes[slot // page, :, slot % page], scales[slot // page, :, slot % page] = c[i], s[i]
        for name, a, b in zip(pages._fields, pages, want):
            assert _same(a, b), (rows, layout, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_of_groups_at_the_edges(dtype):
    big = torch.finfo(dtype).max
    rows = [torch.zeros(64), torch.full((64,), -3.7), torch.full((64,), 1e-30), torch.linspace(-1, 1, 64) * 1e-9,
            torch.linspace(0, 15, 64), torch.arange(64) % 16 + 0.5, torch.arange(64).float() % 31 / 2,
            torch.linspace(-1, 1, 64) * big * 0.99, torch.linspace(1000, 1001, 64), torch.linspace(-1, 1, 64) * 2.0 ** -130]
    for bad in (math.inf, -math.inf, math.nan):
        r = torch.linspace(-1, 1, 64)
        r[17] = bad
        rows.append(r)
    rows.append(torch.full((64,), big))            # rounds to an infinity of bf16 from fp32
    x = torch.stack(rows).to(dtype).cuda()[:, None]
    n = x.shape[0]
    for group in (32, 64):
        pages = _pages(2, 1, 16, 64, group)
        bf.paged_q4_append(x, x.flip(0), pages, torch.arange(n, device="cuda"))
        for t, codes, scales in ((x, pages.k_codes, pages.k_scales), (x.flip(0), pages.v_codes, pages.v_scales)):
            c, s = q4_plain.packed(t, group)
            assert torch.equal(codes[0, 0, :n], c[:, 0]) and _same(scales[0, 0, :n], s[:, 0])
        k, _ = bf.paged_q4_read(pages, _i32([[0]]), n, dtype=torch.float32)
        # a bad group reads as NaN as a whole, the others within half a step and the roundings of scale and bias
        nan = k[0, 0].isnan().view(n, -1, group)
        want = ~torch.isfinite(pages.k_scales[0, 0, :n, :, 0])
        assert torch.equal(nan, want[..., None].expand_as(nan))


def test_scales_are_rounded_to_fp32_and_then_to_bf16():
    """Ranges whose 15th is within 2^-30 of a middle between two bf16 numbers: its fp32 number is that middle, and
    goes to the even one of the two."""
    rows = []
    for t in (1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8):
        for lo in (-2.0 ** -30, 0.0, 2.0 ** -30):
            r = torch.linspace(1, 14, 64)
            r[3], r[40] = lo, 15 * t
            rows.append(r)
    x = torch.stack(rows).cuda()[:, None]
    pages = _pages(1, 1, 16, 64, 64)
    bf.paged_q4_append(x, x, pages, torch.arange(len(rows), device="cuda"))
    assert pages.k_scales[0, 0, :6, 0, 0].tolist() == [1.0] * 3 + [1 + 2.0 ** -6] * 3
    c, s = q4_plain.packed(x, 64)
    assert torch.equal(pages.k_codes[0, 0, :6], c[:, 0]) and _same(pages.v_scales[0, 0, :6], s[:, 0])


# --------------------------------------------------------------------------- norm and RoPE on the way
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (128, 128), (128, 64), (256, 256), (256, 64), (256, 48)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope_append(dtype, d, rot, group):
    g = _gen(d + rot)
    for rows, hq, hkv, norm in ((1, 4, 4, True), (33, 6, 2, True), (50, 5, 1, False)):
        page, context = 32, 300
        pages = _pages(3, hkv, page, d, group)
        fused = torch.randn(rows, hq + 2 * hkv, d, generator=g, device="cuda").to(dtype)
        q, k, v = fused.split((hq, hkv, hkv), 1)
        positions = torch.randint(context, (rows,), generator=g, device="cuda")
        slots = torch.randperm(3 * page, generator=torch.Generator().manual_seed(1))[:rows].cuda()
        if rows > 4:
            slots[2], positions[4], positions[5] = -1, -1, context
        ang = torch.arange(context, device="cuda").double()[:, None] * torch.rand(rot, generator=g, device="cuda").double()
        cos, sin = ang.cos().float(), ang.sin().float()
        qw, kw = ((torch.rand(d, generator=g, device="cuda") + 0.5).to(dtype) for _ in range(2))
        if not norm:
            qw = kw = None
        before = bf.Q4Pages(*(t.clone() for t in pages))
        out = bf.paged_q4_rope_append(q, k, v, pages, slots, positions, cos, sin, q_weight=qw, k_weight=kw, eps=1e-5)
        want = q4_plain.rope(q, qw, cos, sin, positions, 1e-5)
        nan = want.isnan()
        assert out.dtype is dtype and torch.equal(out.isnan(), nan)
        # fp32 on the way: some 8 roundings of the terms (at most 2 max |y| for a rotated pair), then one of the output
        room = HALF[dtype] * want.abs() + 16 * 2.0 ** -24 * want.abs().nan_to_num().amax(-1, keepdim=True)
        assert bool(((out.double() - want).abs() <= room)[~nan].all())
        for t, codes, scales in ((q4_plain.rope(k, kw, cos, sin, positions, 1e-5), before.k_codes, before.k_scales),
                                 (v, before.v_codes, before.v_scales)):
            c, s = q4_plain.packed(t, group)
            live = (slots >= 0).nonzero()[:, 0]
            codes[slots[live] // page, :, slots[live] % page] = c[live]
            scales[slots[live] // page, :, slots[live] % page] = s[live]
        for name, a, b in zip(pages._fields, pages, before):
            assert _same(a, b), (rows, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope_append_of_many_groups_equals_the_definition(dtype):
    """Half a million groups: each rounding of a scale and a bias meets its ties."""
    rows, hq, hkv, d, group = 8000, 8, 8, 256, 32
    q, k, v = torch.randn(rows, hq + 2 * hkv, d, generator=_gen(5), device="cuda").to(dtype).split((hq, hkv, hkv), 1)
    ang = torch.rand(500, d // 4, generator=_gen(2), device="cuda") * 9
    positions = torch.randint(500, (rows,), generator=_gen(3), device="cuda")
    pages = _pages(63, hkv, 128, d, group)
    kw = torch.rand(d, generator=_gen(4), device="cuda").to(dtype)
    bf.paged_q4_rope_append(q, k, v, pages, torch.arange(rows, device="cuda"), positions, ang.cos(), ang.sin(),
                            q_weight=kw, k_weight=kw, eps=1e-6)
    for x, codes, scales in ((q4_plain.rope(k, kw, ang.cos(), ang.sin(), positions, 1e-6), pages.k_codes, pages.k_scales),
                             (v, pages.v_codes, pages.v_scales)):
        c, s = q4_plain.packed(x, group)
        for got, want in ((codes, c), (scales, s)):
            assert _same(got.transpose(1, 2).flatten(0, 1)[:rows], want)


@pytest.mark.parametrize("dtype,d,group,hq,hkv", [(torch.bfloat16, 64, 64, 14, 1), (torch.bfloat16, 128, 32, 6, 6),
                                                  (torch.float32, 256, 64, 5, 5), (torch.bfloat16, 256, 32, 8, 4)])
def test_rope_append_of_many_rows_is_that_of_its_parts(dtype, d, group, hq, hkv):
    """Rows enough that heads are taken four at a time, against calls of a few hundred: the same bits."""
    rows, page = (1 << 17) // (hq + 2 * hkv) + 37, 128
    q, k, v = torch.randn(rows, hq + 2 * hkv, d, generator=_gen(1), device="cuda").to(dtype).split((hq, hkv, hkv), 1)
    ang = torch.rand(500, d // 2, generator=_gen(2), device="cuda") * 9
    positions = torch.randint(-1, 501, (rows,), generator=_gen(3), device="cuda")
    slots = torch.randperm(-(-rows // page) * page, generator=torch.Generator().manual_seed(1))[:rows].cuda()
    slots[5::11] = -1
    qw, kw = (torch.rand(d, generator=_gen(4 + i), device="cuda").to(dtype) for i in range(2))
    outs, pools = [], []
    for part in (rows, 700):
        pages = _pages(-(-rows // page), hkv, page, d, group)
        outs.append(torch.cat([bf.paged_q4_rope_append(a, b, c, pages, s, p, ang.cos(), ang.sin(), q_weight=qw, k_weight=kw, eps=1e-6)
                               for a, b, c, s, p in zip(*(x.split(part) for x in (q, k, v, slots, positions)))]))
        pools.append(pages)
    assert torch.equal(outs[0].nan_to_num(9.0), outs[1].nan_to_num(9.0))
    assert all(_same(a, b) for a, b in zip(*pools))


# --------------------------------------------------------------------------- rows out of pages
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_read(d, group):
    pages = _pages(9, 3, 16, d, group)
    table = _table([60, 41], 16, 9)
    for tokens in (0, 1, 17, 41):
        for dtype in (torch.float32, torch.bfloat16):
            k, v = bf.paged_q4_read(pages, table, tokens, dtype=dtype)
            for got, codes, scales in ((k, pages.k_codes, pages.k_scales), (v, pages.v_codes, pages.v_scales)):
                x = q4_plain.values(codes[table.long().clamp_min(0)], scales[table.long().clamp_min(0)])
                x = x.transpose(1, 2).flatten(2, 3)[:, :, :tokens]
                # (a product of 4 and 8 bits is exact in fp32, the sum rounded once)
                assert got.shape == (2, 3, tokens, d) and torch.equal(got, x.float().to(dtype))
    k, v = bf.paged_q4_read(pages, table, 64, dtype=torch.float32)
    assert bool(k[1, :, 48:].isnan().all()) and bool(v[1, :, 48:].isnan().all())     # entries of -1
    assert not bool(k[0].isnan().any()) and not bool(k[1, :, :48].isnan().any())
    odd = table.clone()
    odd[0, 1] = 9
    assert bool(bf.paged_q4_read(pages, odd, 20)[0][0, :, 16:].isnan().all())


# --------------------------------------------------------------------------- attention
def _check(out, q, pages, table, lengths, stats=None, **kw):
    want, l, m = q4_plain.attention(q, *pages, table, lengths, **kw)
    assert out.dtype is q.dtype and out.shape == q.shape
    nan = want.isnan()
    assert torch.equal(out.isnan(), nan)
    sc = pages.v_scales.double().abs().nan_to_num(0.0, 0.0, 0.0)
    terms = (31 * sc[..., 0] + sc[..., 1]).max()
    err = (out.double() - want).abs()
    assert bool((err <= HALF[q.dtype] * want.abs() + 2.0 ** -15 * terms)[~nan].all()), err[~nan].max()
    if q.dtype is torch.float32:
        assert (out.double() - want)[~nan].norm() <= 2.0 ** -16 * want[~nan].norm()
    if stats is not None:
        sk = pages.k_scales.double().abs().nan_to_num(0.0, 0.0, 0.0)
        each = q.double().abs().unflatten(-1, (sk.shape[3], -1)).sum(-1).flatten(0, 2).amax(0)      # by group
        size = ((31 * sk[..., 0] + sk[..., 1]).flatten(0, 2).amax(0) * each).sum() * abs(kw.get("scale") or q.shape[-1] ** -0.5)
        delta = 24 * 2.0 ** -24 * size
        for got, w, room in ((stats[0], l, (2 * delta + 2.0 ** -18) * l), (stats[1], m, delta + 2.0 ** -23 * m.abs())):
            assert torch.equal(got.isnan(), w.isnan())
            assert bool(((got.double() - w).abs() <= room)[~w.isnan()].all())


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_ragged_requests(dtype, d, group):
    g = _gen(d * group)
    for page, lens, hq, hkv, window in ((16, [1, 0, 17, 300, 33, 32, 31], 4, 2, 0), (64, [700, 65, 128, 5], 16, 1, 0),
                                        (128, [1000, 1, 0, 513], 6, 2, 100), (32, [257, 95], 3, 3, 1), (1024, [1500, 40], 5, 1, 600)):
        pages = _pages(sum(-(-n // page) for n in lens) + 1, hkv, page, d, group, seed=page)
        table = _table(lens, page, pages.k_codes.shape[0])
        q = torch.randn(len(lens), hq, 1, d, generator=g, device="cuda").to(dtype)
        out, l, m = bf.paged_q4_attention(q, pages, table, _i32(lens), window=window, return_stats=True)
        _check(out, q, pages, table, _i32(lens), (l, m), window=window)
        assert torch.equal(bf.paged_q4_attention(q, pages, table, _i32(lens), window=window), out)


@pytest.mark.parametrize("dtype,d,group,hq,hkv,lens,page,window", [
    (torch.bfloat16, 128, 64, 16, 4, [9000], 128, 0),
    (torch.float32, 64, 32, 8, 2, [5000, 3, 20000], 64, 0),
    (torch.bfloat16, 256, 64, 4, 1, [30000, 100], 256, 0),
    (torch.bfloat16, 64, 64, 34, 1, [4000] * 3, 16, 0),               # three 16-row parts of query heads
    (torch.float32, 256, 32, 17, 1, [2500], 32, 0),
    (torch.bfloat16, 128, 32, 8, 8, [12000, 0, 7000], 128, 8001),
    (torch.bfloat16, 128, 64, 4, 2, [700] * 40 + [40000], 128, 0),    # one long request among short ones
])
def test_attention_of_split_requests(dtype, d, group, hq, hkv, lens, page, window):
    pages = _pages(sum(-(-n // page) for n in lens) + 1, hkv, page, d, group, spread=2.0)
    table = _table(lens, page, pages.k_codes.shape[0])
    q = torch.randn(len(lens), hq, 1, d, generator=_gen(3), device="cuda").to(dtype)
    out, l, m = bf.paged_q4_attention(q, pages, table, _i32(lens), window=window, return_stats=True)
    _check(out, q, pages, table, _i32(lens), (l, m), window=window)


@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (6, 2), (14, 2), (17, 1)])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_narrow_and_wide_tables(dtype, d, group, hq, hkv, page):
    """Tables of the same requests on both sides of 2^16 keys in all, where the kernel's form changes: entries behind
    a request's pages say nothing, keys that it does not see are never part of the result."""
    lens, window = [300, 0, 47, 129, 1], 90 if page == 32 else 0
    pages = _pages(sum(-(-n // page) for n in lens) + 1, hkv, page, d, group, seed=hq)
    units = len(lens) * hkv * -(-hq // hkv // 16)
    q = torch.randn(len(lens), hq, 1, d, generator=_gen(hq), device="cuda").to(dtype)
    q[3, 1] *= 8.0                                    # a row whose maximum moves a lot
    seen = torch.zeros(pages.k_codes.shape[0], page, dtype=torch.bool, device="cuda")
    narrow = _table(lens, page, pages.k_codes.shape[0])
    for b, n in enumerate(lens):
        for t in range(max(0, n - window) if window else 0, n):
            seen[int(narrow[b, t // page]), t % page] = True
    for codes, scales in ((pages.k_codes, pages.k_scales), (pages.v_codes, pages.v_scales)):
        codes.masked_fill_(~seen[:, None, :, None], 0xff)
        scales.masked_fill_(~seen[:, None, :, None, None], math.nan)
    clean = bf.Q4Pages(pages.k_codes, pages.k_scales.nan_to_num(0.0), pages.v_codes, pages.v_scales.nan_to_num(0.0))
    for width in (narrow.shape[1], -(-(1 << 16) // (units * page))):
        table = _table(lens, page, pages.k_codes.shape[0], width=width)
        out, l, m = bf.paged_q4_attention(q, pages, table, _i32(lens), window=window, return_stats=True)
        _check(out, q, clean, table, _i32(lens), (l, m), window=window)
        bad = table.clone()
        bad[3, (lens[3] - 1) // page] = pages.k_codes.shape[0]
        bad[4, 0] = -1
        nan = bf.paged_q4_attention(q, pages, bad, _i32(lens), window=window)
        assert bool(nan[3:].isnan().all()) and torch.equal(nan[:3], out[:3])


@pytest.mark.parametrize("scale", [0.0, -0.25, 3.0, 1e-4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_scales(dtype, scale):
    pages = _pages(20, 2, 32, 64, 32)
    lens = [500, 33]
    table = _table(lens, 32, 20)
    q = (torch.randn(2, 4, 1, 64, generator=_gen(1), device="cuda") * 0.5).to(dtype)
    out, l, m = bf.paged_q4_attention(q, pages, table, _i32(lens), scale=scale, return_stats=True)
    _check(out, q, pages, table, _i32(lens), (l, m), scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [-80, -20, 50, 100])
def test_attention_of_small_and_large_queries(dtype, power):
    """Powers of two between queries and scale move every number on the way alike: the same bits."""
    pages, lens = _pages(20, 2, 32, 128, 64), [500, 33]
    table = _table(lens, 32, 20)
    q = (torch.randn(2, 8, 1, 128, generator=_gen(1), device="cuda")).to(dtype)
    want = bf.paged_q4_attention(q, pages, table, _i32(lens), scale=0.125, return_stats=True)
    got = bf.paged_q4_attention(q * 2.0 ** power, pages, table, _i32(lens), scale=0.125 * 2.0 ** -power, return_stats=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_reads_nothing_that_a_request_does_not_see(d, group):
    """NaN and infinities in scales, and any codes, behind the last token, before the window and in free pages."""
    page, lens, window = 32, [40, 75, 33], 20
    pages = _pages(9, 2, page, d, group)
    table = _table(lens, page, 9)
    q = torch.randn(3, 4, 1, d, generator=_gen(2), device="cuda").bfloat16()
    want = bf.paged_q4_attention(q, pages, table, _i32(lens), window=window, return_stats=True)
    seen = torch.zeros(9, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for t in range(n - window, n):
            seen[int(table[b, t // page]), t % page] = True
    for fill in (math.nan, math.inf, -3e38):
        other = bf.Q4Pages(*(t.clone() for t in pages))
        for codes, scales in ((other.k_codes, other.k_scales), (other.v_codes, other.v_scales)):
            codes.masked_fill_(~seen[:, None, :, None], 0xff)
            scales.masked_fill_(~seen[:, None, :, None, None], fill)
        got = bf.paged_q4_attention(q, other, table, _i32(lens), window=window, return_stats=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_of_bad_values_and_tables():
    pages = _pages(6, 2, 16, 64, 32)
    lens = [40, 30, 20]
    q = torch.randn(3, 4, 1, 64, generator=_gen(2), device="cuda")
    for outside in (6, -1, 1 << 30):                  # page ids outside the pages
        table = _i32([[0, 1, 2], [3, outside, 4], [5, 0, outside]])
        out, l, m = bf.paged_q4_attention(q, pages, table, _i32(lens), return_stats=True)
        for x in (out, l, m):
            assert bool(x[1].isnan().all()) and not bool(x[::2].isnan().any())
    table = _table([32, 32], 16, 6)
    over = bf.paged_q4_attention(q[:2], pages, table, _i32([33, 32]))
    assert bool(over[0].isnan().all()) and not bool(over[1].isnan().any())
    neg, l, m = bf.paged_q4_attention(q[:2], pages, table, _i32([-5, 0]), return_stats=True)
    assert not neg.any() and not l.any() and bool((m == -1e30).all())
    # a scale of NaN that is seen: in k the whole head's rows, in v the group's elements
    nan = bf.Q4Pages(*(t.clone() for t in pages))
    nan.k_scales[int(table[0, 1]), 1, 3, 0, 0] = math.nan
    nan.v_scales[int(table[1, 0]), 0, 5, 1, 0] = math.nan
    y = bf.paged_q4_attention(q[:2], nan, table, _i32([32, 32])).isnan()
    assert bool(y[0, 2:].all()) and not bool(y[0, :2].any())
    assert bool(y[1, :2, :, 32:].all()) and not bool(y[1, :2, :, :32].any()) and not bool(y[1, 2:].any())
    # an infinite query
    q2 = q[:2].clone()
    q2[0, 1, 0, 7] = math.inf
    y = bf.paged_q4_attention(q2, pages, table, _i32([32, 32])).isnan()
    assert bool(y[0, 1].all()) and int(y.any(-1).sum()) == 1


def test_attention_weights_one_key_among_many():
    """Each key in turn stands out: the result is its value (to the weight the others keep)."""
    d, n = 128, 200
    pages = _pages(8, 1, 32, d, 64)
    table = _table([n], 32, 8)
    k, v = bf.paged_q4_read(pages, table, n, dtype=torch.float32)
    for t in range(0, n, 7):
        q = k[:, :, t:t + 1].clone()
        out = bf.paged_q4_attention(q, pages, table, _i32([n]), scale=8.0)
        _check(out, q, pages, table, _i32([n]), scale=8.0)


def test_layouts_of_pages_tables_and_queries():
    """Page tensors that are slices of larger ones (layers, heads apart), a block table's columns, strided queries and
    lengths."""
    d, group, hkv, page = 128, 64, 2, 32
    lens = [100, 64, 7]
    base = _pages(10, hkv, page, d, group)
    table = _table(lens, page, 10)
    q = torch.randn(3, 4, 1, d, generator=_gen(2), device="cuda").bfloat16()
    want = bf.paged_q4_attention(q, base, table, _i32(lens))

    def other(t):
        big = torch.zeros(10, 3, hkv + 1, page, *t.shape[3:], dtype=t.dtype, device="cuda")
        view = big[:, 1, 1:]
        view.copy_(t)
        return view

    def rows_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    wide = torch.full((3, 9), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    for pages in (bf.Q4Pages(*map(other, base)), bf.Q4Pages(*map(rows_first, base)),
                  bf.Q4Pages(base.k_codes, other(base.k_scales), other(base.v_codes), base.v_scales)):
        assert torch.equal(bf.paged_q4_attention(q, pages, table, _i32(lens)), want)
        assert torch.equal(bf.paged_q4_attention(q, pages, wide[:, 2:2 + table.shape[1]], _i32(lens)), want)
        assert all(torch.equal(a, b) for a, b in zip(bf.paged_q4_read(pages, table, 32), bf.paged_q4_read(base, table, 32)))
    strided = torch.empty(3, 7, 2, d, dtype=torch.bfloat16, device="cuda")[:, 1:5, 1:]
    strided.copy_(q)
    odd = torch.empty(3, 4, 1, d + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(q)
    both = torch.stack([_i32(lens), _i32([1, 2, 3])], 1)
    for x in (strided, odd, q.expand(3, 4, 1, d)):
        assert torch.equal(bf.paged_q4_attention(x, base, table, both[:, 0]), want)
    k = torch.randn(5, hkv, d, generator=_gen(5), device="cuda")
    slots = torch.tensor([0, 33, 64, 5, 319], device="cuda")
    for make in (other, rows_first):
        pages = bf.Q4Pages(*map(make, base))
        plain = bf.Q4Pages(*(t.clone() for t in base))
        bf.paged_q4_append(k, -k, pages, slots)
        bf.paged_q4_append(k, -k, plain, slots)
        assert all(_same(a, b) for a, b in zip(pages, plain))


def test_offsets_beyond_32_bits():
    """Pages more than 2^32 bytes apart."""
    d, group, page = 64, 64, 16
    stride = (1 << 32) + 4096
    codes = torch.zeros(2 * stride + (1 << 16), dtype=torch.uint8, device="cuda")
    small = _pages(3, 2, page, d, group)
    far = codes.as_strided((3, 2, page, d // 2), (stride, page * d // 2, d // 2, 1))
    far.copy_(small.v_codes)
    scales = torch.zeros(2 * stride // 2 + (1 << 16), dtype=torch.bfloat16, device="cuda")
    fars = scales.as_strided((3, 2, page, 1, 2), (stride // 2, page * 2, 2, 2, 1))
    fars.copy_(small.v_scales)
    pages = bf.Q4Pages(small.k_codes, small.k_scales, far, fars)
    table = _i32([[2, 0, 1]])
    q = torch.randn(1, 4, 1, d, generator=_gen(2), device="cuda")
    assert torch.equal(bf.paged_q4_attention(q, pages, table, _i32([45])), bf.paged_q4_attention(q, small, table, _i32([45])))
    assert torch.equal(bf.paged_q4_read(pages, table, 45)[1], bf.paged_q4_read(small, table, 45)[1])
    k = torch.randn(2, 2, d, generator=_gen(5), device="cuda")
    bf.paged_q4_append(k, k, pages, torch.tensor([40, 47], device="cuda"))
    assert torch.equal(far[2, :, [8, 15]], small.k_codes[2, :, [8, 15]])
    assert torch.equal(fars[2, :, [8, 15]], small.k_scales[2, :, [8, 15]])


def test_no_requests_no_rows():
    pages = _pages(2, 2, 16, 64, 64)
    e = torch.empty
    assert bf.paged_q4_attention(e(0, 4, 1, 64, device="cuda"), pages, e(0, 3, dtype=torch.int32, device="cuda"), _i32([])).shape == (0, 4, 1, 64)
    out = bf.paged_q4_attention(e(2, 4, 1, 64, device="cuda"), pages, e(2, 0, dtype=torch.int32, device="cuda"), _i32([0, 0]))
    assert not out.any()
    none = e(0, 2, 64, device="cuda")
    bf.paged_q4_append(none, none, pages, e(0, dtype=torch.int64, device="cuda"))
    k, v = bf.paged_q4_read(pages, e(0, 3, dtype=torch.int32, device="cuda"), 5)
    assert k.shape == v.shape == (0, 2, 5, 64)


# --------------------------------------------------------------------------- streams, graphs, a decode loop
def test_a_captured_step_of_plan_rows_and_attention():
    """Requests that grow token by token: the plan, the rows and the attention captured together; every replay equals
    the eager step on copies of the same state, with eager work between the replays."""
    d, group, hq, hkv, page, b = 128, 64, 8, 2, 16, 3
    pages = _pages(24, hkv, page, d, group)
    lens = [37, 0, 90]
    state = dict(table=_table(lens, page, 24, width=10), lengths=_i32(lens), state=None)
    used = sum(-(-n // page) for n in lens)
    order = torch.randperm(24, generator=torch.Generator().manual_seed(0)).int()
    free = torch.cat([order[used:], torch.full((used,), -1, dtype=torch.int32)]).cuda()
    st = _i32([24 - used, 0])
    rows = torch.empty(b, hq + 2 * hkv, d, dtype=torch.bfloat16, device="cuda")
    ang = torch.arange(200, device="cuda")[:, None] * torch.rand(d, generator=_gen(1), device="cuda")
    cos, sin = ang.cos(), ang.sin()
    w = (torch.rand(d, generator=_gen(2), device="cuda") + 0.5).bfloat16()
    counts = _i32([1, 1, 1])

    def step(pages, table, lengths, free, st, rows):
        p = bf.paged_plan(table, lengths, counts, free, st, page_size=page, num_rows=b, rows_each=1, in_place=True)
        q, k, v = rows.split((hq, hkv, hkv), 1)
        q = bf.paged_q4_rope_append(q, k, v, pages, p.slots, p.positions, cos, sin, q_weight=w, k_weight=w)
        return bf.paged_q4_attention(q.unsqueeze(2), pages, table, p.lengths, return_stats=True)

    live = (pages, state["table"], state["lengths"], free, st, rows)
    twin = (bf.Q4Pages(*(t.clone() for t in pages)), *(t.clone() for t in live[1:5]), rows)
    rows.copy_(torch.randn(rows.shape, generator=_gen(9), device="cuda"))
    step(*live)
    step(*twin)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = step(*live)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(20):
        rows.copy_(torch.randn(rows.shape, generator=_gen(10 + i), device="cuda"))
        graph.replay()
        want = step(*twin)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
        assert all(_same(x, y) for x, y in zip(live[0], twin[0]))
        assert torch.equal(live[2], twin[2]) and torch.equal(live[1], twin[1])
        if i % 5 == 0:
            _check(want[0], bf_q(twin, rows, cos, sin, w, hq, hkv), twin[0], twin[1], twin[2], want[1:])
        torch.cuda.synchronize()


def bf_q(twin, rows, cos, sin, w, hq, hkv):
    """The step's rotated queries, once more (into pages of their own)."""
    q, k, v = rows.split((hq, hkv, hkv), 1)
    spare = bf.Q4Pages(*(t.clone() for t in twin[0]))
    none = torch.full((rows.shape[0],), -1, dtype=torch.int64, device="cuda")
    return bf.paged_q4_rope_append(q, k, v, spare, none, twin[2].long() - 1, cos, sin, q_weight=w, k_weight=w).unsqueeze(2)


def test_on_another_stream_and_twice_at_once():
    """The same split call on two streams at a time: each has a workspace of its own."""
    pages = _pages(90, 2, 128, 128, 64)
    table = _table([11000], 128, 90)
    qs = [torch.randn(1, 8, 1, 128, generator=_gen(i), device="cuda").bfloat16() for i in range(2)]
    want = [bf.paged_q4_attention(q, pages, table, _i32([11000])) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    lengths = _i32([11000])
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(bf.paged_q4_attention(q, pages, table, lengths))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


# --------------------------------------------------------------------------- refusals
def test_refusals():
    pages = _pages(4, 2, 16, 64, 32)
    kc, ks, vc, vs = pages
    i64 = lambda *x: torch.tensor(x, device="cuda")
    rows = torch.randn(3, 2, 64, device="cuda")
    q = torch.randn(2, 4, 1, 64, device="cuda")
    table, lens, slots, pos = _i32([[0, 1], [2, 3]]), _i32([5, 20]), i64(0, 1, 2), i64(0, 1, 2)
    cos = torch.randn(8, 64, device="cuda")
    att = lambda q=q, p=pages, t=table, n=lens, **kw: bf.paged_q4_attention(q, p, t, n, **kw)
    app = lambda k=rows, v=rows, p=pages, s=slots: bf.paged_q4_append(k, v, p, s)
    rop = lambda q=rows, k=rows, v=rows, p=pages, s=slots, at=pos, c=cos, n=cos, **kw: bf.paged_q4_rope_append(q, k, v, p, s, at, c, n, **kw)
    red = lambda p=pages, t=table, n=5, **kw: bf.paged_q4_read(p, t, n, **kw)
    P = pages._replace
    bad_pages = [P(k_codes=kc.to(torch.int8)), P(v_scales=vs.float()), P(v_codes=vc[:3]), P(k_scales=ks[..., :1]),
                 P(k_scales=ks[:, :, :8]), P(k_codes=kc.transpose(2, 3)), P(k_codes=kc[..., :24]),
                 bf.Q4Pages(*(t[:, :, :12] for t in pages)), bf.Q4Pages(*(t[:0] for t in pages)),
                 P(k_codes=torch.empty(4 * 2 * 16 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(4, 2, 16, 32)),
                 P(k_scales=ks[:, :, :, :1], v_scales=vs[:, :, :, :1].expand(-1, -1, -1, 4, -1)),
                 P(k_codes=kc.cpu())]
    for p in bad_pages:
        for f in (att, app, red):
            with pytest.raises(ValueError):
                f(p=p)
        with pytest.raises(ValueError):
            rop(p=p)
    with pytest.raises(NotImplementedError):
        app(p=bf.Q4Pages(*(torch.zeros(4, 2, 16, *s, dtype=t, device="cuda") for s, t in
                           (((48,), torch.uint8), ((3, 2), torch.bfloat16)) * 2)), k=torch.zeros(3, 2, 96, device="cuda"),
            v=torch.zeros(3, 2, 96, device="cuda"))
    for p in (P(v_codes=kc), P(k_codes=kc[:1].expand(4, -1, -1, -1)), P(v_scales=vs[:, :1].expand(-1, 2, -1, -1, -1))):
        with pytest.raises(ValueError, match="overlap"):
            app(p=p)
    assert att(p=P(v_codes=kc)).shape == q.shape            # (read only: allowed)
    for f in (lambda: att(q=q[:, :3]), lambda: att(q=q.half()), lambda: att(q=q[0]), lambda: att(q=q[..., :32]),
              lambda: att(t=table.long()), lambda: att(t=table[:1]), lambda: att(n=lens.long()), lambda: att(n=lens[:1]),
              lambda: att(window=-1), lambda: att(window=1 << 31), lambda: att(q=q.cpu()), lambda: att(n=lens.cpu()),
              lambda: att(t=table.t()), lambda: app(k=rows[:2]), lambda: app(k=rows[:, :1], v=rows[:, :1]),
              lambda: app(k=rows.half(), v=rows.half()), lambda: app(v=rows.bfloat16()), lambda: app(s=slots.int()),
              lambda: app(s=slots[:2]), lambda: app(k=rows.cpu()), lambda: rop(q=rows[:, :1]), lambda: rop(at=pos.int()),
              lambda: rop(c=cos.double(), n=cos.double()), lambda: rop(c=cos[:0], n=cos[:0]), lambda: rop(c=cos[:, :24], n=cos[:, :24]),
              lambda: rop(q_weight=cos[0]), lambda: rop(q_weight=cos[0].bfloat16(), k_weight=cos[0].bfloat16()),
              lambda: red(n=33), lambda: red(n=-1), lambda: red(dtype=torch.float16), lambda: red(t=table.cpu())):
        with pytest.raises(ValueError):
            f()
    grad = rows.clone().requires_grad_()
    for f in (lambda: app(k=grad), lambda: rop(v=grad), lambda: att(q=q.clone().requires_grad_()), lambda: rop(c=cos.clone().requires_grad_())):
        with pytest.raises(ValueError, match="inference"):
            f()
    with torch.no_grad():
        app(k=grad)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(rows, rows)
        with pytest.raises(ValueError, match="tangents"):
            app(k=dual)
    with pytest.raises(ValueError):
        bf.empty_q4_pages(4, 2, 16, 64, group=16)
    with pytest.raises(NotImplementedError):
        bf.empty_q4_pages(4, 2, 16, 96)
