"""GPU: the paged operators against plain implementations in 64 bits.

Tolerances are bounds on the arithmetic, computed from the inputs: u = 2^-24 is half a step of fp32,
and an output of n bits of mantissa may be off by half a step of its own (bf16 2^-8)."""
from __future__ import annotations

import math
import random

import pytest
import torch

import butterfly_amd as bf

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}
NAN = float("nan")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------- attention
def _paged_case(lens, hq, hkv, d, page, dtype, *, seed=0, layout="plain", spread=1.0, stale=NAN, width=None):
    """Pages in random order with stale values in every row that holds no token; returns the call's tensors
    and the dense keys and values of each request."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g).tolist()
    width = width or max(1, max(need)) + 1
    table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)    # entries behind the last page: garbage
    if layout == "one":                      # keys and values in one tensor, token-major pages
        store = torch.full((total, 2, page, hkv, d), stale, dtype=dtype)
        kp, vp = store[:, 0].transpose(1, 2), store[:, 1].transpose(1, 2)
    else:
        kp = torch.full((total, hkv, page, d), stale, dtype=dtype)
        vp = kp.clone()
        store = None
    dense, at = [], 0
    for b, n in enumerate(lens):
        k = (torch.randn(hkv, n, d, generator=g) * spread).to(dtype)
        v = torch.randn(hkv, n, d, generator=g).to(dtype)
        dense.append((k, v))
        for j in range(need[b]):
            p, rows = order[at], slice(j * page, min(n, (j + 1) * page))
            table[b, j] = p
            kp[p, :, :rows.stop - rows.start] = k[:, rows]
            vp[p, :, :rows.stop - rows.start] = v[:, rows]
            at += 1
    q = torch.randn(len(lens), hq, 1, d, generator=g).to(dtype)
    if store is not None:
        store = store.cuda()
        kp, vp = store[:, 0].transpose(1, 2), store[:, 1].transpose(1, 2)
    return q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), _i32(lens), dense


def _attention64(q, dense, window, scale):
    """o, l, m in 64 bits and the error bounds of each."""
    b, hq, _, d = q.shape
    q = q[:, :, 0].double().cpu()
    o, bo = torch.zeros(b, hq, d, dtype=torch.float64), torch.zeros(b, hq, d, dtype=torch.float64)
    l, m = torch.zeros(b, hq, dtype=torch.float64), torch.full((b, hq), -1e30, dtype=torch.float64)
    bl, bm = torch.zeros_like(l), torch.zeros_like(m)
    for i, (k, v) in enumerate(dense):
        n = k.shape[1]
        lo = max(0, n - window) if window else 0
        if n == lo:
            continue
        g = hq // k.shape[0]
        k = k[:, lo:].double().repeat_interleave(g, 0)
        v = v[:, lo:].double().repeat_interleave(g, 0)
        s = (k @ q[i][:, :, None])[..., 0] * scale
        m[i] = s.amax(-1)
        p = (s - m[i][:, None]).exp()
        l[i] = p.sum(-1)
        w = p / l[i][:, None]
        o[i] = (w[:, None] @ v)[:, 0]
        # a score: d products and sums, the scale (each within u of its partial sums); a weight: the scores'
        # errors and a few u of exp's argument and value; a sum over n keys: n u in any order
        ds = ((k.abs() @ q[i][:, :, None].abs())[..., 0] * abs(scale) * (d + 4) * U).amax(-1)
        dw = torch.expm1(2 * ds) + 16 * U
        # two bf16 parts of a weight (16 bits of it) enter the bf16 product
        split = 2.0 ** -16 if q.dtype == torch.float64 else 0.0
        bo[i] = (w[:, None] @ v.abs())[:, 0] * (2 * dw + 2 * (n + 16) * U + split)[:, None]
        bl[i], bm[i] = l[i] * (dw + (n + 16) * U), ds + 2 * U * m[i].abs()
    return (o, l, m), (bo, bl, bm)


def _check_attention(q, kp, vp, table, lens, dense, *, window=0, scale=None):
    scale_ = scale if scale is not None else q.shape[-1] ** -0.5
    o, l, m = bf.paged_attention(q, kp, vp, table, lens, window=window, scale=scale, return_stats=True)
    alone = bf.paged_attention(q, kp, vp, table, lens, window=window, scale=scale)
    assert torch.equal(alone, o)
    assert o.shape == q.shape and o.dtype == q.dtype and l.shape == m.shape == (*q.shape[:2], 1, 1)
    (eo, el, em), (bo, bl, bm) = _attention64(q, dense, window, scale_)
    h = HALF_STEP[q.dtype]
    do = (o[:, :, 0].double().cpu() - eo).abs()
    assert bool((do <= bo + h * (eo.abs() + bo)).all()), (do - bo - h * eo.abs()).max()
    dl, dm = (l[:, :, 0, 0].double().cpu() - el).abs(), (m[:, :, 0, 0].double().cpu() - em).abs()
    assert bool((dl <= bl).all()), (dl - bl).max()
    assert bool((dm <= bm + 1e30 * U * (em == -1e30)).all()), (dm - bm).max()


HEADS = [(1, 1), (8, 2), (16, 4), (5, 1), (24, 1), (40, 2), (7, 7)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_attention_heads(dtype, d, hq, hkv):
    _check_attention(*_paged_case([1, 0, 37, 130, 515], hq, hkv, d, 32, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("layout", ["plain", "one"])
def test_attention_pages_and_layouts(dtype, page, layout):
    lens = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700, 1023, 1024, 1025]
    _check_attention(*_paged_case(lens, 8, 2, 128, page, dtype, layout=layout))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 100, 333, 5000])
def test_attention_windows(dtype, window):
    _check_attention(*_paged_case([0, 1, 2, 64, 65, 99, 100, 101, 333, 1200], 8, 2, 64, 16, dtype), window=window)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (BF, 128), (BF, 256), (F32, 64), (F32, 128), (F32, 256)])
@pytest.mark.parametrize("lens", [[20011], [1, 9000, 0, 3], [4097] * 5, [0, 0, 0]])
def test_attention_long_and_ragged(dtype, d, lens):
    _check_attention(*_paged_case(lens, 4, 2, d, 64, dtype, seed=len(lens)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_many_requests(dtype):
    r = random.Random(5)
    lens = [r.choice([0, 1, 5, 40, 64, 200]) for _ in range(700)]
    lens[411] = 6000
    _check_attention(*_paged_case(lens, 2, 1, 64, 16, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [0.01, 1.0, -0.3])
def test_attention_scale_and_peaked_scores(dtype, scale):
    _check_attention(*_paged_case([400, 1030], 8, 2, 128, 64, dtype, spread=4.0), scale=scale)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_strided_q(dtype):
    q, kp, vp, table, lens, dense = _paged_case([50, 300], 8, 2, 128, 32, dtype)
    wide = torch.zeros(2, 12, 128, dtype=dtype, device="cuda")
    wide[:, 2:10] = q[:, :, 0]
    view = wide[:, 2:10].unsqueeze(2)
    want = bf.paged_attention(q, kp, vp, table, lens)
    assert torch.equal(bf.paged_attention(view, kp, vp, table, lens), want)
    odd = torch.zeros(2, 8, 1, 129, dtype=dtype, device="cuda")[..., 1:]      # rows that are not 16-byte aligned
    odd.copy_(q)
    assert torch.equal(bf.paged_attention(odd, kp, vp, table, lens), want)
    assert torch.equal(bf.paged_attention(q, kp, vp, table[:, :], lens.repeat_interleave(2)[::2]), want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [40, 3000])
def test_attention_infinities_and_nan_in_seen_rows(dtype, n):
    """What one softmax over the seen keys gives: rows of other kv heads and requests are untouched."""
    q, kp, vp, table, lens, dense = _paged_case([n, n], 4, 2, 64, 32, dtype)
    want = bf.paged_attention(q, kp, vp, table, lens)
    page = int(table[0, (n // 2) // 32])
    vp[page, 0, n // 2 % 32, 5] = float("inf")
    o = bf.paged_attention(q, kp, vp, table, lens)
    assert bool((o[0, :2, 0, 5] == float("inf")).all())
    keep = torch.ones(64, dtype=torch.bool)
    keep[5] = False
    assert torch.equal(o[0, :2, 0][:, keep], want[0, :2, 0][:, keep])
    assert torch.equal(o[0, 2:], want[0, 2:]) and torch.equal(o[1], want[1])
    kp[page, 0, n // 2 % 32] = NAN
    o = bf.paged_attention(q, kp, vp, table, lens)
    assert bool(torch.isnan(o[0, :2]).all())
    assert torch.equal(o[0, 2:], want[0, 2:]) and torch.equal(o[1], want[1])
    # a key of -inf scores: weight 0 where q is positive there
    kp[page, 0, n // 2 % 32] = 0.0
    vp[page, 0, n // 2 % 32] = 0.0
    q[0, :2, 0, 3] = 1.0
    kp[page, 0, n // 2 % 32, 3] = -float("inf")
    o, l, m = bf.paged_attention(q, kp, vp, table, lens, return_stats=True)
    assert bool(torch.isfinite(o[0, :2]).all()) and bool(torch.isfinite(l).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_all_scores_minus_infinity_is_nan_and_empty_is_zero(dtype):
    q, kp, vp, table, lens, _ = _paged_case([40, 0, 2000], 2, 1, 64, 32, dtype)
    q.fill_(1.0)
    k2 = torch.where(torch.isnan(kp), kp, torch.full_like(kp, -float("inf")))
    o, l, m = bf.paged_attention(q, k2, vp, table, lens, return_stats=True)
    assert bool(torch.isnan(o[0]).all()) and bool(torch.isnan(o[2]).all())
    assert bool((o[1] == 0).all()) and bool((l[1] == 0).all()) and bool((m[1] == -1e30).all())
    assert bool(torch.isnan(l[[0, 2]]).all()) and bool((m[[0, 2]] == -float("inf")).all())
    # NaN scores: the maximum is NaN too, whether some keys or all of them have one
    for keys in (slice(0, 1), slice(None)):
        k3 = kp.clone()
        k3[table[0, :1].long(), :, keys] = NAN
        if keys == slice(None):
            k3[table[0, 1].long()] = NAN
        o, l, m = bf.paged_attention(q, k3, vp, table, lens, return_stats=True)
        assert all(bool(torch.isnan(x[0]).all()) for x in (o, l, m)) and bool(torch.isfinite(m[2]).all())


def test_attention_bad_tables_give_nan_for_their_request_only():
    for n in (100, 5000):
        q, kp, vp, table, lens, _ = _paged_case([n, n, n], 4, 2, 64, 32, BF)
        want = bf.paged_attention(q, kp, vp, table, lens)
        bad = table.clone()
        bad[0, (n - 1) // 32] = kp.shape[0]
        bad[1, 0] = -1
        o, l, m = bf.paged_attention(q, kp, vp, bad, lens, return_stats=True)
        for x in (o, l, m):
            assert bool(torch.isnan(x[:2]).all())
        assert torch.equal(o[2], want[2])
        # with a window that does not read the bad entry, the request is whole
        o = bf.paged_attention(q, kp, vp, bad, lens, window=20)
        assert bool(torch.isfinite(o[1]).all()) and bool(torch.isnan(o[0]).all())
        cap = table.shape[1] * 32
        long = _i32([cap + 1, -5, 2 ** 31 - 1])
        o, l, m = bf.paged_attention(q, kp, vp, torch.zeros_like(table), long, return_stats=True)
        assert bool(torch.isnan(o[0]).all()) and bool(torch.isnan(o[2]).all())
        assert bool((o[1] == 0).all()) and bool((m[1] == -1e30).all())


def test_attention_stats_merge_with_another_stream():
    """Two halves of a context, one paged, merge to the whole (online_softmax_merge takes the stream)."""
    q, kp, vp, table, lens, dense = _paged_case([512, 512], 8, 2, 64, 64, F32)
    whole = bf.paged_attention(q, kp, vp, table, lens)
    a = bf.paged_attention(q, kp, vp, table, _i32([256, 0]), return_stats=True)
    b = bf.paged_attention(q, kp, vp, table, lens, window=256, return_stats=True)
    merged = bf.online_softmax_merge(a, b)
    (e, _, _), (bo, _, _) = _attention64(q, dense, 0, 64 ** -0.5)
    assert bool(((merged[0, :, 0].double().cpu() - e[0]).abs() <= 4 * bo[0] + 8 * U * e[0].abs()).all())
    # beside an empty stream the merge is (l o) / l: one rounding of the product, one of the quotient, u each
    assert bool(((merged[1] - b[0][1]).abs() <= 2.5 * U * b[0][1].abs()).all()) and whole.shape == merged.shape


def test_attention_on_another_stream_and_two_at_once():
    q, kp, vp, table, lens, _ = _paged_case([9000, 7000], 8, 2, 128, 64, BF)
    q2 = q.flip(0).contiguous()
    want = [bf.paged_attention(x, kp, vp, table, lens) for x in (q, q2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for x, s in zip((q, q2), streams):
            with torch.cuda.stream(s):
                got.append(bf.paged_attention(x, kp, vp, table, lens))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_offsets_beyond_32_bits():
    """Pages past 2^32 bytes of their tensor, with one row of a request in each."""
    page, hkv, d = 1024, 1, 256
    per = page * d * 2
    pages = (1 << 32) // per + 40
    kp = torch.empty(pages, hkv, page, d, dtype=BF, device="cuda")
    vp = torch.empty_like(kp)
    g = torch.Generator().manual_seed(1)
    lens = [page * 2 + 7]
    ids = [pages - 1, 3, pages - 20]
    k = torch.randn(hkv, lens[0], d, generator=g).to(BF)
    v = torch.randn(hkv, lens[0], d, generator=g).to(BF)
    slots = torch.tensor([ids[t // page] * page + t % page for t in range(lens[0])], device="cuda")
    bf.paged_append(k.cuda().transpose(0, 1), v.cuda().transpose(0, 1), kp, vp, slots)
    q = torch.randn(1, 4, 1, d, generator=g).to(BF).cuda()
    _check_attention(q, kp, vp, _i32([ids]), _i32(lens), [(k, v)])


def test_attention_refusals():
    q, kp, vp, table, lens, _ = _paged_case([10, 20], 4, 2, 64, 16, BF)
    bad = [
        dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[:, :, 0]), dict(q=q[:, :0]), dict(kp=kp[:, :, :12]), dict(kp=kp[:2]),
        dict(kp=kp.transpose(2, 3), vp=vp.transpose(2, 3)), dict(table=table.long()), dict(table=table[:1]),
        dict(table=table.t().contiguous().t()), dict(lens=lens.long()), dict(lens=lens[:1]), dict(q=q.half(), kp=kp.half(), vp=vp.half()),
        dict(q=q.cpu()), dict(kp=kp[:0], vp=vp[:0]),
    ]
    for kw in bad:
        a = dict(q=q, kp=kp, vp=vp, table=table, lens=lens)
        a.update(kw)
        with pytest.raises(ValueError):
            bf.paged_attention(*a.values())
    with pytest.raises(ValueError):
        bf.paged_attention(q, kp, vp, table, lens, window=-1)
    with pytest.raises(TypeError):
        bf.paged_attention(q, kp, vp, table, lens, window=3.5)
    with pytest.raises(ValueError, match="inference"):
        bf.paged_attention(q.clone().requires_grad_(), kp, vp, table, lens)
    wide = torch.zeros(3, 2, 16, 96, dtype=BF, device="cuda")
    with pytest.raises(NotImplementedError):
        bf.paged_attention(torch.zeros(2, 4, 1, 96, dtype=BF, device="cuda"), wide, wide, table, lens)
    assert bf.paged_attention(q[:0], kp, vp, table[:0], lens[:0]).shape == (0, 4, 1, 64)
    none = bf.paged_attention(q, kp, vp, table[:, :0], torch.zeros_like(lens))
    assert bool((none == 0).all())


# --------------------------------------------------------------------------- rows into pages
def _pool(pages, hkv, page, d, dtype, layout="plain"):
    g = torch.Generator(device="cuda").manual_seed(9)
    if layout == "one":
        x = torch.randn(pages, 2, page, hkv, d, generator=g, device="cuda").to(dtype)
        return x[:, 0].transpose(1, 2), x[:, 1].transpose(1, 2)
    return tuple(torch.randn(pages, hkv, page, d, generator=g, device="cuda").to(dtype) for _ in range(2))


def _put(pages, rows, slots):
    out = pages.clone()
    page = pages.shape[2]
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pages.shape[0] * page:
            out[s // page, :, s % page] = rows[i]
    return out


@pytest.mark.parametrize("dtype,d", [(BF, 8), (BF, 72), (BF, 128), (BF, 256), (F32, 4), (F32, 64), (F32, 100)])
@pytest.mark.parametrize("n,hkv,page,layout", [(1, 1, 16, "plain"), (7, 3, 32, "one"), (100, 2, 1024, "plain"), (0, 2, 16, "plain")])
def test_append_is_a_copy(dtype, d, n, hkv, page, layout):
    kp, vp = _pool(5, hkv, page, d, dtype, layout)
    g = torch.Generator(device="cuda").manual_seed(n)
    fused = torch.randn(n, 2 * hkv + 1, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(hkv, n, d, generator=g, device="cuda").to(dtype).transpose(0, 1)
    v = fused[:, 1:1 + hkv]
    slots = torch.randperm(5 * page, generator=g, device="cuda")[:n]
    if n > 5:
        slots[2], slots[3], slots[4] = -1, 5 * page, -2 ** 40
    wk, wv = _put(kp, k, slots), _put(vp, v, slots)
    bf.paged_append(k, v, kp, vp, slots)
    assert torch.equal(kp, wk) and torch.equal(vp, wv)


def test_append_rows_that_are_not_aligned_and_refusals():
    kp, vp = _pool(4, 2, 16, 64, BF)
    rows = torch.randn(6, 2, 65, device="cuda").to(BF)[..., 1:]
    slots = torch.tensor([3, 60, 17, 5, 40, 41], device="cuda")
    wk = _put(kp, rows, slots)
    bf.paged_append(rows, rows, kp, vp, slots)
    assert torch.equal(kp, wk)
    for a in [(rows.float(), rows.float(), kp, vp, slots), (rows[:, :1], rows[:, :1], kp, vp, slots), (rows, rows, kp, vp, slots.int()),
              (rows, rows, kp, vp, slots[:5]), (rows, rows[:5], kp, vp, slots), (rows, rows, kp, vp[:3], slots),
              (rows, rows, kp[..., 1:], vp[..., 1:], slots), (rows, rows, kp[:1].expand(4, 2, 16, 64), vp, slots),
              (rows.cpu(), rows, kp, vp, slots), (rows, rows, kp, kp, slots), (rows[..., :60], rows[..., :60], kp[..., :60], vp[..., :60], slots)]:
        with pytest.raises(ValueError):
            bf.paged_append(*a)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rot", [16, 32, 48, 0])
@pytest.mark.parametrize("norm", [True, False])
def test_rope_append(dtype, d, rot, norm):
    rot = rot or d
    n, hq, hkv, page = 37, 6, 2, 32
    g = torch.Generator(device="cuda").manual_seed(d + rot)
    kp, vp = _pool(4, hkv, page, d, dtype, "one" if norm else "plain")
    x = (torch.randn(n, hq + 2 * hkv, d, generator=g, device="cuda") * 3).to(dtype)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    inv = 1.0 / (1e4 ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))
    ang = torch.arange(3000, device="cuda")[:, None] * torch.cat([inv, inv])[None]
    cos, sin = ang.cos().float(), ang.sin().float()
    pos = torch.randint(3000, (n,), generator=g, device="cuda")
    slots = torch.randperm(4 * page, generator=g, device="cuda")[:n]
    slots[7] = -1
    w = [(torch.rand(d, generator=g, device="cuda") + 0.5).to(dtype) for _ in range(2)] if norm else [None, None]
    wv = _put(vp, v, slots)
    wk0 = kp.clone()
    out = bf.paged_rope_append(q, k, v, kp, vp, slots, pos, cos, sin, q_weight=w[0], k_weight=w[1], eps=1e-5)

    def exact(y, w):
        y = y.double()
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
        r = y[..., :rot]
        turned = torch.cat([-r[..., rot // 2:], r[..., :rot // 2]], -1)
        z = torch.cat([r * c + turned * s, y[..., rot:]], -1)
        # y: d/2 u of the mean square's sum, a few u of rsqrt and the products; z: three more roundings
        size = torch.cat([(r * c).abs() + (turned * s).abs(), y[..., rot:].abs()], -1)
        bound = size * (d / 2 + 16) * U
        return z, bound + HALF_STEP[dtype] * (z.abs() + bound)

    z, bound = exact(q, w[0])
    assert bool(((out.double() - z).abs() <= bound).all())
    assert torch.equal(vp, wv)
    z, bound = exact(k, w[1])
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            assert bool(((kp[s // page, :, s % page].double() - z[i]).abs() <= bound[i]).all())
            wk0[s // page, :, s % page] = kp[s // page, :, s % page]
    assert torch.equal(kp, wk0)                       # nothing else was written


def test_rope_append_positions_outside_the_table():
    kp, vp = _pool(2, 1, 16, 64, BF)
    q = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    k = v = torch.ones(3, 1, 64, dtype=BF, device="cuda")
    cos, sin = torch.ones(4, 64, device="cuda"), torch.zeros(4, 64, device="cuda")
    pos = torch.tensor([4, -1, 3], device="cuda")
    slots = torch.tensor([1, 2, 3], device="cuda")
    out = bf.paged_rope_append(q, k, v, kp, vp, slots, pos, cos, sin)
    assert bool(torch.isnan(out[:2]).all()) and torch.equal(out[2], q[2])
    assert bool(torch.isnan(kp[0, 0, 1:3]).all()) and torch.equal(kp[0, :, 3], k[2]) and torch.equal(vp[0, 0, 1:4], v[:, 0])


def test_rope_append_refusals():
    kp, vp = _pool(2, 1, 16, 64, BF)
    q = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    k = torch.ones(3, 1, 64, dtype=BF, device="cuda")
    tab = torch.ones(4, 64, device="cuda")
    i = torch.arange(3, device="cuda")
    w = torch.ones(64, dtype=BF, device="cuda")
    ok = dict(q=q, k=k, v=k, kp=kp, vp=vp, slots=i, pos=i, cos=tab, sin=tab)
    for kw in [dict(q=q[:2]), dict(q=q.float()), dict(pos=i.int()), dict(pos=i[:2]), dict(cos=tab.double(), sin=tab.double()),
               dict(cos=tab[:, :24], sin=tab[:, :24]), dict(cos=tab[:0], sin=tab[:0]), dict(sin=tab[:3]), dict(q_weight=w),
               dict(q_weight=w.float(), k_weight=w.float()), dict(q_weight=w[:32], k_weight=w[:32])]:
        a = {**ok, **kw}
        extra = {x: a.pop(x) for x in ("q_weight", "k_weight") if x in a}
        with pytest.raises(ValueError):
            bf.paged_rope_append(*a.values(), **extra)
    with pytest.raises(ValueError, match="inference"):
        bf.paged_rope_append(*{**ok, "q": q.clone().requires_grad_()}.values())
    p = torch.zeros(2, 1, 16, 80, dtype=BF, device="cuda")
    z = torch.ones(3, 1, 80, dtype=BF, device="cuda")
    with pytest.raises(NotImplementedError):
        bf.paged_rope_append(z, z, z, p, p.clone(), i, i, tab, tab)


# --------------------------------------------------------------------------- bookkeeping
def _plan_ref(table, lens, counts, free, state, page, rows):
    """The contract on Python lists; updates table and free."""
    top, err = state
    width = len(table[0]) if table else 0
    new = [max(0, a + c) for a, c in zip(lens, counts)]
    up = lambda x: -(-x // page)
    if not err:
        give = sum(max(0, up(a) - up(b)) for a, b in zip(lens, new) if 0 <= a <= width * page)
        take = sum(max(0, up(b) - up(a)) for a, b in zip(lens, new))
        if any(a < 0 or a > width * page for a in lens):
            err = 1
        elif any(b > width * page for b in new):
            err = 2
        elif sum(max(0, c) for c in counts) > rows:
            err = 3
        elif top + give < take:
            err = 4
        elif not 0 <= top <= len(free) or top + give > len(free):
            err = 5
    if err:
        return lens, [top, err], [0] * (len(lens) + 1), [-1] * rows, [0] * rows
    stack = free[:top] + [table[b][j] for b, (a, n) in enumerate(zip(lens, new)) for j in range(up(n), up(a))][::-1]
    free[:len(stack)] = stack
    slots, pos, starts = [], [], [0]
    for b, (a, n) in enumerate(zip(lens, new)):
        for j in range(up(a), up(n)):
            table[b][j] = stack.pop()
        for p in range(a, n):
            slots.append(table[b][p // page] * page + p % page)
            pos.append(p)
        starts.append(len(slots))
    pad = rows - len(slots)
    return new, [len(stack), 0], starts, slots + [-1] * pad, pos + [0] * pad


def _check_plan(table, lens, counts, free, state, page, rows, in_place=False):
    t, f = _i32(table).view(len(table), -1), _i32(free)
    p = bf.paged_plan(t, _i32(lens), _i32(counts), f, _i32(state), page_size=page, num_rows=rows, in_place=in_place)
    want = _plan_ref(table, lens, counts, free, state, page, rows)
    got = [x.tolist() for x in (p.lengths, p.state, p.starts, p.slots, p.positions)]
    for g, w in zip(got, want):
        assert g == list(w)
    assert t.tolist() == table and f.tolist() == free
    return want


@pytest.mark.parametrize("b,page,biggest", [(1, 16, 40), (3, 32, 100), (64, 16, 60), (65, 64, 30), (300, 16, 20), (1500, 16, 40)])
def test_plan_random_steps(b, page, biggest):
    r = random.Random(b)
    width = 12
    pages = b * 8
    table, free, state = [[-1] * width for _ in range(b)], r.sample(range(pages), pages), [pages, 0]
    lens = [0] * b
    for step in range(6):
        counts = [r.choice([0, 1, 1, 1, r.randint(1, biggest), -r.randint(1, 2 * biggest), -n]) for n in lens]
        counts = [min(c, width * page - n) for c, n in zip(counts, lens)]
        rows = sum(max(0, c) for c in counts) + r.choice([0, 0, 1, 300])
        lens, state, *_ = _check_plan(table, lens, counts, free, state, page, rows, in_place=step % 2 == 0)
        if state[1]:
            assert state[1] == 4
            state = [state[0], 0]


@pytest.mark.parametrize("b,rows", [(5000, 6000), (9000, 100), (3, 20000), (4096, 4096), (4097, 4096), (20, 4097)])
def test_plan_many_requests_and_rows(b, rows):
    r = random.Random(rows)
    page = 16
    lens = [r.randint(0, 40) for _ in range(b)]
    width = max(8, -(-(40 + rows) // page)) if b < 100 else 8
    used = [-(-n // page) for n in lens]
    ids = list(range(sum(used) + (rows // page) + 2 * b + 5))
    r.shuffle(ids)
    table, at = [], 0
    for u in used:
        table.append(ids[at:at + u] + [-1] * (width - u))
        at += u
    free, state = ids[at:] + [-1] * at, [len(ids) - at, 0]
    counts, left = [], rows
    for n in lens:
        c = r.choice([0, 1, 2, -3, -n]) if b > 100 else rows // b
        c = min(c, left)
        left -= max(0, c)
        counts.append(c)
    _check_plan(table, lens, counts, free, state, page, rows)


def test_plan_taken_back_leaves_the_free_list_as_it_was():
    page, b, width = 32, 9, 10
    t = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(64, device="cuda").int()
    state, lens = _i32([64, 0]), torch.zeros(b, dtype=torch.int32, device="cuda")
    grow = _i32([5, 0, 33, 64, 1, 320, 31, 32, 100])
    bf.paged_plan(t, lens, grow, free, state, page_size=page, num_rows=600, in_place=True)
    before, f0, s0 = lens.clone(), free.clone(), state.clone()
    more = _i32([40, 7, 0, 1, 32, 0, 1, 1, 29])
    first = bf.paged_plan(t, lens, more, free, state, page_size=page, num_rows=600)
    again = bf.paged_plan(t, lens, more, free, state, page_size=page, num_rows=600)
    assert all(torch.equal(getattr(first, x), getattr(again, x)) for x in ("lengths", "state", "starts", "slots", "positions"))
    back = bf.paged_plan(t, first.lengths, -more, free, first.state, page_size=page, num_rows=0)
    assert torch.equal(back.lengths, before) and torch.equal(back.state, s0) and torch.equal(free, f0)


@pytest.mark.parametrize("rows", [50, 5000])
def test_plan_errors_change_nothing_and_stay(rows):
    page, width = 16, 4
    base = dict(table=[[7, -1, -1, -1], [3, 9, -1, -1]], lens=[10, 20], counts=[1, 1], free=[4, 5, 6, -1, -1, -1, -1, -1],
                state=[3, 0])
    cases = [(1, dict(lens=[-1, 20])), (1, dict(lens=[65, 20])), (1, dict(lens=[2 ** 31 - 1, 20], counts=[2 ** 31 - 1, 0])),
             (2, dict(counts=[55, 0])), (2, dict(counts=[2 ** 31 - 1, 2 ** 31 - 1])), (3, dict(counts=[40, 44], rows=50)),
             (4, dict(counts=[23, 13], state=[2, 0])), (5, dict(state=[9, 0])), (4, dict(state=[-1, 0])), (5, dict(state=[8, 0], counts=[-10, 0])),
             (77, dict(state=[3, 77])), (1, dict(lens=[-2 ** 31, 20], counts=[-2 ** 31, 0]))]
    for code, kw in cases:
        c = dict(base, rows=rows)
        c.update(kw)
        table, free = [list(x) for x in c["table"]], list(c["free"])
        want = _check_plan(table, c["lens"], c["counts"], free, c["state"], page, c["rows"])
        assert want[1][1] == code, (kw, want)
        assert table == base["table"] and free == base["free"]
    # 66 rows: too many for 50; with room for them the step takes exactly the three pages there are
    want = _check_plan([list(x) for x in base["table"]], base["lens"], [38, 28], list(base["free"]), base["state"], page, rows)
    assert want[1] == ([3, 3] if rows == 50 else [0, 0])
    # the lowest and highest counts that fit
    c = dict(base)
    _check_plan([list(x) for x in c["table"]], c["lens"], [-2 ** 31, 28], list(c["free"]), c["state"], page, rows)


def test_plan_strided_table_and_refusals():
    page = 16
    wide = torch.full((3, 9), -7, dtype=torch.int32, device="cuda")
    t = wide[:, 2:6]
    free, state, lens = torch.arange(12, device="cuda").int(), _i32([12, 0]), torch.zeros(3, dtype=torch.int32, device="cuda")
    p = bf.paged_plan(t, lens, _i32([20, 0, 64]), free, state, page_size=page, num_rows=90)
    assert t.tolist() == [[11, 10, -7, -7], [-7] * 4, [9, 8, 7, 6]]
    assert bool((wide[:, :2] == -7).all()) and bool((wide[:, 6:] == -7).all()) and p.state.tolist() == [6, 0]
    ok = dict(t=t, l=lens, c=lens, f=free, s=state)
    for kw in [dict(t=t.long()), dict(t=wide.t()[:4].t()), dict(t=t[:2]), dict(l=lens.long()), dict(c=lens[:2]), dict(s=state[:1]),
               dict(f=free.long()), dict(f=free[::2]), dict(t=t[:1].expand(3, 4)), dict(c=lens.cpu()), dict(l=lens[None])]:
        if "t" in kw and kw["t"].dtype == torch.int32 and kw["t"].shape == t.shape and kw["t"].stride(1) == 1 and kw["t"].stride(0) > 0:
            continue
        with pytest.raises(ValueError):
            bf.paged_plan(*{**ok, **kw}.values(), page_size=page, num_rows=3)
    for kw in [dict(page_size=24, num_rows=3), dict(page_size=16, num_rows=-1)]:
        with pytest.raises(ValueError):
            bf.paged_plan(*ok.values(), **kw)
    none = bf.paged_plan(t[:0], lens[:0], lens[:0], free, state, page_size=page, num_rows=3)
    assert none.slots.tolist() == [-1] * 3 and none.starts.tolist() == [0] and none.state.tolist() == [12, 0]


# --------------------------------------------------------------------------- together, and captured
def _step(s, i):
    """One decode step of one layer for all requests: plan, projection tail into pages, attention."""
    plan = bf.paged_plan(s["table"], s["lens"], s["counts"], s["free"], s["state"], page_size=s["page"], num_rows=s["rows"],
                         in_place=True)
    q = bf.paged_rope_append(s["q"], s["k"], s["v"], s["kp"], s["vp"], plan.slots, plan.positions, s["cos"], s["sin"],
                             q_weight=s["w"], k_weight=s["w"])
    o = bf.paged_attention(q.unsqueeze(2), s["kp"], s["vp"], s["table"], plan.lengths)
    s["out"].index_copy_(0, s["i"], o[None])
    s["i"].add_(1)


def _state(b, steps, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, d, page, pages = 8, 2, 64, 16, 200
    ang = torch.arange(400, device="cuda")[:, None] * torch.rand(d // 2, generator=g, device="cuda").repeat(2)[None]
    x = torch.randn(b, hq + 2 * hkv, d, generator=g, device="cuda").to(BF)
    s = dict(table=torch.full((b, 20), -1, dtype=torch.int32, device="cuda"), lens=torch.zeros(b, dtype=torch.int32, device="cuda"),
             counts=torch.ones(b, dtype=torch.int32, device="cuda"), free=torch.randperm(pages, generator=g, device="cuda").int(),
             state=_i32([pages, 0]), page=page, rows=b, q=x[:, :hq], k=x[:, hq:hq + hkv], v=x[:, hq + hkv:],
             kp=torch.full((pages, hkv, page, d), NAN, dtype=BF, device="cuda"),
             vp=torch.full((pages, hkv, page, d), NAN, dtype=BF, device="cuda"), cos=ang.cos(), sin=ang.sin(),
             w=torch.ones(d, dtype=BF, device="cuda"), out=torch.zeros(steps, b, hq, 1, d, dtype=BF, device="cuda"),
             i=torch.zeros(1, dtype=torch.long, device="cuda"))
    # a ragged start: request b holds 5 b tokens
    start = _i32([5 * i for i in range(b)])
    rows = int(start.sum())
    p = bf.paged_plan(s["table"], s["lens"], start, s["free"], s["state"], page_size=page, num_rows=rows, in_place=True)
    k = torch.randn(rows, hkv, d, generator=g, device="cuda").to(BF)
    bf.paged_append(k, k.flip(0), s["kp"], s["vp"], p.slots)
    return s


def test_a_captured_step_replays_as_the_eager_ones():
    b, steps = 6, 40
    eager, graph = _state(b, steps, 3), _state(b, steps, 3)
    for i in range(steps):
        _step(eager, i)
    _step(graph, 0)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        _step(graph, 1)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(1, steps):
        g.replay()
        if i % 7 == 0:
            torch.cuda.synchronize()
            torch.randn(1 << 20, device="cuda").sum()          # the program's own work between replays
    torch.cuda.synchronize()
    assert torch.equal(eager["out"], graph["out"]) and bool(torch.isfinite(eager["out"]).all())
    for x in ("lens", "state", "table", "free"):
        assert torch.equal(eager[x], graph[x])
    assert eager["lens"].tolist() == [5 * i + steps for i in range(b)]


def test_a_chain_against_dense_attention():
    """Ragged requests that grow, leave and are replaced: every step's output against dense softmax
    attention in 64 bits over the keys and values that the pages were given."""
    b, d, hq, hkv, page = 5, 64, 4, 2, 16
    g = torch.Generator().manual_seed(11)
    pages = 60
    table = torch.full((b, 16), -1, dtype=torch.int32, device="cuda")
    free, state = torch.arange(pages, dtype=torch.int32, device="cuda"), _i32([pages, 0])
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    kp = torch.full((pages, hkv, page, d), NAN, dtype=BF, device="cuda")
    vp = kp.clone()
    held = [(torch.zeros(hkv, 0, d, dtype=BF), torch.zeros(hkv, 0, d, dtype=BF)) for _ in range(b)]
    r = random.Random(2)
    for step in range(12):
        counts = [r.choice([1, 1, 1, 0, 40, -3, -10 ** 6]) for _ in range(b)]
        rows = sum(max(0, c) for c in counts) + 3
        plan = bf.paged_plan(table, lens, _i32(counts), free, state, page_size=page, num_rows=rows, in_place=True)
        k = torch.randn(rows, hkv, d, generator=g).to(BF)
        v = torch.randn(rows, hkv, d, generator=g).to(BF)
        bf.paged_append(k.cuda(), v.cuda(), kp, vp, plan.slots)
        at = 0
        for i, c in enumerate(counts):
            hk, hv = held[i]
            if c < 0:
                n = max(0, hk.shape[1] + c)
                held[i] = hk[:, :n], hv[:, :n]
            else:
                held[i] = torch.cat([hk, k[at:at + c].transpose(0, 1)], 1), torch.cat([hv, v[at:at + c].transpose(0, 1)], 1)
                at += c
        assert lens.tolist() == [x.shape[1] for x, _ in held] and int(state[1]) == 0
        q = torch.randn(b, hq, 1, d, generator=g).to(BF).cuda()
        _check_attention(q, kp, vp, table, lens, held)


@pytest.mark.parametrize("b,each", [(5, 1), (5, 3), (700, 8), (3000, 2), (1, 5000)])
def test_plan_with_rows_of_its_own_for_every_request(b, each):
    """rows_each: row b * each + i is request b's, idle rows have slot -1; lengths, pages and positions are the
    packed call's."""
    r = random.Random(b)
    page, width = 16, max(8, each // 16 + 6)
    lens = [r.randint(0, 60) for _ in range(b)]
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need) + b * (each // page + 2)))
    r.shuffle(ids)
    table, at = [], 0
    for u in need:
        table.append(ids[at:at + u] + [-1] * (width - u))
        at += u
    free = _i32(ids[at:] + [-1] * at)
    counts = [r.choice([0, 1, each, r.randint(0, each), -r.randint(0, 70)]) for _ in range(b)]
    t, state = _i32(table), _i32([len(ids) - at, 0])
    t2, free2 = t.clone(), free.clone()
    rows = sum(max(0, c) for c in counts)
    packed = bf.paged_plan(t, _i32(lens), _i32(counts), free, state, page_size=page, num_rows=rows)
    fixed = bf.paged_plan(t2, _i32(lens), _i32(counts), free2, state, page_size=page, num_rows=b * each, rows_each=each)
    assert torch.equal(t, t2) and torch.equal(free, free2)
    assert torch.equal(packed.lengths, fixed.lengths) and torch.equal(packed.state, fixed.state) and int(fixed.state[1]) == 0
    assert fixed.starts.tolist() == [each * i for i in range(b + 1)]
    slots, pos = [-1] * (b * each), [0] * (b * each)
    for i, (s, c) in enumerate(zip(packed.starts.tolist(), counts)):
        for j in range(max(0, c)):
            slots[i * each + j], pos[i * each + j] = int(packed.slots[s + j]) if b < 100 else None, None
    if b < 100:
        real = [s for s in slots if s >= 0]
        assert real == packed.slots.tolist()
        assert fixed.slots.tolist() == slots
    live = fixed.slots >= 0
    assert torch.equal(fixed.slots[live], packed.slots) and torch.equal(fixed.positions[live], packed.positions)
    want = torch.tensor([[j < c for j in range(each)] for c in counts], device="cuda").view(-1)
    assert torch.equal(live, want) and bool((fixed.positions[~live] == 0).all())
    too_many = [each + 1] + counts[1:]
    over = bf.paged_plan(t2, _i32(lens), _i32(too_many), free2, state, page_size=page, num_rows=b * each, rows_each=each)
    assert over.state.tolist() == [int(state[0]), 3] and bool((over.slots == -1).all()) and torch.equal(over.lengths, _i32(lens))
    with pytest.raises(ValueError, match="rows"):
        bf.paged_plan(t2, _i32(lens), _i32(counts), free2, state, page_size=page, num_rows=b * each + 1, rows_each=each)


def test_two_captured_attentions_replayed_at_once():
    """Each capture has a workspace of its own: replays on two streams at once give each its own result."""
    q, kp, vp, table, lens, _ = _paged_case([9000, 300, 7000], 8, 2, 128, 64, BF)
    qs = [q, q.flip(0).contiguous()]
    want = [bf.paged_attention(x, kp, vp, table, lens) for x in qs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in qs], [], []
    torch.cuda.synchronize()
    for x, s in zip(qs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            outs.append(bf.paged_attention(x, kp, vp, table, lens))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(6):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("batch,width", [(40, 8), (40, 70), (130, 20), (130, 200), (520, 12), (520, 400)])
def test_attention_batches_on_both_sides_of_each_split_rule(dtype, batch, width):
    """Narrow tables (one run a request, one launch) and wide ones, for few, some and many pairs of request and head."""
    r = random.Random(batch + width)
    lens = [r.choice([0, 1, 17, 64, r.randint(1, 32 * min(width, 60))]) for _ in range(batch)]
    _check_attention(*_paged_case(lens, 8, 4, 64, 32, dtype, width=width if width >= 60 else None))
