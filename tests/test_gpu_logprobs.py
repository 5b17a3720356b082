"""GPU: log probabilities, entropy and top alternatives against 64 bits.

Tolerances, with u = 2^-24 and a row of V logits: every term exp(x - m) is off by 4 u (the difference, its product with
log2 e -- differences beyond 88 add nothing -- and the exponential; |x - m| <= 20 counts and gives 20 u more), a thread
adds at most V / 256 of them with error u each in a random walk and the joins some 20 more: l and s are off by
less than 64 u (V up to 2^18: sqrt(1024) = 32), so log l by 64 u, and a log probability by 64 u + 2 u |lp| + 2 u |m|; s / l by
128 u of itself, and so the entropy by 64 u + 128 u H' with H' = |s / l| <= log V."""
from __future__ import annotations

import math

import pytest
import torch

import butterfly_amd as bf

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _oracle(x, tokens, top):
    x = x.double()
    v = x.shape[-1]
    logp = torch.log_softmax(x, -1)
    given = torch.where((tokens >= 0) & (tokens < v), logp.gather(-1, tokens.clamp(0, v - 1)[..., None])[..., 0], math.nan)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.where(p.isnan(), math.nan, 0.0)).sum(-1)
    # NaN first, then by value, equal ones by the lower index
    rank = torch.where(x.isnan(), math.inf, x)
    ids = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    ids = torch.stack([torch.cat([r[n[r]], r[~n[r]]]) for r, n in zip(ids.reshape(-1, v), x.isnan().reshape(-1, v))]) if \
        bool(x.isnan().any()) else ids.reshape(-1, v)
    ids = ids.view(x.shape)[..., :top]
    return given, entropy, logp.gather(-1, ids), ids


def _check(x, tokens, top):
    got = bf.token_logprobs(x, tokens, top=top)
    want = _oracle(x, tokens, top)
    assert torch.equal(got.top_tokens, want[3])
    m = x.double().nan_to_num(0.0, 0.0, 0.0).abs().amax(-1)
    for name, a, b in zip(got._fields, got[:3], want[:3]):
        assert a.shape == b.shape and a.dtype is torch.float32
        assert torch.equal(a.isnan(), b.isnan()), name
        # (a log probability of -6.8e38, between the type's lowest and its largest, is -inf in fp32)
        assert torch.equal(a == -math.inf, b.float() == -math.inf), name
        ok = torch.isfinite(b.float())
        size = m if b.dim() == m.dim() else m[..., None]
        room = 64 * U + 128 * U * (b.abs() + 13.0) if name == "entropy" else 64 * U + 2 * U * b.abs() + 2 * U * size
        assert bool(((a.double() - b).abs() <= room)[ok].all()), (name, ((a.double() - b).abs() - room)[ok].max())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 64), (1, 100), (4, 255), (3, 4097), (1, 8193), (2, 32003),
                                        (1, 151936), (40, 32000), (700, 5000), (1500, 129), (1, 262143)])
def test_rows_of_all_sizes(rows, vocab, dtype):
    g = _gen(vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    tokens = torch.randint(vocab, (rows,), generator=g, device="cuda")
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}):
        _check(x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [70001, 700001])
def test_orders_that_fill_the_list(dtype, v):
    """Rows that rise, fall, are all equal, hold few values, or rise in jumps: every round has more than its part of
    the top, and ties everywhere; 700001: two rounds of a workgroup to a kept maximum where it has the whole row."""
    i = torch.arange(v, device="cuda")
    rows = [i / v * 8, -i / v * 8, torch.zeros(v, device="cuda"), (i % 3).float(), (i * 7919 % v) / v * 8,
            (i // 8192).float(), -(i // 8192).float(), torch.where(i >= v - 64, 5.0, 0.0), torch.where(i % 257 == 0, 5.0, -1.0)]
    for parts in (1, len(rows)):                     # few rows: parts of a row; many: a workgroup a row
        x = torch.stack(rows).to(dtype)
        if parts == 1:
            x = x.repeat(150 if v < 100000 else 120, 1)
        tokens = torch.arange(x.shape[0], device="cuda") * 31 % v
        for top in (1, 20, 64):
            _check(x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [50, 9000])
def test_masks_infinities_and_nan(dtype, vocab):
    inf, low = math.inf, torch.finfo(dtype).min
    x = torch.randn(14, vocab, generator=_gen(3), device="cuda") * 2
    x[0, ::2] = -inf                                 # half ruled out
    x[1] = -inf                                      # everything: no distribution
    x[2] = low                                       # everything by the type's lowest value: uniform
    x[3, 1:] = low
    x[4, :40] = -inf
    x[5, 7] = inf
    x[6, 9] = math.nan
    x[7] = math.nan
    x[8, 3:] = -inf                                  # fewer left than asked for
    x[9] = torch.finfo(dtype).max
    x[10, ::3] = -0.0
    x[10, 1::3] = 0.0
    x[10, 2::3] = -1.0
    x[11, 5], x[11, 6] = math.nan, inf
    x[12] = low
    x[12, 11] = torch.finfo(dtype).max               # the widest difference there is
    x[13, 30:] = -inf
    x[13, 4] = math.nan
    x = x.to(dtype)
    tokens = torch.tensor([1, 0, 3, 0, 2, 7, 9, 1, 40, 0, 2, 5, 11, 8], device="cuda")
    for top in (0, 1, 5, 50):
        _check(x, tokens, top)
        got = _check(x, torch.tensor([-1, vocab, 1 << 40, -(1 << 40)] * 3 + [0, 1], device="cuda"), top)
        assert bool(got.logprobs[:12].isnan().all())
    # rows by themselves (parts of a row)
    for r in range(14):
        _check(x[r:r + 1], tokens[r:r + 1], 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 1100])
def test_few_tokens_left(dtype, rows):
    """Constrained rows: from none to some hundred logits are not -inf, in one place or all over; the rest of the top is
    the first -inf ones."""
    v = 20001
    x = torch.full((rows, v), -math.inf, device="cuda")
    g = _gen(rows)
    for r in range(rows):
        n = (0, 1, 3, 49, 50, 51, 64, 65, 200, 2000)[r % 10] if rows > 3 else (3, 63, 700)[r]
        at = torch.randperm(v, generator=g, device="cuda")[:n] if r % 3 else torch.arange(v - n, v, device="cuda") if r % 2 else \
            torch.arange(n, device="cuda")
        x[r, at] = torch.randn(n, generator=g, device="cuda") * 2
    for top in (5, 50, 64):
        _check(x.to(dtype), torch.arange(rows, device="cuda") % v, top)


def test_sure_rows():
    """One logit far above the rest: entropies near zero."""
    x = torch.randn(6, 4000, generator=_gen(5), device="cuda")
    x[torch.arange(6), torch.arange(6) * 600] = torch.tensor([10.0, 20.0, 40.0, 80.0, 300.0, 1e30], device="cuda")
    got = _check(x, torch.arange(6, device="cuda") * 600, 3)
    assert bool((got.entropy > -U * 64).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(dtype):
    """Rows at odd distances and addresses, expanded and transposed logits, leading dimensions."""
    g = _gen(8)
    base = (torch.randn(7, 6100, generator=g, device="cuda") * 3).to(dtype)
    tokens = torch.randint(3001, (7,), generator=g, device="cuda")
    for lo, hi in ((0, 3001), (1, 3002), (3, 3004), (5, 3006), (2, 2 + 3001)):
        y = base[:, lo:hi]
        # (sums are grouped by where 16-byte pieces lie: other roundings, the same order)
        assert torch.equal(_check(y, tokens, 9).top_tokens, _check(y.contiguous(), tokens, 9).top_tokens)
    flat = base.view(-1)[3:]                          # rows of an odd length, back to back
    _check(flat[:7 * 3001].view(7, 3001), tokens, 9)
    _check(base.t()[:3001], torch.arange(3001, device="cuda") % 7, 3)
    _check(base[:1, :3001].expand(7, 3001), tokens, 4)
    x = base[:6, :3000].reshape(2, 3, 3000)
    got = _check(x, torch.randint(3000, (2, 3), generator=g, device="cuda"), 4)
    assert got.logprobs.shape == (2, 3) and got.top_tokens.shape == (2, 3, 4)
    one = bf.token_logprobs(x[0, 0], torch.tensor(5, device="cuda"), top=2)
    assert one.logprobs.shape == () and one.top_tokens.shape == (2,)
    none = bf.token_logprobs(x[:0], torch.empty(0, 3, dtype=torch.int64, device="cuda"), top=2)
    assert none.logprobs.shape == (0, 3) and none.top_tokens.shape == (0, 3, 2)


def test_beyond_32_bits_of_offset():
    v = 1 << 20
    x = torch.zeros(2100, v, dtype=torch.bfloat16, device="cuda")       # 4.4 GB
    x[2099, 777] = 9.0
    x[2098, v - 1] = 4.0
    got = bf.token_logprobs(x, torch.full((2100,), 777, device="cuda"), top=1)
    assert got.top_tokens[2099].item() == 777 and got.top_tokens[2098].item() == v - 1 and got.top_tokens[0].item() == 0
    want = 9.0 - math.log(v - 1 + math.exp(9.0))
    assert abs(got.logprobs[2099].item() - want) <= 64 * U + 2 * U * (9 + abs(want))


def test_captured_and_on_other_streams():
    """Two captured graphs of split rows (workspaces of their own), replayed in turn with eager work between."""
    xs = [(torch.randn(2, 40000, generator=_gen(i), device="cuda") * 3).bfloat16() for i in range(2)]
    tokens = torch.tensor([5, 39999], device="cuda")
    side, graphs, outs = torch.cuda.Stream(), [], []
    for x in xs:
        bf.token_logprobs(x, tokens, top=7)
        graph = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            outs.append(bf.token_logprobs(x, tokens, top=7))
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(graph)
    for i in range(6):
        for x in xs:
            x.copy_((torch.randn(2, 40000, generator=_gen(100 + i), device="cuda") * 3).roll(i).bfloat16())
        for graph in graphs:
            graph.replay()
        for x, out in zip(xs, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, bf.token_logprobs(x, tokens, top=7)))
        torch.cuda.synchronize()


def test_refusals():
    x = torch.randn(3, 100, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    for a, b, kw in ((x.half(), t, {}), (x, t.int(), {}), (x, t[:2], {}), (x, t[:, None], {}), (x.cpu(), t, {}), (x, t.cpu(), {}),
                     (x, t, dict(top=65)), (x, t, dict(top=-1)), (x[:, :10], t, dict(top=11)), (x[:, :0], t, {}),
                     (x[0, 0], t[0], {}), (x.clone().requires_grad_(), t, {})):
        with pytest.raises(ValueError):
            bf.token_logprobs(a, b, **kw)
    with pytest.raises(TypeError):
        bf.token_logprobs(x, t, top=1.5)
    with torch.no_grad():
        bf.token_logprobs(x.clone().requires_grad_(), t)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangents"):
            bf.token_logprobs(torch.autograd.forward_ad.make_dual(x, x), t)
