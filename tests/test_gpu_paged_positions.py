"""GPU: the decoder's attention over pages, given a ``PagedLayer`` by itself, against the same attention over a list
cache for each request alone.

Both round q, k, the softmax weights and the output to bf16 at places of their own, half a step of 2^-8 each, and the
scores (at most sqrt(d) for normed heads) move by about 2^-8: 2^-5 of the largest output covers them.  A row at
another position or behind another history differs by the output's own size."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd.decoder import Attention, Decoder, DecoderConfig, RopeTable, add_rms_norm, rope_cos_sin

pytestmark = pytest.mark.gpu


def _config(head_dim):
    return DecoderConfig(vocab_size=64, hidden_size=512, num_layers=1, num_heads=4, num_kv_heads=2, head_dim=head_dim,
                         intermediate_size=512)


def _cache(cfg, requests, pages=40, page=16):
    return bf.PagedKVCache(num_layers=1, num_pages=pages, max_requests=requests, num_kv_heads=cfg.num_kv_heads,
                           head_dim=cfg.head_dim, page_size=page)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check_history(attn, cfg, layer, request, rows, start):
    """The request's keys and values from ``start`` on are those of the projection ``rows`` at their positions."""
    n, d = rows.shape[0], cfg.head_dim
    hk, hv = (x[:, :, start:] for x in layer.history(start + n, request))
    heads = rows.view(n, -1, d).transpose(0, 1)[None]
    assert torch.equal(hv, heads[:, -cfg.num_kv_heads:])
    k = heads[:, cfg.num_heads:cfg.num_heads + cfg.num_kv_heads].double()
    k = k / (k.square().mean(-1, keepdim=True) + attn.k_norm.eps).sqrt() * attn.k_norm.weight.double()
    cos, sin = (t.double() for t in rope_cos_sin(torch.arange(start, start + n, device="cuda"), d, cfg.rope_theta))
    turned = torch.cat([-k[..., d // 2:], k[..., :d // 2]], -1) * sin
    # fp32 arithmetic (some d 2^-24) and one or two roundings to bf16, the first before the turn
    bound = 2.0 ** -8 * 1.02 * ((k * cos).abs() + turned.abs()) + 2.0 ** -8 * (k * cos + turned).abs()
    assert bool(((hk.double() - (k * cos + turned)).abs() <= bound).all())


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("table", [False, True])
def test_rows_are_at_the_plans_positions(head_dim, table):
    cfg = _config(head_dim)
    attn = Attention(cfg, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    pool, lists, held, raw = _cache(cfg, 3), [[] for _ in range(3)], [0] * 3, [[] for _ in range(3)]
    rope = RopeTable(*rope_cos_sin(torch.arange(200, device="cuda"), head_dim, cfg.rope_theta), None) if table else None
    g = torch.Generator().manual_seed(5)
    for counts, each in [([20, 7, 0], 20), ([1, 1, 1], 1), ([1, 0, 1], 1), ([3, 3, 3], 3), ([5, 2, 0], 5), ([1, 1, 1], 1)]:
        x = torch.randn(3, each, cfg.hidden_size, generator=g).bfloat16().cuda()
        pool.begin(_i32(counts), each)
        with torch.no_grad():
            y = attn(x, cache=pool.layers[0], position_embeddings=rope)
            rows = attn.qkv(x)
        for r, c in enumerate(counts):
            if c > 0:
                want = attn(x[r:r + 1, :c], cache=lists[r])[0].float()
                assert (y[r, :c].float() - want).abs().max() <= 2.0 ** -5 * want.abs().max(), (counts, r)
                held[r] += c
                raw[r].append(rows[r, :c])
        assert pool.lengths.tolist() == held and pool.sync() >= 0
    for r in range(3):
        _check_history(attn, cfg, pool.layers[0], r, torch.cat(raw[r]), 0)


def test_several_tokens_are_not_captured():
    cfg = _config(64)
    attn = Attention(cfg, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    pool = _cache(cfg, 2)
    x = torch.randn(2, 4, cfg.hidden_size, device="cuda").bfloat16()
    counts = _i32([4, 4])
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.no_grad(), torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        pool.begin(counts, 4)
        with pytest.raises(RuntimeError, match="captured"):
            attn(x, cache=pool.layers[0])
    torch.cuda.synchronize()
    assert pool.lengths.tolist() == [0, 0]


def test_greedy_graph_goes_on_from_the_prefill_it_is_told():
    cfg = _config(64)
    model = Decoder(cfg, seed=1)
    prompt = torch.randint(0, cfg.vocab_size, (2, 9), generator=torch.Generator().manual_seed(1)).cuda()
    pool, other = _cache(cfg, 2), _cache(cfg, 2)
    out = model.greedy_graph(prompt, 6, pool.layers)
    with pytest.raises(ValueError, match="hold"):
        model.greedy_graph(prompt, 6, pool.layers)
    with pytest.raises(ValueError, match="hold"):
        model.greedy_graph(prompt[:, :1], 6, pool.layers)
    logits = model.forward(prompt, other.layers, 0)
    with pytest.raises(ValueError, match="at most 8"):       # the tables of its steps would be too short
        model.greedy_graph_from_logits(logits, 8, 6, other.layers)
    assert torch.equal(model.greedy_graph_from_logits(logits, 9, 6, other.layers), out)


class _Scaled(RopeTable):
    """Positions at half their distance."""

    def rows(self):
        return rope_cos_sin(self.pos.double() / 2, self.cos_tab.shape[1], 1e4)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("own", [False, True])
def test_a_table_with_rows_of_its_own_is_asked_for_them(head_dim, own):
    """A list cache asks it (``RopeTable.fits``): one token over pages turns as over a list."""
    cfg = _config(head_dim)
    attn = Attention(cfg, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    tabs = rope_cos_sin(torch.arange(64, device="cuda"), head_dim, cfg.rope_theta)
    pool, lists = _cache(cfg, 2), []
    g = torch.Generator().manual_seed(5)
    for i in range(8):
        x = torch.randn(2, 1, cfg.hidden_size, generator=g).bfloat16().cuda()
        pos = torch.tensor([i], device="cuda")
        table = _Scaled(*tabs, pos) if own else RopeTable(*tabs, pos)
        if not own:
            table.rows = lambda: rope_cos_sin(pos.double() / 2, head_dim, 1e4)
        pool.begin(_i32([1, 1]))
        with torch.no_grad():
            y = attn(x, cache=pool.layers[0], position_embeddings=table)
        want = attn(x, cache=lists, position_embeddings=table).float()
        assert (y.float() - want).abs().max() <= 2.0 ** -5 * want.abs().max()
    assert torch.equal(pool.layers[0].history(8)[0], lists[0]) and torch.equal(pool.layers[0].history(8)[1], lists[1])


@pytest.mark.parametrize("head_dim", [64, 128])
def test_captured_ragged_steps_leave_each_requests_own_rows(head_dim):
    """First layer: the prompts' keys and values are the list cache's, bit for bit, and each later row is its token's
    projection at its own position."""
    cfg = _config(head_dim)
    model = Decoder(cfg, seed=7)
    attn, norm = model.layers[0].self_attn, model.layers[0].input_layernorm
    g = torch.Generator(device="cuda").manual_seed(head_dim)
    for w in (attn.q_norm.weight, attn.k_norm.weight, norm.weight):
        w.data = (1 + 0.3 * torch.randn(w.shape, generator=g, device="cuda")).bfloat16()
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(n)).cuda() for n in (1, 33, 120, 64)]
    pool = _cache(cfg, 4)
    out = model.greedy_requests(prompts, 30, pool)
    steps = []
    with torch.no_grad():
        for i in range(29):
            x = torch.nn.functional.embedding(out[:, i:i + 1], model.embed_tokens)
            steps.append(attn.qkv(add_rms_norm(x, None, norm.weight, norm.eps)[1]))
    for r, p in enumerate(prompts):
        lists = [[]]
        model.forward(p[None], lists, 0)
        assert all(torch.equal(a, b) for a, b in zip(pool.layers[0].history(p.numel(), r), lists[0]))
        _check_history(attn, cfg, pool.layers[0], r, torch.cat([s[r] for s in steps]), p.numel())


@pytest.mark.parametrize("paged", [False, True])
def test_rows_of_position_embeddings_that_are_not_the_calls_are_refused(paged):
    """Their numbers of rows and columns are the kernel's bounds."""
    cfg = _config(128)
    attn = Attention(cfg, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    x = torch.randn(2, 6, cfg.hidden_size, device="cuda").bfloat16()
    cos, sin = rope_cos_sin(torch.arange(6, device="cuda"), 128, cfg.rope_theta)
    cache = []
    if paged:
        pool = _cache(cfg, 2)
        pool.begin(_i32([6, 6]), 6)
        cache = pool.layers[0]
    with torch.no_grad():
        for rope in [(cos[:, :64], sin[:, :64]), (cos[:5], sin[:5]), (cos, sin[:5]), (cos, sin[:, :64]), (cos.cpu(), sin.cpu()),
                     (cos, sin.cpu())]:
            with pytest.raises(ValueError):
                attn(x, cache=cache, position_embeddings=rope)
        attn(x, cache=cache, position_embeddings=(cos[None], sin[None]))
        if not paged:                  # rows behind the call's are not read
            want = attn(x, cache=[], position_embeddings=(cos, sin))
            longer = rope_cos_sin(torch.arange(9, device="cuda"), 128, cfg.rope_theta)
            assert torch.equal(attn(x, cache=[], position_embeddings=longer), want)


def test_a_captured_begin_and_its_replays():
    """The bookkeeping of several tokens captured, the attention outside: every replay is a step of its own."""
    cfg = _config(64)
    attn = Attention(cfg, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    pool, lists = _cache(cfg, 2), [[], []]
    counts, g = _i32([3, 2]), torch.Generator().manual_seed(1)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        pool.begin(counts, 3)
    for _ in range(4):
        graph.replay()
        x = torch.randn(2, 3, cfg.hidden_size, generator=g).bfloat16().cuda()
        with torch.no_grad():
            y = attn(x, cache=pool.layers[0])
        for r, c in enumerate((3, 2)):
            want = attn(x[r:r + 1, :c], cache=lists[r])[0].float()
            assert (y[r, :c].float() - want).abs().max() <= 2.0 ** -5 * want.abs().max()
    assert pool.lengths.tolist() == [12, 8]
