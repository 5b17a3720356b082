"""GPU: the decoder over ``PagedKVCache(..., quant_bits=4)``, and its scores: eager, captured, beside swapped layers, and with
requests of different lengths.

Two paths that round at other places agree as far as bf16 noise lets them: within a quarter of the logits'
standard deviation, the bound that the swapped decoder is held to against its CPU reference.  Log probabilities differ by the
logit's difference and by the log of the sum's, each at most the largest logit's difference: half a deviation."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd.decoder import Decoder, DecoderConfig

pytestmark = pytest.mark.gpu


def _model(head_dim, layers=3, seed=11):
    cfg = DecoderConfig(vocab_size=2048, hidden_size=512, num_layers=layers, num_heads=512 // head_dim, num_kv_heads=2,
                        head_dim=head_dim, intermediate_size=1024)
    model = Decoder(cfg, seed=seed)
    for layer in model.layers:   # non-trivial q/k norm weights
        g = torch.Generator(device="cuda").manual_seed(head_dim)
        for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
            norm.weight.data = (1 + 0.3 * torch.randn(head_dim, generator=g, device="cuda")).bfloat16()
    return model, cfg


def _cache(cfg, requests, pages=64, page=32, quant_bits=4, **kw):
    return bf.PagedKVCache(num_layers=cfg.num_layers, num_pages=pages, max_requests=requests, num_kv_heads=cfg.num_kv_heads,
                           head_dim=cfg.head_dim, page_size=page, quant_bits=quant_bits, **kw)


def _tokens(cfg, *shape, seed=2):
    return torch.randint(0, cfg.vocab_size, shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _close(got, want):
    diff, spread = (got - want).abs().max().item(), want.std().item()
    assert diff <= 0.25 * spread, (diff, spread)


@pytest.mark.parametrize("batch,head_dim,group", [(1, 128, 64), (3, 64, 32), (2, 128, 32), (1, 256, 64)])
def test_steps_track_list_caches_of_what_the_pages_hold(batch, head_dim, group):
    """(A list cache's new row is exact, the pages' is codes: one of 75 rows and more, far inside the bound.)"""
    model, cfg = _model(head_dim)
    prompt, part = _tokens(cfg, batch, 75), _tokens(cfg, batch, 40, seed=3)
    pool, lists = _cache(cfg, batch, quant_group=group), [[] for _ in range(cfg.num_layers)]

    def held(n):
        for layer, kv in zip(pool.layers, lists):
            kv[:] = [x.clone() for x in layer.history(n)]

    _close(model.forward(prompt, pool.layers, 0), model.forward(prompt, lists, 0))
    held(75)
    _close(model.forward(part, pool.layers, 75), model.forward(part, lists, 75))
    for i in range(12):
        held(115 + i)
        tok = _tokens(cfg, batch, 1, seed=10 + i)
        _close(model.forward(tok, pool.layers, 115 + i), model.forward(tok, lists, 115 + i))
    assert pool.lengths.tolist() == [127] * batch and pool.sync() == 64 - batch * 4


@pytest.mark.parametrize("batch,head_dim,group", [(1, 128, 64), (3, 64, 32), (40, 128, 64)])
def test_captured_steps_equal_eager_ones(batch, head_dim, group):
    model, cfg = _model(head_dim)
    prompt = _tokens(cfg, batch, 50, seed=5)
    a, b = (_cache(cfg, batch, pages=4 * batch, quant_group=group) for _ in range(2))
    eager = model.greedy(prompt, 60, a.layers)
    assert torch.equal(eager, model.greedy_graph(prompt, 60, b.layers))
    assert torch.equal(a.lengths, b.lengths) and torch.equal(a.state, b.state)
    assert all(torch.equal(x, y) for l, m in zip(a.layers, b.layers) for x, y in zip(l.history(109), m.history(109)))


def test_captured_steps_beside_swapped_layers():
    model, cfg = _model(128, layers=4)
    assert bf.swap_qwen_attention_with_butterfly(model, cfg=bf.compressed_butterfly_config(), layer_indices=[0, 2]) == [0, 2]
    prompt = _tokens(cfg, 1, 300, seed=6)

    def caches():
        c = _cache(cfg, 1).layers[:]
        bf.install_compressed_kv_caches(model, c, layer_indices=[0, 2], block_size=128, local_window_tokens=64, max_kv_size=600)
        return c

    assert torch.equal(model.greedy(prompt, 40, caches()), model.greedy_graph(prompt, 40, caches()))


@pytest.mark.parametrize("quant_bits", [4, None])
@pytest.mark.parametrize("head_dim,requests", [(64, 4), (128, 35)])
def test_requests_with_log_probabilities(head_dim, requests, quant_bits):
    """Prompts, captured steps and log probabilities together; each request's are what its whole text scores alone, whose
    attention reads exact rows: over dense pages up to bf16 noise, and over 4-bit pages the same tokens that the run
    without log probabilities gives."""
    model, cfg = _model(head_dim)
    lens = [(1, 33, 120, 64)[r % 4] for r in range(requests)]
    prompts = [_tokens(cfg, n, seed=r) for r, n in enumerate(lens)]
    make = lambda: _cache(cfg, requests, pages=6 * requests, quant_bits=quant_bits)
    plain = model.greedy_requests(prompts, 30, make())
    pool = make()
    out, lps = model.greedy_requests(prompts, 30, pool, top_logprobs=4)
    assert torch.equal(out, plain) and pool.lengths.tolist() == [n + 29 for n in lens]
    assert lps.logprobs.shape == lps.entropy.shape == (requests, 30) and lps.top_tokens.shape == (requests, 30, 4)
    # a pick is the most probable, the lowest of equal ones
    assert torch.equal(lps.top_tokens[..., 0], out) and torch.equal(lps.top_logprobs[..., 0], lps.logprobs)
    assert bool((lps.logprobs < 0).all()) and bool((lps.entropy > 0).all())
    if quant_bits is None:
        for r in range(0, requests, 7):
            text = torch.cat([prompts[r], out[r]])[None]
            alone = model.score(text, [[] for _ in range(cfg.num_layers)], top=4)
            spread = model.forward(text, [[] for _ in range(cfg.num_layers)], 0).std().item()
            assert (alone.logprobs[0, lens[r] - 1:] - lps.logprobs[r]).abs().max().item() <= 0.5 * spread
    none = model.greedy_requests(prompts, 0, make(), top_logprobs=2)
    assert none[0].shape == (requests, 0) and none[1].top_logprobs.shape == (requests, 0, 2)
    for bad in (-1, 65):
        with pytest.raises(ValueError, match="top_logprobs"):
            model.greedy_requests(prompts, 3, make(), top_logprobs=bad)


def test_idle_requests_have_no_log_probabilities():
    model, cfg = _model(64)
    prompts = [_tokens(cfg, n, seed=n) for n in (20, 7, 50)]
    free, want = model.greedy_requests(prompts, 30, _cache(cfg, 3), top_logprobs=2)
    eos = int(free[1, 9])
    out, got = model.greedy_requests(prompts, 30, _cache(cfg, 3), eos_token=eos, top_logprobs=2)
    for r in range(3):
        hits = (free[r] == eos).nonzero()
        n = int(hits[0]) if len(hits) else 29
        assert torch.equal(out[r, :n + 1], free[r, :n + 1])
        assert all(torch.equal(a[r, :n + 1], b[r, :n + 1]) for a, b in zip(got, want))
        assert all(bool(x[r, n + 1:].isnan().all()) for x in got[:3]) and bool((got.top_tokens[r, n + 1:] == -1).all())


@pytest.mark.parametrize("length", [2, 3, 90])
def test_scores_over_each_cache(length):
    model, cfg = _model(128)
    text = _tokens(cfg, 3, length, seed=length)
    caches = [[[] for _ in range(cfg.num_layers)], _cache(cfg, 3, quant_bits=None).layers, _cache(cfg, 3).layers]
    scores = [model.score(text, c, top=5) for c in caches]
    for i in (0, length - 2):
        lg = model.forward(text[:, :i + 1], [[] for _ in range(cfg.num_layers)], 0).double()
        lp, spread = lg.log_softmax(-1), lg.std().item()
        for s in scores[:2] if i == 0 else scores:
            # (one token alone sees its own row only, as codes in the third)
            assert (s.logprobs[:, i] - lp.gather(1, text[:, i + 1:i + 2])[:, 0]).abs().max().item() <= 0.5 * spread
            assert (lp.gather(1, s.top_tokens[:, i]) - s.top_logprobs[:, i]).abs().max().item() <= 0.5 * spread
    assert all(c[0].cache.lengths.tolist() == [length - 1] * 3 for c in caches[1:])
