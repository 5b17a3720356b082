"""GPU: the paged cache behind the decoder's dense layers: eager, captured, beside swapped layers, and with
requests of different lengths.

Two paths that round at other places agree as far as bf16 noise lets them: within a quarter of the logits'
standard deviation, the bound that the swapped decoder is held to against its CPU reference."""
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


def _cache(cfg, requests, pages=64, page=32, **kw):
    return bf.PagedKVCache(num_layers=cfg.num_layers, num_pages=pages, max_requests=requests, num_kv_heads=cfg.num_kv_heads,
                           head_dim=cfg.head_dim, page_size=page, **kw)


def _close(got, want):
    diff = (got - want).abs().max().item()
    spread = want.std().item()
    assert diff <= 0.25 * spread, (diff, spread)
    for g, w in zip(got, want):
        top = w.topk(2).values
        if (top[0] - top[1]).item() > 2 * diff:
            assert g.argmax() == w.argmax()


@pytest.mark.parametrize("batch,head_dim", [(1, 128), (3, 64), (1, 64), (2, 128)])
def test_paged_steps_track_the_list_cache(batch, head_dim):
    model, cfg = _model(head_dim)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, cfg.vocab_size, (batch, 75), generator=g).cuda()
    pool, lists = _cache(cfg, batch), [[] for _ in range(cfg.num_layers)]
    _close(model.forward(prompt, pool.layers, 0), model.forward(prompt, lists, 0))
    # a further part of the prompts: dense attention over what the pages hold and the part
    part = torch.randint(0, cfg.vocab_size, (batch, 40), generator=g).cuda()
    _close(model.forward(part, pool.layers, 75), model.forward(part, lists, 75))
    for i in range(30):
        tok = torch.randint(0, cfg.vocab_size, (batch, 1), generator=g).cuda()
        _close(model.forward(tok, pool.layers, 115 + i), model.forward(tok, lists, 115 + i))
    assert pool.lengths.tolist() == [145] * batch and pool.sync() == 64 - batch * 5
    for layer, (k, v) in zip(pool.layers, lists):        # the pages hold what the list does, up to q/k rounding
        hk, hv = layer.history(145)
        assert hk.shape == k.shape
        # first layer: the values are the same projection rows
        if layer is pool.layers[0]:
            assert torch.equal(hv, v)
            torch.testing.assert_close(hk.float(), k.float(), rtol=2.0 ** -6, atol=2.0 ** -6)


@pytest.mark.parametrize("batch,head_dim", [(1, 128), (3, 64)])
def test_captured_paged_steps_equal_eager_ones(batch, head_dim):
    model, cfg = _model(head_dim)
    prompt = torch.randint(0, cfg.vocab_size, (batch, 50), generator=torch.Generator().manual_seed(5)).cuda()
    a, b = _cache(cfg, batch), _cache(cfg, batch)
    eager = model.greedy(prompt, 60, a.layers)
    graphed = model.greedy_graph(prompt, 60, b.layers)
    assert torch.equal(eager, graphed)
    assert torch.equal(a.lengths, b.lengths) and torch.equal(a.state, b.state)
    assert all(torch.equal(x, y) for l, m in zip(a.layers, b.layers) for x, y in zip(l.history(109), m.history(109)))


def test_captured_steps_of_swapped_and_dense_layers_together():
    """Layers 0 and 2 swapped (compressed caches), 1 and 3 dense over pages: the captured steps give the eager
    steps' tokens, and track the same model with list caches in the dense layers."""
    model, cfg = _model(128, layers=4)
    swapped = bf.swap_qwen_attention_with_butterfly(model, cfg=bf.compressed_butterfly_config(), layer_indices=[0, 2])
    assert swapped == [0, 2]
    prompt = torch.randint(0, cfg.vocab_size, (1, 300), generator=torch.Generator().manual_seed(6)).cuda()

    def caches(paged):
        pool = _cache(cfg, 1)
        c = pool.layers[:] if paged else [[] for _ in range(4)]
        bf.install_compressed_kv_caches(model, c, layer_indices=[0, 2], block_size=128, local_window_tokens=64, max_kv_size=600)
        return c

    eager = model.greedy(prompt, 40, caches(True))
    graphed = model.greedy_graph(prompt, 40, caches(True))
    assert torch.equal(eager, graphed)
    paged, lists = caches(True), caches(False)
    toks = torch.cat([prompt, eager], 1)
    _close(model.forward(toks[:, :300], paged, 0), model.forward(toks[:, :300], lists, 0))
    for i in range(300, 320):
        _close(model.forward(toks[:, i:i + 1], paged, i), model.forward(toks[:, i:i + 1], lists, i))


@pytest.mark.parametrize("head_dim", [64, 128])
def test_requests_of_different_lengths_decode_as_each_alone(head_dim):
    model, cfg = _model(head_dim)
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).cuda() for n in (1, 33, 120, 64)]
    pool = _cache(cfg, 4, pages=40)
    out = model.greedy_requests(prompts, 50, pool)
    assert out.shape == (4, 50) and pool.lengths.tolist() == [p.numel() + 49 for p in prompts]
    used = sum(-(-(p.numel() + 49) // 32) for p in prompts)
    assert pool.sync() == 40 - used
    for r, p in enumerate(prompts):
        lists = [[] for _ in range(cfg.num_layers)]
        lg, at = model.forward(p[None], lists, 0), p.numel()
        for i in range(50):
            spread = lg.std().item()
            # the batch's pick is the largest logit of the request alone, up to the noise between the two
            assert (lg.max() - lg[0, out[r, i]]).item() <= 0.5 * spread, (r, i)
            lg, at = model.forward(out[r:r + 1, i:i + 1], lists, at), at + 1
    pool.release([0, 2])
    assert pool.lengths.tolist() == [0, 33 + 49, 0, 64 + 49]
    assert pool.sync() == 40 - 3 - 4
    with pytest.raises(ValueError, match="empty"):
        model.greedy_requests(prompts, 50, pool)
    for bad in ([4], [-1]):
        with pytest.raises(ValueError):
            pool.release(bad)
    pool.release([])
    pool.release([1, 3, 1])
    again = model.greedy_requests(prompts, 50, pool)
    assert torch.equal(out, again)


def test_requests_stop_at_the_eos_token():
    model, cfg = _model(64)
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).cuda() for n in (20, 7, 50)]
    free = model.greedy_requests(prompts, 30, _cache(cfg, 3))
    eos = int(free[1, 9])
    pool = _cache(cfg, 3)
    out = model.greedy_requests(prompts, 30, pool, eos_token=eos)
    for r in range(3):
        hits = (free[r] == eos).nonzero()
        n = int(hits[0]) if len(hits) else 29
        assert torch.equal(out[r, :n + 1], free[r, :n + 1]) and bool((out[r, n:] == out[r, n]).all())
        # tokens 0..n - 1 went through a step (n is the eos itself: it is not fed)
        assert int(pool.lengths[r]) == prompts[r].numel() + n


def test_running_out_of_pages_is_reported():
    model, cfg = _model(64)
    prompt = torch.randint(0, cfg.vocab_size, (2, 60), generator=torch.Generator().manual_seed(1)).cuda()
    with pytest.raises(RuntimeError, match="too few pages"):
        model.greedy_graph(prompt, 20, _cache(cfg, 2, pages=4).layers)
    pool = _cache(cfg, 2, pages=4)
    with pytest.raises(RuntimeError, match="too few pages"):
        model.greedy(prompt, 20, pool.layers)
    assert pool.lengths.tolist() == [64, 64] and pool.sync() == 0       # the error is cleared, the rest stands
    with pytest.raises(RuntimeError, match="outgrow"):
        model.greedy(prompt, 20, _cache(cfg, 2, pages=40, max_tokens=64).layers)
    with pytest.raises(ValueError, match="batch"):
        model.forward(prompt, _cache(cfg, 3).layers, 0)
    with pytest.raises(ValueError):
        model.greedy_requests([prompt[0]], 5, _cache(cfg, 2))
    with pytest.raises(ValueError):
        model.greedy_requests([prompt[0], prompt[0, :0]], 5, _cache(cfg, 2))
    with pytest.raises(RuntimeError, match="begin"):
        pool = _cache(cfg, 2)
        pool.layers[0].append(torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda"))
    for kw in (dict(page=48), dict(pages=0), dict(max_tokens=0), dict(dtype=torch.float16)):
        with pytest.raises(ValueError):
            _cache(cfg, 2, **kw)


def test_one_request_rides_its_norm_in_the_projection_and_hooks_are_seen():
    """hidden 2048: the step's input norm rides in the q|k|v product's launch (bit-identical to the two); a hook on the
    attention or its projection takes the separate calls, and runs."""
    cfg = DecoderConfig(vocab_size=1024, hidden_size=2048, num_layers=2, num_heads=16, num_kv_heads=4, head_dim=128,
                        intermediate_size=1024)
    model = Decoder(cfg, seed=4)
    prompt = torch.randint(0, cfg.vocab_size, (1, 70), generator=torch.Generator().manual_seed(3)).cuda()
    want = model.greedy_graph(prompt, 20, _cache(cfg, 1).layers)
    for module in (model.layers[0].self_attn, model.layers[1].self_attn.qkv):
        seen = []
        hook = module.register_forward_hook(lambda *a: seen.append(1))
        got = model.greedy(prompt, 20, _cache(cfg, 1).layers)
        hook.remove()
        assert len(seen) == 20 and torch.equal(got, want)
    assert torch.equal(model.greedy(prompt, 20, _cache(cfg, 1).layers), want)
