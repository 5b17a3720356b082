"""GPU: ``Decoder.score`` in parts over each kind of cache, and ``greedy_requests``' log probabilities by value.

Log probabilities of logits that went other ways (products of one row and of many round at other places) agree as far as bf16
noise lets them: half the logits' standard deviation, as for scores in one call.  Those of the same logits agree to fp32
rounding."""
from __future__ import annotations

import weakref

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd.decoder import RopeTable

from .test_gpu_paged_q4_decoder import _cache, _model, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,head_dim,kind", [(1, 128, "lists"), (3, 64, "pages"), (2, 128, "codes"), (3, 256, "codes"),
                                                 (1, 128, "swapped")])
@pytest.mark.parametrize("part", [1, 50, 64])
def test_parts_score_what_steps_over_the_same_caches_give(batch, head_dim, kind, part):
    model, cfg = _model(head_dim)
    if kind == "swapped":
        assert bf.swap_qwen_attention_with_butterfly(model, cfg=bf.compressed_butterfly_config(), layer_indices=[1]) == [1]
    text = _tokens(cfg, batch, 161, seed=part)

    def caches():
        if kind == "lists":
            return [[] for _ in range(cfg.num_layers)]
        c = _cache(cfg, batch, quant_bits=None if kind == "pages" else 4).layers[:]
        if kind == "swapped":
            bf.install_compressed_kv_caches(model, c, layer_indices=[1], block_size=128, local_window_tokens=64, max_kv_size=600)
        return c

    scored, stepped = caches(), caches()
    got = model.score(text, scored, top=4, part=part)
    assert got.logprobs.shape == (batch, 160) and got.top_tokens.shape == (batch, 160, 4)
    for i in range(0, 160, part):
        end = min(i + part, 160)
        lg = model.forward(text[:, i:end], stepped, i).double()
        lp, spread = lg.log_softmax(-1), lg.std().item()
        assert (got.logprobs[:, end - 1] - lp.gather(1, text[:, end:end + 1])[:, 0]).abs().max().item() <= 0.5 * spread
        assert (lp.gather(1, got.top_tokens[:, end - 1]) - got.top_logprobs[:, end - 1]).abs().max().item() <= 0.5 * spread
    for a, b in zip(scored, stepped):
        if isinstance(a, bf.PagedLayer):      # the same calls of the layers leave the same bits
            assert all(torch.equal(x, y) for x, y in zip(a.history(160), b.history(160)))
    if isinstance(scored[0], bf.PagedLayer):
        assert scored[0].cache.lengths.tolist() == [160] * batch


def test_codes_count_in_parts_and_not_in_one_call():
    model, cfg = _model(128)
    text = _tokens(cfg, 2, 161, seed=1)
    one, one4, parts, parts4 = (model.score(text, _cache(cfg, 2, quant_bits=bits).layers, part=part).logprobs
                                for part in (None, 16) for bits in (None, 4))
    assert torch.equal(one, one4)
    first = parts[:, :16] - parts4[:, :16]
    assert not bool(first.any()) and float((parts - parts4)[:, 16:].abs().mean()) > 0


@pytest.mark.parametrize("quant_bits", [4, None])
@pytest.mark.parametrize("head_dim,requests,top", [(64, 3, 5), (128, 35, 1), (128, 1, 0)])
def test_requests_log_probabilities_are_those_of_their_steps(head_dim, requests, top, quant_bits):
    """``greedy_requests``' steps once more, eagerly: the same logits, whose log-softmax in 64 bits is what it said."""
    model, cfg = _model(head_dim)
    prompts = [_tokens(cfg, (40, 1, 77)[r % 3], seed=r) for r in range(requests)]
    make = lambda: _cache(cfg, requests, pages=5 * requests, quant_bits=quant_bits)
    out, said = model.greedy_requests(prompts, 12, make(), top_logprobs=top)
    assert said.top_tokens.shape == said.top_logprobs.shape == (requests, 12, top)
    cache = make()
    steps = [torch.cat([model.forward(p[None], [[] for _ in range(cfg.num_layers)], 0) for p in prompts])]
    for r, p in enumerate(prompts):
        held = [[] for _ in range(cfg.num_layers)]
        model.forward(p[None], held, 0)
        counts = torch.zeros_like(cache.lengths)
        counts[r] = len(p)
        cache.begin_packed(counts, len(p))
        for layer, (k, v) in zip(cache.layers, held):
            layer.append(k[0].transpose(0, 1), v[0].transpose(0, 1))
    model._rope(0, 200, out.device)
    for i in range(11):
        cache.begin(torch.ones_like(cache.lengths))
        x = torch.nn.functional.embedding(out[:, i:i + 1], model.embed_tokens)
        steps.append(model._last_logits(x, None, cache.layers, RopeTable(*model._rope_tab, None)))
    for i, lg in enumerate(steps):
        assert torch.equal(lg.argmax(-1), out[:, i])
        lp = lg.double().log_softmax(-1)
        # sums of 2048 positive fp32 terms, 32 of them one after another and the rest pairwise: fewer than 64 steps of
        # 2^-24 of l, whose logarithm moves by as much; the entropy's second sum counts terms up to |x - m| <= 64
        near = dict(rtol=2.0 ** -20, atol=2.0 ** -17)
        torch.testing.assert_close(said.logprobs[:, i].double(), lp.gather(1, out[:, i:i + 1])[:, 0], **near)
        torch.testing.assert_close(said.entropy[:, i].double(), -(lp.exp() * lp).sum(-1), rtol=2.0 ** -14, atol=2.0 ** -14)
        torch.testing.assert_close(said.top_logprobs[:, i].double(), lp.sort(-1, descending=True).values[:, :top], **near)
        order = lg.float().sort(stable=True, dim=-1, descending=True).indices[:, :top]
        assert torch.equal(said.top_tokens[:, i], order)


@pytest.mark.parametrize("top", [None, 2])
def test_no_prompts_logits_wait_for_the_next(monkeypatch, top):
    model, cfg = _model(64)
    seen, alive, forward = [], [], model.forward

    def one(*args):
        alive.append(sum(x() is not None for x in seen))
        lg = forward(*args)
        seen.append(weakref.ref(lg))
        return lg

    monkeypatch.setattr(model, "forward", one)
    model.greedy_requests([_tokens(cfg, n, seed=n) for n in (20, 7, 50, 3)], 3, _cache(cfg, 4), top_logprobs=top)
    assert alive == [0] * 4 and not any(x() is not None for x in seen)
