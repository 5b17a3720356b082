"""GPU: ``Decoder.score`` in parts over each kind of cache.

Log probabilities of logits that went other ways (products of one row and of many round at other places) agree as far as bf16
noise lets them: half the logits' standard deviation, as for scores in one call."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf

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
