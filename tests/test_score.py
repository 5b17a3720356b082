"""``Decoder.score``: what it refuses, and before what.  On the CPU, the paged operators in plain torch operations."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd.decoder import Decoder, DecoderConfig, _token_logprobs

from . import paged_plain, q4_plain

CFG = DecoderConfig(vocab_size=64, hidden_size=128, num_layers=2, num_heads=2, num_kv_heads=1, head_dim=64, intermediate_size=128)


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    paged_plain.install(monkeypatch)
    q4_plain.install(monkeypatch)


def _model():
    return Decoder(CFG, seed=1, device="cpu").float()


def _cache(requests, pages=40, quant_bits=4, **kw):
    return bf.PagedKVCache(num_layers=CFG.num_layers, num_pages=pages, max_requests=requests, num_kv_heads=CFG.num_kv_heads,
                           head_dim=CFG.head_dim, page_size=16, dtype=torch.float32, device="cpu", quant_bits=quant_bits, **kw)


def _text(b, t, seed=4):
    return torch.randint(0, CFG.vocab_size, (b, t), generator=torch.Generator().manual_seed(seed))


# --------------------------------------------------------------------------- caches that hold something
def test_list_caches_that_hold_a_text_are_refused():
    model, text, lists = _model(), _text(2, 9), [[] for _ in range(2)]
    first = model.score(text, lists)
    with pytest.raises(ValueError, match="empty caches: layer 0's holds 8"):
        model.score(text, lists)
    assert lists[0][0].shape[2] == 8
    with pytest.raises(ValueError, match="layer 1's holds 8"):
        model.score(text, [[], lists[1]])
    assert torch.equal(model.score(text, [None, None]).logprobs, first.logprobs)     # no cache at all


def test_a_compressed_cache_that_holds_a_text_is_refused():
    cache = bf.CompressedKVCache(block_size=16, local_window_tokens=32)
    cache.offset = 5
    with pytest.raises(ValueError, match="layer 1's holds 5"):
        _model().score(_text(2, 9), [[], cache])


# --------------------------------------------------------------------------- tops
@pytest.mark.parametrize("top,error", [(-1, ValueError), (65, ValueError), (2.5, TypeError)])
def test_a_top_out_of_range_is_refused_before_the_caches_change(top, error):
    model, text, pool, lists = _model(), _text(2, 9), _cache(2), [[], []]
    for caches in (pool.layers, lists):
        with pytest.raises(error, match="top 65|top -1|float"):
            model.score(text, caches, top=top)
    assert pool.lengths.tolist() == [0, 0] and pool.plan is None and lists == [[], []]


def test_a_top_beyond_a_small_vocabulary_is_refused():
    model = Decoder(DecoderConfig(**{**vars(CFG), "vocab_size": 40}), seed=1, device="cpu").float()
    with pytest.raises(ValueError, match="top 41 must be 0 to 40"):
        model.score(_text(1, 5) % 40, [[], []], top=41)
    assert model.score(_text(1, 5) % 40, [[], []], top=40).top_tokens.shape == (1, 4, 40)


# --------------------------------------------------------------------------- pages that cannot hold the text
@pytest.mark.parametrize("quant_bits", [4, None])
@pytest.mark.parametrize("kw,msg", [(dict(pages=3), "too few pages"), (dict(max_tokens=32), "outgrow")])
def test_a_text_that_does_not_fit_is_an_error(quant_bits, kw, msg):
    model, pool = _model(), _cache(2, quant_bits=quant_bits, **kw)
    with pytest.raises(RuntimeError, match=msg):
        model.score(_text(2, 40), pool.layers)
    assert pool.lengths.tolist() == [0, 0] and pool.state[1] == 0
    assert model.score(_text(2, 16), pool.layers).logprobs.shape == (2, 15)


def test_an_earlier_steps_error_is_reported_before_the_prefill():
    model, pool = _model(), _cache(1, pages=1)
    pool.begin(torch.tensor([20], dtype=torch.int32), 20)        # does not fit
    with pytest.raises(RuntimeError, match="outgrow"):
        model.score(_text(1, 9), pool.layers)
    assert pool.lengths.tolist() == [0]
    model.score(_text(1, 9), pool.layers)


# --------------------------------------------------------------------------- the CPU form
def test_the_cpu_form_ranks_and_marks_as_the_operator_does():
    """Ties go to the lower token, NaN above every number, a token outside the vocabulary is NaN."""
    nan, inf = float("nan"), float("inf")
    logits = torch.tensor([[1.0, 3.0, -0.0, 3.0, 0.0, -inf], [0.0, nan, 2.0, nan, inf, 1.0], [-inf] * 6, [5.0] * 6])
    own, entropy, tops, ids = _token_logprobs(logits, torch.tensor([5, 0, 1, -1]), 5)
    assert ids.tolist() == [[1, 3, 0, 2, 4], [1, 3, 4, 2, 5], [0, 1, 2, 3, 4], [0, 1, 2, 3, 4]]
    assert own[0] == -inf and bool(own[1:].isnan().all()) and bool(entropy[1:3].isnan().all())
    assert bool(tops[1:3].isnan().all()) and bool((tops[3] == tops[3, 0]).all()) and bool((tops[0].diff() <= 0).all())
    # one unit in the last place of log 6 and of the sum of six terms
    assert abs(entropy[3].item() - 1.791759469228055) <= 8 * 2.0 ** -24 * 1.8
    many = torch.zeros(3, 5000)
    assert _token_logprobs(many, torch.tensor([0, 5000, 4999]), 64).top_tokens.tolist() == [list(range(64))] * 3
    assert _token_logprobs(many, torch.tensor([0, 5000, 4999]), 0).logprobs.isnan().tolist() == [False, True, False]


def test_a_last_token_outside_the_vocabulary_scores_nan():
    text = _text(1, 6)
    text[0, -1] = CFG.vocab_size
    got = _model().score(text, [[], []]).logprobs[0]
    assert got.isnan().tolist() == [False] * 4 + [True]


# --------------------------------------------------------------------------- in parts
# Logits of some unit's size, fp32 sums of at most 128 terms through the layers in other orders: 2^-14 is 2^10 steps.
NEAR = dict(rtol=0, atol=2.0 ** -14)


@pytest.mark.parametrize("part", [1, 2, 7, 39, 100])
def test_parts_over_exact_caches_score_as_one_call(part):
    model, text = _model(), _text(2, 40)
    want = model.score(text, [[], []], top=3)
    for caches in ([[], []], _cache(2, quant_bits=None).layers):
        got = model.score(text, caches, top=3, part=part)
        for x, y in zip(got[:3], want[:3]):
            torch.testing.assert_close(x, y, **NEAR)
        held = caches[0][0].shape[2] if isinstance(caches[0], list) else caches[0].cache.lengths.tolist()[0]
        assert held == 39


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("part", [2, 7, 20])
def test_parts_over_pages_in_4_bits_read_their_codes(part, group):
    """Each token's score from a list cache of what the pages hold of earlier parts, and of its own part exactly."""
    model, text, pool = _model(), _text(2, 41), _cache(2, quant_group=group)
    got, exact = model.score(text, pool.layers, part=part), model.score(text, [[], []])
    for i in range(40):
        s = i // part * part
        lists = [[x.clone() for x in layer.history(s)] if s else [] for layer in pool.layers]
        lp = torch.log_softmax(model.forward(text[:, s:i + 1], lists, s).double(), -1)
        torch.testing.assert_close(got.logprobs[:, i].double(), lp.gather(1, text[:, i + 1:i + 2])[:, 0], **NEAR)
        torch.testing.assert_close(got.entropy[:, i].double(), -(lp.exp() * lp).sum(-1), **NEAR)
    # the first part reads no code; what 4 bits leave of the others is far from rounding
    torch.testing.assert_close(got.logprobs[:, :part], exact.logprobs[:, :part], **NEAR)
    assert (got.logprobs - exact.logprobs)[:, part:].abs().max() > 16 * NEAR["atol"]


def test_one_token_at_a_time_scores_what_decode_steps_see():
    model, text, pool, steps = _model(), _text(2, 30), _cache(2), _cache(2)
    got, exact = model.score(text, pool.layers, part=1), model.score(text, [[], []])
    for i in range(29):
        lp = torch.log_softmax(model.forward(text[:, i:i + 1], steps.layers, i).double(), -1)
        torch.testing.assert_close(got.logprobs[:, i].double(), lp.gather(1, text[:, i + 1:i + 2])[:, 0], **NEAR)
    assert (got.logprobs - exact.logprobs).abs().max() > 16 * NEAR["atol"]


def test_parts_that_are_refused():
    model, text, pool = _model(), _text(2, 9), _cache(2)
    for part, error in ((0, ValueError), (-3, ValueError), (2.5, TypeError)):
        with pytest.raises(error, match="at least 1|float"):
            model.score(text, pool.layers, part=part)
        with pytest.raises(error, match="at least 1|float"):
            model.score(text[:, :1], pool.layers, part=part)
    with pytest.raises(ValueError, match="layer 1 has none"):
        model.score(text, [[], None], part=4)
    with pytest.raises(RuntimeError, match="too few pages"):
        model.score(_text(2, 40), _cache(2, pages=3).layers, part=8)
    assert pool.lengths.tolist() == [0, 0] and pool.plan is None
    assert model.score(text, [None, None], part=8).logprobs.shape == (2, 8)
