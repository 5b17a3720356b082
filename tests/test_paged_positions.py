"""A ``PagedLayer`` given to the decoder's attention: every row at the position that the plan has for it, and every part
of a prompt behind what its own request holds.  On the CPU, the operators in plain torch operations.

Against the same attention over a list cache for each request alone, in fp32: the two do the same arithmetic in
other orders over at most 128 terms a sum (128 * 2^-24 of the terms' sizes) through four stages, well inside
2^-12 of the largest output; a row at another position differs by the output's own size."""
from __future__ import annotations

from dataclasses import replace

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd.decoder import Attention, Decoder, DecoderConfig, RopeTable, rope_cos_sin

from . import paged_plain

CFG = DecoderConfig(vocab_size=64, hidden_size=128, num_layers=2, num_heads=2, num_kv_heads=1, head_dim=64, intermediate_size=128)


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    paged_plain.install(monkeypatch)


def _attention():
    return Attention(CFG, generator=torch.Generator().manual_seed(3), device="cpu").float()


def _cache(requests, dtype=torch.float32, pages=40, page=16, layers=1):
    return bf.PagedKVCache(num_layers=layers, num_pages=pages, max_requests=requests, num_kv_heads=CFG.num_kv_heads,
                           head_dim=CFG.head_dim, page_size=page, dtype=dtype, device="cpu")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _close(got, want):
    assert got.shape == want.shape
    assert (got - want).abs().max() <= 2.0 ** -12 * want.abs().max()


class _Requests:
    """Requests over pages, and each of them over a list cache of its own."""

    def __init__(self, n):
        self.attn, self.pool, self.lists = _attention(), _cache(n), [[] for _ in range(n)]
        self.held, self.g = [0] * n, torch.Generator().manual_seed(n)

    def step(self, counts, each, rope=None):
        x = torch.randn(len(counts), each, CFG.hidden_size, generator=self.g)
        self.pool.begin(_i32(counts), each)
        y = self.attn(x, cache=self.pool.layers[0], position_embeddings=rope(self) if rope else None)
        for r, c in enumerate(counts):
            if c > 0:
                _close(y[r, :c], self.attn(x[r:r + 1, :c], cache=self.lists[r])[0])
                self.held[r] += c
        assert self.pool.lengths.tolist() == self.held and self.pool.sync() >= 0


def _table(_):
    return RopeTable(*rope_cos_sin(torch.arange(200), CFG.head_dim, CFG.rope_theta), None)


@pytest.mark.parametrize("rope", [None, _table])
def test_one_token_of_requests_of_different_lengths(rope):
    s = _Requests(4)
    s.step([7, 20, 0, 1], 20, rope)
    for counts in ([1, 1, 1, 1], [1, 0, 1, 1], [1, 1, 0, 0]):
        s.step(counts, 1, rope)


@pytest.mark.parametrize("rope", [None, _table])
def test_parts_behind_what_each_request_holds(rope):
    s = _Requests(3)
    s.step([20, 20, 20], 20, rope)        # prompts of one length
    s.step([3, 3, 3], 3, rope)            # drafts behind them
    s.step([5, 2, 0], 5, rope)            # counts below the step's rows, an idle request
    s.step([4, 4, 4], 4, rope)            # requests of different lengths
    s.step([0, 0, 0], 2, rope)
    s.step([1, 1, 1], 1, rope)


def test_rows_of_position_embeddings_of_each_requests_own():
    s = _Requests(2)
    s.step([9, 4], 9)
    own = lambda s: rope_cos_sin(torch.cat([torch.arange(n, n + 3) for n in s.held]), CFG.head_dim, CFG.rope_theta)
    s.step([3, 3], 3, own)
    one = lambda s: rope_cos_sin(torch.tensor(s.held), CFG.head_dim, CFG.rope_theta)
    s.step([1, 1], 1, one)
    shared = lambda s: rope_cos_sin(torch.arange(12, 15), CFG.head_dim, CFG.rope_theta)
    with pytest.raises(ValueError, match="own"):
        s.step([3, 3], 3, shared)
    with pytest.raises(ValueError, match="rows of position_embeddings"):
        s.step([3, 3], 3, lambda s: rope_cos_sin(torch.arange(4), CFG.head_dim, CFG.rope_theta))


def test_a_step_that_starts_elsewhere_is_refused():
    pool = _cache(2)
    pool.begin(_i32([7, 7]), 7, start=0)
    before = [x.clone() for x in (pool.lengths, pool.state, pool.block_table)]
    for start in (0, 6, 8):
        with pytest.raises(ValueError, match="hold"):
            pool.begin(_i32([2, 2]), 2, start=start)
    assert all(torch.equal(a, b) for a, b in zip(before, (pool.lengths, pool.state, pool.block_table)))
    pool.begin(_i32([2, 1]), 2, start=7)
    with pytest.raises(ValueError, match="hold"):
        pool.begin(_i32([2, 2]), 2, start=9)
    pool.begin(_i32([2, 2]), 2)


def test_a_part_of_a_prompt_goes_behind_the_tokens_that_are_there():
    model = Decoder(CFG, seed=1, device="cpu")
    tokens = torch.randint(0, CFG.vocab_size, (2, 30), generator=torch.Generator().manual_seed(1))
    pool = _cache(2, torch.bfloat16, layers=2)
    model.forward(tokens[:, :20], pool.layers, 0)
    for start in (0, 19, 30):
        with pytest.raises(ValueError, match="hold"):
            model.forward(tokens[:, 20:], pool.layers, start)
    got = model.forward(tokens[:, 20:], pool.layers, 20)
    lists = [[] for _ in range(2)]
    model.forward(tokens[:, :20], lists, 0)
    assert torch.equal(got, model.forward(tokens[:, 20:], lists, 20))
    assert pool.lengths.tolist() == [30, 30]


@pytest.mark.parametrize("tokens", [1, 5])
def test_greedy_starts_from_an_empty_cache(tokens):
    model = Decoder(CFG, seed=1, device="cpu")
    prompt = torch.randint(0, CFG.vocab_size, (2, tokens), generator=torch.Generator().manual_seed(1))
    pool = _cache(2, torch.bfloat16, layers=2)
    out = model.greedy(prompt, 4, pool.layers)
    held = pool.lengths.clone()
    for run in (model.greedy, model.greedy_graph):
        with pytest.raises(ValueError, match="hold"):
            run(prompt, 4, pool.layers)
    assert torch.equal(pool.lengths, held)
    pool.release(range(2))
    assert torch.equal(model.greedy(prompt, 4, pool.layers), out)


def test_steps_of_other_rows_are_refused():
    attn, pool = _attention(), _cache(3)
    x = torch.randn(3, 4, CFG.hidden_size)
    pool.begin_packed(_i32([6, 2, 4]), 12)
    for y in (x, x.view(1, 12, -1), x.view(12, 1, -1)):
        with pytest.raises(ValueError, match="packed rows"):
            attn(y, cache=pool.layers[0])
    pool.begin_packed(_i32([2, 0, 1]), 3)                     # three rows of two requests
    with pytest.raises(ValueError, match="packed rows"):
        attn(x[:, :1], cache=pool.layers[0])
    pool.begin(_i32([4, 4, 4]), 4)
    for y in (x.view(4, 3, -1), x.view(1, 12, -1), x[:, :1]):
        with pytest.raises(ValueError, match="4 rows of each"):
            attn(y, cache=pool.layers[0])


@pytest.mark.parametrize("head_dim,dtype,kv,error", [(32, torch.bfloat16, 1, NotImplementedError),
                                                     (96, torch.bfloat16, 1, NotImplementedError),
                                                     (64, torch.float32, 1, ValueError), (64, torch.bfloat16, 2, ValueError),
                                                     (128, torch.bfloat16, 1, ValueError)])
def test_a_cache_the_model_cannot_decode_over_is_refused_before_the_prompt(head_dim, dtype, kv, error):
    """head_dim is the cache's; the model has it too where no decode step would take it, else 64."""
    cfg = replace(CFG, head_dim=head_dim if head_dim in (32, 96) else 64)
    model = Decoder(cfg, seed=1, device="cpu")
    pool = bf.PagedKVCache(num_layers=2, num_pages=8, max_requests=2, num_kv_heads=kv, head_dim=head_dim, page_size=16,
                           dtype=dtype, device="cpu")
    prompt = torch.zeros(2, 5, dtype=torch.long)
    for run in (lambda: model.forward(prompt, pool.layers, 0), lambda: model.greedy(prompt, 3, pool.layers),
                lambda: model.greedy_graph(prompt, 3, pool.layers)):
        with pytest.raises(error):
            run()
    assert pool.lengths.tolist() == [0, 0] and pool.plan is None
    pool.begin(_i32([5, 5]), 5)
    x = torch.zeros(2, 5, CFG.hidden_size, dtype=torch.bfloat16)
    pages = pool.k_pages.zero_().clone()
    with pytest.raises(error):
        model.layers[0].self_attn(x, cache=pool.layers[0])
    assert torch.equal(pages, pool.k_pages)


def test_two_layers_do_not_share_their_pages():
    model, pool = Decoder(CFG, seed=1, device="cpu"), _cache(2, torch.bfloat16, layers=2)
    prompt = torch.zeros(2, 5, dtype=torch.long)
    for run in (lambda c: model.forward(prompt, c, 0), lambda c: model.greedy(prompt, 3, c)):
        with pytest.raises(ValueError, match="its own"):
            run([pool.layers[0]] * 2)
    assert pool.lengths.tolist() == [0, 0]


def test_an_fp32_attention_under_autocast_takes_bf16_pages():
    """The products' type counts.  (q, k and v are the same bf16 rows for both caches; the softmax's weights and its output
    are rounded at other places, half steps of 2^-8: 2^-5 of the largest covers them.)"""
    attn, pool, lists = _attention(), _cache(2, torch.bfloat16), []
    with torch.no_grad(), torch.autocast("cpu", torch.bfloat16):
        for t in (5, 1):
            x = torch.randn(2, t, CFG.hidden_size)
            pool.begin(_i32([t, t]), t)
            rope = rope_cos_sin(torch.arange(6)[-t:] if t == 1 else torch.arange(t), CFG.head_dim, CFG.rope_theta)
            y = attn(x, cache=pool.layers[0], position_embeddings=rope)
            want = attn(x, cache=lists, position_embeddings=rope)
            assert (y.float() - want.float()).abs().max() <= 2.0 ** -5 * want.float().abs().max()


@pytest.mark.parametrize("tokens", [1, 4])
def test_a_step_that_has_not_begun_is_refused(tokens):
    with pytest.raises(RuntimeError, match="begin"):
        _attention()(torch.zeros(2, tokens, CFG.hidden_size), cache=_cache(2).layers[0])
