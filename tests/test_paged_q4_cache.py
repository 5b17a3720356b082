"""``PagedKVCache(..., quant_bits=4)`` given to the decoder's attention, and ``Decoder.score``.  On the CPU, the operators in
plain torch operations.

Each request's step against the same attention over dense tensors: what the pages hold, read back, and behind it the
step's own rows (of one token its row as the pages hold it, as ``attend`` reads it).  In fp32 both do the same arithmetic
in other orders over at most 128 terms a sum (128 * 2^-24 of the terms' sizes) through four stages, well inside 2^-12 of the
largest output; a row at another position differs by the output's own size."""
from __future__ import annotations

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd import decoder
from butterfly_amd.decoder import Attention, Decoder, DecoderConfig, RopeTable, rope_cos_sin

from . import paged_plain, q4_plain

CFG = DecoderConfig(vocab_size=64, hidden_size=128, num_layers=2, num_heads=2, num_kv_heads=1, head_dim=64, intermediate_size=128)


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    paged_plain.install(monkeypatch)
    q4_plain.install(monkeypatch)


def _cache(requests, dtype=torch.float32, pages=40, page=16, layers=1, **kw):
    return bf.PagedKVCache(num_layers=layers, num_pages=pages, max_requests=requests, num_kv_heads=CFG.num_kv_heads,
                           head_dim=CFG.head_dim, page_size=page, dtype=dtype, device="cpu", quant_bits=4, **kw)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _close(got, want):
    assert got.shape == want.shape
    assert (got - want).abs().max() <= 2.0 ** -12 * want.abs().max()


class _Requests:
    def __init__(self, n, group):
        self.attn = Attention(CFG, generator=torch.Generator().manual_seed(3), device="cpu").float()
        self.pool, self.group = _cache(n, quant_group=group), group
        self.rows, self.g = [None] * n, torch.Generator().manual_seed(n)

    def step(self, counts, each, rope=None):
        attn, layer = self.attn, self.pool.layers[0]
        x = torch.randn(len(counts), each, CFG.hidden_size, generator=self.g)
        self.pool.begin(_i32(counts), each)
        y = attn(x, cache=layer, position_embeddings=rope)
        for r, c in enumerate(counts):
            if c <= 0:
                continue
            held = 0 if self.rows[r] is None else self.rows[r][0].shape[2]
            q, *new = attn.project(x[r:r + 1, :c], torch.arange(held, held + c), None)
            self.rows[r] = new if self.rows[r] is None else [torch.cat(z, 2) for z in zip(self.rows[r], new)]
            pages = layer.history(held + c, r)
            for got, want in zip(pages, self.rows[r]):
                # half a step of the group, and the roundings (2^-8 each) of its scale, 15 of them, and its bias
                z = want.unflatten(-1, (-1, self.group))
                span = z.amax(-1, keepdim=True) - z.amin(-1, keepdim=True)
                bound = span / 30 + 2.0 ** -7 * (span + z.abs().amax(-1, keepdim=True))
                assert ((got.unflatten(-1, (-1, self.group)) - z).abs() <= bound).all()
            kv = pages if each == 1 else [torch.cat((p[:, :, :held], z), 2) for p, z in zip(pages, new)]
            _close(y[r, :c], attn.output(attn._dense(q, *kv))[0])
        assert self.pool.lengths.tolist() == [0 if z is None else z[0].shape[2] for z in self.rows] and self.pool.sync() >= 0


@pytest.mark.parametrize("rope", [None, RopeTable(*rope_cos_sin(torch.arange(200), CFG.head_dim, CFG.rope_theta), None)])
@pytest.mark.parametrize("group", [32, 64])
def test_steps_over_pages_in_4_bits(rope, group):
    s = _Requests(4, group)
    s.step([7, 20, 0, 1], 20, rope)
    for counts in ([1, 1, 1, 1], [1, 0, 1, 1]):
        s.step(counts, 1, rope)
    s.step([5, 2, 0, 16], 16, rope)       # parts behind what each holds
    s.step([0, 0, 0, 0], 2, rope)
    s.step([1, 1, 1, 1], 1, rope)


def test_the_cache_and_its_refusals():
    dense = bf.PagedKVCache(num_layers=2, num_pages=8, max_requests=2, num_kv_heads=1, head_dim=128, page_size=16, device="cpu")
    packed = bf.PagedKVCache(num_layers=2, num_pages=8, max_requests=2, num_kv_heads=1, head_dim=128, page_size=16, device="cpu",
                             quant_bits=4)
    assert dense.pages is None and packed.k_pages is None
    assert dense.nbytes * 9 == packed.nbytes * 32        # (128 + 8) / 2 bits an element more: 16 to 4.5
    assert len(packed.layers) == 2 and all(isinstance(x, bf.PagedLayer) for x in packed.layers)
    packed.layers[1].pages.k_codes.fill_(3)
    assert int(packed.pages.k_codes[1].min()) == 3       # the layers are views of the cache's tensors
    packed.check_heads(1, 128, torch.bfloat16)
    for heads, d, dtype in ((2, 128, torch.bfloat16), (1, 64, torch.bfloat16), (1, 128, torch.float32)):
        with pytest.raises(ValueError, match="cannot take"):
            packed.check_heads(heads, d, dtype)
    for kw, error in ((dict(quant_bits=8), ValueError), (dict(quant_bits=0), ValueError), (dict(quant_group=16), ValueError),
                      (dict(page=24), ValueError)):
        with pytest.raises(error):
            _cache(1, **{"layers": 1, **kw}) if "quant_bits" not in kw else bf.PagedKVCache(
                num_layers=1, num_pages=4, max_requests=1, num_kv_heads=1, head_dim=64, device="cpu", **kw)
    with pytest.raises(NotImplementedError, match="head_dim"):
        bf.PagedKVCache(num_layers=1, num_pages=4, max_requests=1, num_kv_heads=1, head_dim=96, device="cpu", quant_bits=4)


def test_a_model_over_pages_in_4_bits():
    model = Decoder(CFG, seed=1, device="cpu")
    prompt = torch.randint(0, CFG.vocab_size, (2, 20), generator=torch.Generator().manual_seed(1))
    pool, lists = _cache(2, torch.bfloat16, layers=2), [[] for _ in range(2)]
    # a prompt attends to its own rows, not to their codes
    assert torch.equal(model.forward(prompt, pool.layers, 0), model.forward(prompt, lists, 0))
    with pytest.raises(ValueError, match="hold"):
        model.forward(prompt, pool.layers, 19)
    again = _cache(2, torch.bfloat16, layers=2)
    out = model.greedy(prompt, 6, again.layers)
    for i in range(5):
        lg = model.forward(out[:, i:i + 1], pool.layers, 20 + i)
        assert torch.equal(lg.argmax(-1), out[:, i + 1])
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for x, y in zip(pool.layers, again.layers)
               for a, b in zip(x.history(25), y.history(25)))
    with pytest.raises(ValueError, match="empty|hold"):
        model.greedy(prompt, 3, again.layers)
    with pytest.raises(ValueError, match="cannot take"):
        model.forward(prompt, _cache(2, layers=2).layers, 0)         # fp32 rows


# --------------------------------------------------------------------------- Decoder.score
def _float_model():
    return Decoder(CFG, seed=1, device="cpu").float()


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("rows", [None, 1, 5])
def test_score_is_the_log_softmax_of_each_prefix(monkeypatch, paged, rows):
    if rows:
        monkeypatch.setattr(decoder, "SCORE_LOGITS", rows * CFG.vocab_size + 3)
    model = _float_model()
    tokens = torch.randint(0, CFG.vocab_size, (2, 9), generator=torch.Generator().manual_seed(4))
    caches = _cache(2, layers=2).layers if paged else [[] for _ in range(2)]
    got = model.score(tokens, caches, top=3)
    assert got.logprobs.shape == got.entropy.shape == (2, 8) and got.top_logprobs.shape == got.top_tokens.shape == (2, 8, 3)
    for i in range(8):
        lp = torch.log_softmax(model.forward(tokens[:, :i + 1], [[] for _ in range(2)], 0).double(), -1)
        # logits of some unit's size, fp32 sums of at most 128 terms through the layers: 2^-14 is 2^10 steps
        near = dict(rtol=0, atol=2.0 ** -14)
        torch.testing.assert_close(got.logprobs[:, i].double(), lp.gather(1, tokens[:, i + 1:i + 2])[:, 0], **near)
        torch.testing.assert_close(got.entropy[:, i].double(), -(lp.exp() * lp).sum(-1), **near)
        torch.testing.assert_close(got.top_logprobs[:, i].double(), lp.topk(3).values, **near)
        torch.testing.assert_close(lp.gather(1, got.top_tokens[:, i]), lp.topk(3).values, **near)
    held = caches[0].cache.lengths.tolist() if paged else [caches[0][0].shape[2]] * 2
    assert held == [8, 8]


def test_score_of_short_texts_and_its_refusals():
    model = _float_model()
    one = model.score(torch.zeros(3, 1, dtype=torch.long), [[], []], top=2)
    assert one.logprobs.shape == (3, 0) and one.top_tokens.shape == (3, 0, 2) and one.top_tokens.dtype is torch.long
    two = model.score(torch.zeros(3, 2, dtype=torch.long), _cache(3, layers=2).layers)
    assert two.logprobs.shape == (3, 1) and two.top_tokens.shape == (3, 1, 0) and bool((two.logprobs < 0).all())
    for bad in (torch.zeros(3, 0, dtype=torch.long), torch.zeros(3, dtype=torch.long)):
        with pytest.raises(ValueError, match="at least one token"):
            model.score(bad, [[], []])
    pool = _cache(1, layers=2)
    text = torch.zeros(1, 5, dtype=torch.long)
    model.score(text, pool.layers)
    with pytest.raises(ValueError, match="hold"):
        model.score(text, pool.layers)
