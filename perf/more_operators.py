"""Serving from a 4-bit paged cache, and what a decoder's logits say, as cases that can be timed and compared.

Keys and values of the dense layers are held in pages of 4-bit codes (``codes`` uint8 [pages, kv heads, page, d / 2])
with a scale and a bias for each ``group`` of elements (``scales`` bf16 [pages, kv heads, page, d / group, 2]).
Five operators (``op``):

* ``append``: rows of keys and values into their slots, quantised; then the pages read back as values.
* ``rope_append``: the same for a decoder's projection rows, with the q/k norm and RoPE on the way.
* ``read``: the first tokens of every request as dense keys and values.
* ``attention``: one new token of every request over its pages.
* ``logprobs``: log probabilities of given tokens, with entropy and the top alternatives, from logits.

``run`` computes a case with the framework's kernels where ``own`` is true and in plain torch operations
otherwise; ``exact`` computes the same outputs in 64 bits, by another route.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # a further part of a prompt: its rows go in, heads first as the prefill leaves them, and the layer reads back
        # what its dense attention sees
        dict(name="append_part", op="append", dtype="bf16", rows=4099, hkv=4, d=128, page=128, group=64, heads_first=True),
        # a step's rows of an fp32 layer, in the finer groups
        dict(name="append_fp32_step", op="append", dtype="fp32", rows=8, hkv=2, d=128, page=64, group=32, heads_first=False),
        # a decode step of 32 requests: columns of one fused projection row each
        dict(name="rope_step_b32", op="rope_append", dtype="bf16", rows=32, hq=16, hkv=4, d=128, rot=128, page=128, group=64,
             context=32768, norm=True),
        # prompts through wide heads, a quarter of each rotated
        dict(name="rope_prompt", op="rope_append", dtype="bf16", rows=16411, hq=16, hkv=4, d=256, rot=64, page=128, group=64,
             context=32768, norm=True),
        # the 4-bit decoder's benchmark prompt, read for a further part's dense attention
        dict(name="read_32k_b1", op="read", dtype="bf16", batch=1, tokens=32768, hkv=4, d=128, page=128, group=64),
        # a few short requests in small pages
        dict(name="read_b5", op="read", dtype="fp32", batch=5, tokens=777, hkv=2, d=64, page=16, group=32),
        # short requests in small pages, an empty one among them: latency
        dict(name="attn_short_b8", op="attention", dtype="fp32", batch=8, hq=8, hkv=2, d=64, context=300, page=16, group=32,
             window=0, ragged=4, stats=True),
        # one sequence of the 4-bit decoder's benchmark after its 32k-token prompt
        dict(name="attn_32k_b1", op="attention", dtype="bf16", batch=1, hq=16, hkv=4, d=128, context=32768, page=128, group=64,
             window=0, ragged=0, stats=False),
        # the batched decode benchmark's heads and contexts, lengths of a mixed load
        dict(name="attn_131k_b32", op="attention", dtype="bf16", batch=32, hq=8, hkv=2, d=128, context=131072, page=128,
             group=64, window=0, ragged=5, stats=False),
        # a decode step that reports its pick: one row of the decoder's vocabulary
        dict(name="logprobs_step", op="logprobs", dtype="bf16", rows=1, vocab=151936, top=5, masked=0.0),
        # constrained decoding of a batch: fp32 logits over an odd vocabulary, most of it ruled out
        dict(name="logprobs_masked_b32", op="logprobs", dtype="fp32", rows=32, vocab=32003, top=50, masked=0.97),
        # a text scored by the decoder
        dict(name="logprobs_score", op="logprobs", dtype="bf16", rows=2048, vocab=151936, top=20, masked=0.0),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "rope_append", "read", "attention", "attention", "attention", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "logprobs":
        vocab = _log(rng, 100, 262144)
        most = 2048 * 151936 // vocab
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(16384, most if dtype == "bf16" else most // 2)), vocab=vocab,
                    top=rng.choice([0, 1, 5, 20, 50, 64]), masked=rng.choice([0.0, 0.0, 0.5, 0.999]))
    page, group = rng.choice([16, 32, 64, 128, 256]), rng.choice([32, 64, 64])
    hkv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    c = dict(op=op, dtype=dtype, hkv=hkv, d=d, page=page, group=group)
    if op == "append":
        return dict(c, rows=_log(rng, 1, 8192), heads_first=rng.random() < 0.5)
    if op == "read":
        batch = _log(rng, 1, 16)
        return dict(c, batch=batch, tokens=_log(rng, 1, min(32768, (1 << 25) // (batch * hkv * d))))
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    if op == "rope_append":
        most = 16411 * 24 * 256 // ((hq + 2 * hkv) * d)
        return dict(c, rows=_log(rng, 1, min(16384, most)), hq=hq, rot=rng.choice([d, d, d // 2, d // 4]),
                    context=_log(rng, 64, 131072), norm=rng.random() < 0.75)
    batch = _log(rng, 1, 64)
    # keys and values take at most a billion elements (the largest listed case has more)
    most = (1 << 29) // (batch * hkv * d)
    return dict(c, batch=batch, hq=hq, context=_log(rng, 1, max(1, min(131072, most))),
                window=rng.choice([0, 0, rng.randint(1, 5000)]), ragged=rng.choice([0, 1, 1]) * rng.randint(1, 1 << 30),
                stats=rng.random() < 0.5)


def _lengths(c):
    """The requests' lengths: every one the context, or (ragged) from a mixed load with empty places."""
    if not c["ragged"]:
        return [c["context"]] * c["batch"]
    r = random.Random(c["ragged"])
    lens = [0 if r.random() < 0.08 else _log(r, max(1, c["context"] // 32), c["context"]) for _ in range(c["batch"])]
    lens[r.randrange(len(lens))] = c["context"]
    return lens


def work(c):
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "logprobs":
        return {"bytes": c["rows"] * (c["vocab"] * e + 16 + 12 * c["top"]), "flops": 4 * c["rows"] * c["vocab"]}
    d, hkv = c["d"], c["hkv"]
    row = d // 2 + 4 * d // c["group"]                  # codes, scales and biases of a head's row
    if c["op"] == "read":
        return {"bytes": c["batch"] * c["tokens"] * hkv * 2 * (row + d * e), "flops": 2 * c["batch"] * c["tokens"] * hkv * d}
    if c["op"] == "attention":
        w = c["window"]
        keys = sum(min(n, w) if w else n for n in _lengths(c))
        return {"bytes": 2 * keys * hkv * row + 2 * c["batch"] * c["hq"] * d * e, "flops": 4 * keys * c["hq"] * d}
    # rows in, and (append, rope_append) the pages read back as values
    stored = (-(-c["rows"] // c["page"]) + 3) * c["page"]
    back = stored * hkv * 2 * (row + d * e)
    if c["op"] == "append":
        return {"bytes": c["rows"] * (2 * hkv * (d * e + row) + 8) + back, "flops": 10 * c["rows"] * hkv * d}
    heads = c["hq"] + c["hkv"]
    return {"bytes": c["rows"] * (2 * c["hq"] * d * e + 2 * hkv * (d * e + row) + 16)
            + 8 * min(c["rows"], c["context"]) * c["rot"] + back,
            "flops": c["rows"] * (heads * ((4 * d if c["norm"] else 0) + 3 * c["rot"]) + 10 * hkv * d)}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _keys(g, *shape, dtype):
    """N(0, 1) with per-channel scales from U(0.5, 2): keys have outlier channels."""
    x = torch.randn(*shape, generator=g, device="cuda")
    return x.mul_(torch.rand(shape[-1], generator=g, device="cuda") * 1.5 + 0.5).to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _quantise(x, group):
    """Rows [..., d] as codes [..., d] (whole numbers of 0..15 in x's type) and bf16 scales [..., d / group, 2]."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15.0).clamp_min(1e-8).float().bfloat16()
    bias = lo.float().bfloat16()
    codes = torch.round((g - bias.to(x.dtype)) / scale.to(x.dtype)).clamp_(0, 15)
    return codes.flatten(-2), torch.cat([scale, bias], -1)


def _pack(codes, group):
    """Codes [..., d] two to a byte, the lower first: the n-th of 16 equal pieces of a row holds the n-th sixteenth
    of every group."""
    c = codes.to(torch.uint8).unflatten(-1, (-1, 16, group // 16)).transpose(-3, -2).flatten(-3)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _unpack(packed, group):
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    return c.unflatten(-1, (16, -1, group // 16)).transpose(-3, -2).flatten(-3)


def _values(codes, scales, group):
    """What rows of packed codes and their scales stand for, in fp32 (one rounding: the products are exact)."""
    q = _unpack(codes, group).float().unflatten(-1, (-1, group))
    return (q * scales[..., :1].float() + scales[..., 1:].float()).flatten(-2)


def _fill(g, c, pages, channels):
    """Pages of quantised N(0, 1) rows (with scales for each channel), a stretch of pages at a time."""
    hkv, page, d, group = c["hkv"], c["page"], c["d"], c["group"]
    codes = torch.empty(pages, hkv, page, d // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, hkv, page, d // group, 2, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 26) // (hkv * page * d))
    for at in range(0, pages, step):
        x = torch.randn(min(step, pages - at), hkv, page, d, generator=g, device="cuda")
        if channels is not None:
            x.mul_(channels)
        q, scales[at:at + step] = _quantise(x, group)
        codes[at:at + step] = _pack(q, group)
    return codes, scales


def _cache(g, c, pages):
    channels = torch.rand(c["d"], generator=g, device="cuda") * 1.5 + 0.5
    return (*_fill(g, c, pages, channels), *_fill(g, c, pages, None))


def _tables(lens, page, order):
    """Block table rows (unused entries -1) over the page order."""
    table, at = torch.full((len(lens), max(1, -(-max(lens) // page))), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        p = -(-n // page)
        table[b, :p] = order[at:at + p]
        at += p
    return table.cuda()


def prepare(c, seed):
    g, host = _gen(seed), torch.Generator().manual_seed(int(seed))
    dt = _DTYPES[c["dtype"]]
    if c["op"] == "logprobs":
        n, v = c["rows"], c["vocab"]
        x = torch.randn(n, v, generator=g, device="cuda").mul_(2.0)
        x.mul_(torch.rand(n, 1, generator=g, device="cuda") * 2 + 0.5)      # sure and unsure rows
        tokens = torch.randint(v, (n,), generator=g, device="cuda")
        if c["masked"]:
            ruled = torch.rand(n, v, generator=g, device="cuda") < c["masked"]
            ruled[torch.arange(n, device="cuda"), tokens] = False
            x.masked_fill_(ruled, -math.inf)
        if n > 8:
            tokens[torch.rand(n, generator=g, device="cuda") < 0.05] = -1   # rows without a next token
        return dict(c, logits=x.to(dt), tokens=tokens)
    page = c["page"]
    if c["op"] in ("attention", "read"):
        lens = _lengths(c) if c["op"] == "attention" else [c["tokens"]] * c["batch"]
        pages = sum(-(-n // page) for n in lens) + 2
        order = torch.randperm(pages, generator=host).to(torch.int32)
        s = dict(c, cache=_cache(g, c, pages), table=_tables(lens, page, order), lengths=_i32(lens))
        if c["op"] == "attention":
            s["q"] = _randn(g, c["batch"], c["hq"], 1, c["d"], dtype=dt)
        return s
    n, hkv, d = c["rows"], c["hkv"], c["d"]
    pages = -(-n // page) + 3
    # distinct slots, consecutive within a page as a plan gives them; the last few rows are padding
    order = torch.randperm(pages, generator=host)
    slots = (order[torch.arange(n) // page] * page + torch.arange(n) % page)
    if n > 4:
        slots[n - n // 16 - 1:] = -1
    # what earlier requests left in the pages, and all of them in order
    s = dict(c, cache=_cache(g, c, pages), slots=slots.cuda(), table=torch.arange(pages, dtype=torch.int32, device="cuda")[None])
    if c["op"] == "append":
        if c["heads_first"]:
            s["k"] = _keys(g, hkv, n, d, dtype=dt).transpose(0, 1)
            s["v"] = _randn(g, hkv, n, d, dtype=dt).transpose(0, 1)
        else:
            s["k"], s["v"] = _keys(g, n, hkv, d, dtype=dt), _randn(g, n, hkv, d, dtype=dt)
        return s
    hq = c["hq"]
    fused = _randn(g, n, (hq + 2 * hkv) * d, dtype=dt).view(n, hq + 2 * hkv, d)
    s["q"], s["k"], s["v"] = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    s["positions"] = torch.randint(c["context"], (n,), generator=g, device="cuda")
    inv = 1.0 / (1e6 ** (torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"]))
    ang = torch.arange(c["context"], device="cuda", dtype=torch.float64)[:, None] * torch.cat([inv, inv])[None]
    s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    s["qw"] = s["kw"] = None
    if c["norm"]:
        s["qw"] = (torch.rand(d, generator=g, device="cuda") + 0.5).to(dt)
        s["kw"] = (torch.rand(d, generator=g, device="cuda") + 0.5).to(dt)
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "rope_append": _plain_rope, "read": _plain_read, "attention": _plain_attention,
            "logprobs": _plain_logprobs}[s["op"]](s)


def _run_own(s):
    import butterfly_amd as bf

    if s["op"] == "logprobs":
        y = bf.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        return dict(logprobs=y.logprobs, entropy=y.entropy, top_logprobs=y.top_logprobs, top_tokens=y.top_tokens)
    pages = bf.Q4Pages(*s["cache"])
    if s["op"] == "attention":
        y = bf.paged_q4_attention(s["q"], pages, s["table"], s["lengths"], window=s["window"], return_stats=s["stats"])
        return dict(zip("olm", y)) if s["stats"] else dict(o=y)
    if s["op"] == "read":
        k, v = bf.paged_q4_read(pages, s["table"], s["tokens"], dtype=_DTYPES[s["dtype"]])
        return dict(k=k, v=v)
    out = {}
    if s["op"] == "append":
        bf.paged_q4_append(s["k"], s["v"], pages, s["slots"])
    else:
        out["q"] = bf.paged_q4_rope_append(s["q"], s["k"], s["v"], pages, s["slots"], s["positions"], s["cos"], s["sin"],
                                           q_weight=s["qw"], k_weight=s["kw"], eps=1e-6)
    out["k"], out["v"] = bf.paged_q4_read(pages, s["table"], s["table"].shape[1] * s["page"], dtype=_DTYPES[s["dtype"]])
    return out


def _put(s, codes, scales, rows):
    """Rows [N, Hkv, d] (64 bits: a value next to a border between two codes) into their slots; rows without one repeat
    the first row's write."""
    q, sc = _quantise(rows, s["group"])
    q = _pack(q, s["group"])
    live = s["slots"] >= 0
    at = torch.where(live, s["slots"], s["slots"][0])
    page, row = at // s["page"], at % s["page"]
    codes[page, :, row] = torch.where(live[:, None, None], q, q[:1])
    scales[page, :, row] = torch.where(live[:, None, None, None], sc, sc[:1])


def _dense(s, ids, codes, scales):
    """The pages ``ids`` [B, P] of every request as fp32 [B, Hkv, P page, d]."""
    x = _values(codes[ids], scales[ids], s["group"])
    return x.transpose(1, 2).flatten(2, 3)


def _plain_read(s, tokens=None):
    kc, ks, vc, vs = s["cache"]
    ids, dt, n = s["table"].long().clamp_min(0), _DTYPES[s["dtype"]], s["tokens"] if tokens is None else tokens
    return dict(k=_dense(s, ids, kc, ks)[:, :, :n].to(dt), v=_dense(s, ids, vc, vs)[:, :, :n].to(dt))


def _plain_append(s):
    kc, ks, vc, vs = s["cache"]
    _put(s, kc, ks, s["k"].double())
    _put(s, vc, vs, s["v"].double())
    return _plain_read(s, s["table"].shape[1] * s["page"])


def _plain_rope(s):
    kc, ks, vc, vs = s["cache"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    rot = cos.shape[-1]

    def turn(x, w):
        if w is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.to(x.dtype)
        y = x[..., :rot]
        half = torch.cat([-y[..., rot // 2:], y[..., :rot // 2]], -1)
        return torch.cat([y * cos + half * sin, x[..., rot:]], -1)

    q = turn(s["q"].float(), s["qw"]).to(s["q"].dtype)
    _put(s, kc, ks, turn(s["k"].double(), s["kw"]))
    _put(s, vc, vs, s["v"].double())
    return dict(q=q, **_plain_read(s, s["table"].shape[1] * s["page"]))


def _plain_attention(s):
    q, ids = s["q"], s["table"].long().clamp_min(0)
    kc, ks, vc, vs = s["cache"]
    b, hq, _, d = q.shape
    hkv = s["hkv"]
    k = _dense(s, ids, kc, ks)
    t, n = torch.arange(k.shape[2], device=q.device), s["lengths"].long()[:, None]
    seen = t < n
    if s["window"]:
        seen &= t >= n - s["window"]
    seen = seen[:, None, None]
    x = torch.matmul(q.float().view(b, hkv, hq // hkv, d), k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    del k
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    some = seen.any(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - m), 0.0)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, torch.where(seen.transpose(2, 3), _dense(s, ids, vc, vs), 0.0)) / l
    o = torch.where(some, o, 0.0).to(q.dtype).view(b, hq, 1, d)
    if not s["stats"]:
        return dict(o=o)
    m = torch.where(some, m, -1e30).view(b, hq, 1, 1)
    return dict(o=o, l=l.view(b, hq, 1, 1), m=m)


def _plain_logprobs(s):
    x, tok, v = s["logits"].float(), s["tokens"], s["vocab"]
    m = x.amax(-1, keepdim=True)
    z = x - m
    e = torch.exp(z)
    l = e.double().sum(-1)                              # (a long sum)
    log = torch.log(l)
    given = z.gather(1, tok.clamp(0, v - 1)[:, None])[:, 0].double() - log
    given = torch.where((tok >= 0) & (tok < v), given, math.nan).float()
    entropy = (log - torch.where(e > 0, e * z, 0.0).double().sum(-1) / l).float()
    # the largest of unique keys: the value's order, then the lower place
    bits = x.view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    order = (bits << 20) + (v - 1 - torch.arange(v, device=x.device))
    at = v - 1 - (torch.topk(order, s["top"], dim=-1).values & ((1 << 20) - 1))
    return dict(logprobs=given, entropy=entropy, top_logprobs=(z.gather(1, at).double() - log[:, None]).float(), top_tokens=at)


# --------------------------------------------------------------------------- 64 bits, by another route
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "logprobs":
        return _exact_logprobs(s)
    if c["op"] == "attention":
        return _exact_attention(s)
    k, v = (_exact_values(*s["cache"][i:i + 2], c["group"]) for i in (0, 2))
    q, tokens = None, c.get("tokens")
    if c["op"] != "read":
        rows = [s["k"].double(), s["v"].double()]
        if c["op"] == "rope_append":
            q, rows[0] = (_exact_rope(s[x].double(), s[w], s) for x, w in (("q", "qw"), ("k", "kw")))
        live = (s["slots"] >= 0).nonzero()[:, 0]
        at, tokens = s["slots"][live], s["table"].shape[1] * c["page"]
        k, v = (_exact_put(pages, _exact_nearest(r, c["group"])[live], at) for pages, r in zip((k, v), rows))
    ids = s["table"].long().clamp_min(0)
    k, v = (x[ids].transpose(1, 2).flatten(2, 3)[:, :, :tokens] for x in (k, v))
    return dict(k=k, v=v) if q is None else dict(q=q, k=k, v=v)


def _exact_values(codes, scales, group):
    """Byte by byte: element e of a row is the (e % group // (group / 16))-th piece's."""
    d, dev = 2 * codes.shape[-1], codes.device
    e = torch.arange(d, device=dev)
    per, n = group // 16, d // group
    at = (e % group) // per * (n * per) + e // group * per + e % per
    q = (codes[..., at // 2].long() >> (4 * (at % 2))) & 15
    sc = scales.double()[..., e // group, :]
    return q.double() * sc[..., 0] + sc[..., 1]


def _exact_nearest(x, group):
    """Each element's nearest of its group's 16 levels, the even one of two at the same distance."""
    g = x.view(*x.shape[:-1], -1, group)
    ends = g.sort(-1).values[..., [0, -1]]
    bias = ends[..., :1].float().to(torch.bfloat16).double()
    step = ((ends[..., 1:] - ends[..., :1]) / 15).clamp(min=1e-8).float().to(torch.bfloat16).double()
    below = ((g - bias) / step).floor().clamp(0, 15)
    rest = (g - bias) - below * step
    up = (rest > step / 2) | ((rest == step / 2) & (below % 2 == 1))
    return ((below + up).clamp(0, 15) * step + bias).view(x.shape)


def _exact_put(pages, rows, at):
    flat = pages.transpose(1, 2).reshape(-1, *rows.shape[1:]).clone()
    flat[at] = rows
    return flat.view(pages.shape[0], pages.shape[2], pages.shape[1], -1).transpose(1, 2)


def _exact_rope(x, w, s):
    if w is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
    half = s["rot"] // 2
    turn = torch.complex(s["cos"][:, :half].double(), s["sin"][:, :half].double())[s["positions"]][:, None]
    z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _exact_attention(s):
    b, hq, _, d = s["q"].shape
    hkv, page = s["hkv"], s["page"]
    kc, ks, vc, vs = s["cache"]
    o = torch.zeros(b, hq, 1, d, dtype=torch.float64, device="cuda")
    l, m = torch.zeros_like(o[..., :1]), torch.full_like(o[..., :1], -1e30)
    for i, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - s["window"]) if s["window"] else 0
        if n == lo:
            continue
        ids = s["table"][i, :-(-n // page)].long()
        for h in range(hkv):
            k, v = (_exact_values(x[ids, h], y[ids, h], s["group"]).reshape(-1, d)[lo:n] for x, y in ((kc, ks), (vc, vs)))
            rows = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            x = s["q"][i, rows, 0].double() @ k.t() / math.sqrt(d)
            m[i, rows, 0] = x.amax(-1, keepdim=True)
            p = (x - m[i, rows, 0]).exp()
            l[i, rows, 0] = p.sum(-1, keepdim=True)
            o[i, rows, 0] = p @ v / l[i, rows, 0]
    return dict(o=o, l=l, m=m) if s["stats"] else dict(o=o)


def _exact_logprobs(s):
    n, v = s["logits"].shape
    given, entropy, tops, ids = [], [], [], []
    for at in range(0, n, 256):
        x, tok = s["logits"][at:at + 256].double(), s["tokens"][at:at + 256]
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        entropy.append(-(logp.exp() * logp.clamp_min(-1e300)).sum(-1))
        given.append(torch.where(tok >= 0, logp.gather(1, tok.clamp_min(0)[:, None])[:, 0], math.nan))
        ranked = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["top"]]
        tops.append(logp.gather(1, ranked))
        ids.append(ranked)
    return dict(logprobs=torch.cat(given), entropy=torch.cat(entropy), top_logprobs=torch.cat(tops), top_tokens=torch.cat(ids))
