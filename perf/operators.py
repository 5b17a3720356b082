"""The paged serving operators as cases that can be timed and compared.

Requests that are served together keep their keys and values in pages of ``page`` rows, [pages, kv heads,
page, d], which a block table assigns to them.  Four operators (``op``):

* ``plan``: one step's bookkeeping from the requests' lengths: pages taken from and given back to a free
  list, the block table, and each new row's slot (page * page rows + row) and position.
* ``append``: rows of keys and values into their slots.
* ``rope_append``: the same for a decoder's projection rows, with the q/k norm and RoPE on the way.
* ``attention``: one new token of every request over its pages.

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
        # the smallest call: a decode step's bookkeeping for a handful of requests
        dict(name="plan_step_b8", op="plan", kind="step", batch=8, context=5000, page=128, ragged=1),
        # a large serving batch: most requests grow by a token, some stop, some idle
        dict(name="plan_mixed_b256", op="plan", kind="mixed", batch=256, context=8192, page=16, ragged=2),
        # prompts that arrive together: one slot for each of some 100k tokens
        dict(name="plan_prompts_b64", op="plan", kind="prompts", batch=64, context=4096, page=64, ragged=3),
        # a ragged prompt's keys and values, heads first as the prefill leaves them
        dict(name="append_prompt", op="append", dtype="bf16", rows=10007, hkv=4, d=128, page=128, heads_first=True),
        # a step's rows of an fp32 layer
        dict(name="append_fp32_step", op="append", dtype="fp32", rows=8, hkv=2, d=128, page=64, heads_first=False),
        # a decode step of 32 requests: columns of one fused projection row each
        dict(name="rope_step_b32", op="rope_append", dtype="bf16", rows=32, hq=16, hkv=4, d=128, rot=128, page=128,
             context=32768, norm=True),
        # prompts through wide heads, a quarter of each rotated
        dict(name="rope_prompt", op="rope_append", dtype="bf16", rows=16411, hq=16, hkv=4, d=256, rot=64, page=128,
             context=32768, norm=True),
        # short requests in small pages, an empty one among them: latency
        dict(name="attn_short_b8", op="attention", dtype="bf16", batch=8, hq=8, hkv=2, d=64, context=300, page=16,
             window=0, ragged=4, stats=False),
        # one sequence of the 4-bit decoder's benchmark after its 32k-token prompt
        dict(name="attn_32k_b1", op="attention", dtype="bf16", batch=1, hq=16, hkv=4, d=128, context=32768, page=128,
             window=0, ragged=0, stats=False),
        # the batched decode benchmark's heads and contexts, lengths of a mixed load
        dict(name="attn_131k_b32", op="attention", dtype="bf16", batch=32, hq=8, hkv=2, d=128, context=131072, page=128,
             window=0, ragged=5, stats=False),
        # the long-context layer: wide heads, one sequence, with the stream statistics
        dict(name="attn_262k_d256", op="attention", dtype="bf16", batch=1, hq=16, hkv=4, d=256, context=262144, page=256,
             window=0, ragged=0, stats=True),
        # the reference check's layer in fp32, a small ragged batch
        dict(name="attn_fp32_b4", op="attention", dtype="fp32", batch=4, hq=8, hkv=2, d=128, context=4096, page=64,
             window=0, ragged=6, stats=True),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "rope_append", "rope_append", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128, 256])
    ragged = rng.randint(1, 1 << 30)
    if op == "plan":
        kind = rng.choice(["step", "mixed", "prompts"])
        batch = _log(rng, 1, 64 if kind == "prompts" else 1024)
        return dict(op=op, kind=kind, batch=batch, context=_log(rng, 16, 8192), page=page, ragged=ragged)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    hkv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    if op == "append":
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 16384), hkv=hkv, d=d, page=page, heads_first=rng.random() < 0.5)
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    if op == "rope_append":
        most = 16411 * 24 * 256 // ((hq + 2 * hkv) * d)
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(16384, most)), hq=hq, hkv=hkv, d=d,
                    rot=rng.choice([d, d, d // 2, d // 4]), page=page, context=_log(rng, 64, 131072),
                    norm=rng.random() < 0.75)
    size = 2 if dtype == "bf16" else 4
    batch = _log(rng, 1, 64)
    # the pages take at most a gigabyte (the largest listed case has more)
    most = (1 << 30) // (2 * batch * hkv * d * size)
    return dict(op=op, dtype=dtype, batch=batch, hq=hq, hkv=hkv, d=d, context=_log(rng, 1, max(1, min(131072, most))),
                page=page, window=rng.choice([0, 0, rng.randint(1, 5000)]), ragged=rng.choice([0, ragged, ragged]),
                stats=rng.random() < 0.5)


def _lengths(c):
    """The requests' lengths: every one the context, or (ragged) from a mixed load with empty places."""
    if not c["ragged"]:
        return [c["context"]] * c["batch"]
    r = random.Random(c["ragged"])
    lens = [0 if r.random() < 0.08 else _log(r, max(1, c["context"] // 32), c["context"]) for _ in range(c["batch"])]
    lens[r.randrange(len(lens))] = c["context"]
    return lens


def _counts(c, lens):
    """How many rows each request gains (or gives back) in the step."""
    r = random.Random(c["ragged"] + 1)
    if c["kind"] == "step":
        return [1 if r.random() < 0.9 else 0 for _ in lens]
    if c["kind"] == "prompts":
        return [_log(r, max(1, c["context"] // 16), c["context"]) if r.random() < 0.9 else 0 for _ in lens]
    out = []
    for n in lens:
        x = r.random()
        # grows by a token; idle; leaves; takes a few drafted tokens back; starts with a short prompt
        out.append(1 if x < 0.7 else 0 if x < 0.8 else -n if x < 0.88 else -r.randint(1, 8) if x < 0.94 else r.randint(2, 64))
    return out


def work(c):
    if c["op"] == "plan":
        lens = [0] * c["batch"] if c["kind"] == "prompts" else _lengths(c)
        counts = _counts(c, lens)
        moved = sum(abs(-(-max(0, n + m) // c["page"]) - -(-n // c["page"])) for n, m in zip(lens, counts))
        # lengths, counts, new lengths, row starts; each page id moved; slot and position of each row
        return {"bytes": 16 * c["batch"] + 8 * moved + 16 * sum(max(0, m) for m in counts), "flops": 0}
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "append":
        return {"bytes": c["rows"] * (4 * c["hkv"] * c["d"] * e + 8), "flops": 0}
    if c["op"] == "rope_append":
        heads = c["hq"] + c["hkv"]
        return {"bytes": c["rows"] * (2 * (heads + c["hkv"]) * c["d"] * e + 16) + 8 * min(c["rows"], c["context"]) * c["rot"],
                "flops": c["rows"] * heads * ((4 * c["d"] if c["norm"] else 0) + 3 * c["rot"])}
    w = c["window"]
    keys = sum(min(n, w) if w else n for n in _lengths(c))
    return {"bytes": 2 * keys * c["hkv"] * c["d"] * e + 2 * c["batch"] * c["hq"] * c["d"] * e,
            "flops": 4 * keys * c["hq"] * c["d"]}


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


def _tables(lens, page, width, order):
    """Block table rows (unused entries -1) over the page order, and how many pages they take."""
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        p = -(-n // page)
        table[b, :p] = order[at:at + p]
        at += p
    return table, at


def prepare(c, seed):
    g, page = _gen(seed), c.get("page")
    host = torch.Generator().manual_seed(int(seed))
    if c["op"] == "plan":
        lens = [0] * c["batch"] if c["kind"] == "prompts" else _lengths(c)
        counts = _counts(c, lens)
        width = -(-max(max(0, n + m) for n, m in zip(lens, counts)) // page) + 1
        width = max(width, max(-(-n // page) for n in lens))
        pages = sum(-(-max(n, n + m, 0) // page) for n, m in zip(lens, counts)) + 8
        order = torch.randperm(pages, generator=host).to(torch.int32)
        table, at = _tables(lens, page, width, order)
        free = torch.cat([order[at:], torch.full((at,), -1, dtype=torch.int32)])
        rows = sum(max(0, m) for m in counts)
        rows += rows // 16 + 1                  # a step's rows are padded to a fixed number
        return dict(c, table=table.cuda(), free=free.cuda(), lengths=_i32(lens), counts=_i32(counts), rows=rows,
                    state=_i32([pages - at, 0]))
    dt = _DTYPES[c["dtype"]]
    if c["op"] == "attention":
        lens = _lengths(c)
        width = max(1, -(-max(lens) // page))
        pages = sum(-(-n // page) for n in lens) + 2
        order = torch.randperm(pages, generator=host).to(torch.int32)
        table, _ = _tables(lens, page, width, order)
        kp = torch.empty(pages, c["hkv"], page, c["d"], dtype=dt, device="cuda")
        vp = torch.empty_like(kp)
        step = max(1, (1 << 28) // (c["hkv"] * page * c["d"]))
        scale = torch.rand(c["d"], generator=g, device="cuda") * 1.5 + 0.5
        for at in range(0, pages, step):
            kp[at:at + step] = torch.randn(kp[at:at + step].shape, generator=g, device="cuda").mul_(scale)
            vp[at:at + step] = torch.randn(vp[at:at + step].shape, generator=g, device="cuda")
        q = _randn(g, c["batch"], c["hq"], 1, c["d"], dtype=dt)
        return dict(c, q=q, kp=kp, vp=vp, table=table.cuda(), lengths=_i32(lens))
    n, hkv, d = c["rows"], c["hkv"], c["d"]
    pages = -(-n // page) + 3
    kp = _randn(g, pages, hkv, page, d, dtype=dt)           # what earlier requests left there
    vp = _randn(g, pages, hkv, page, d, dtype=dt)
    # distinct slots, consecutive within a page as a plan gives them; the last few rows are padding
    order = torch.randperm(pages, generator=host)
    slots = (order[torch.arange(n) // page] * page + torch.arange(n) % page)
    if n > 4:
        slots[n - n // 16 - 1:] = -1
    s = dict(c, kp=kp, vp=vp, slots=slots.cuda())
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
    return {"plan": _plain_plan, "append": _plain_append, "rope_append": _plain_rope, "attention": _plain_attention}[s["op"]](s)


def _run_own(s):
    import butterfly_amd as bf

    if s["op"] == "plan":
        p = bf.paged_plan(s["table"], s["lengths"], s["counts"], s["free"], s["state"], page_size=s["page"],
                          num_rows=s["rows"])
        return dict(table=s["table"], free=s["free"], lengths=p.lengths, state=p.state, starts=p.starts, slots=p.slots,
                    positions=p.positions)
    if s["op"] == "append":
        bf.paged_append(s["k"], s["v"], s["kp"], s["vp"], s["slots"])
        return dict(k_pages=s["kp"], v_pages=s["vp"])
    if s["op"] == "rope_append":
        q = bf.paged_rope_append(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["slots"], s["positions"], s["cos"], s["sin"],
                                 q_weight=s["qw"], k_weight=s["kw"], eps=1e-6)
        return dict(q=q, k_pages=s["kp"], v_pages=s["vp"])
    y = bf.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lengths"], window=s["window"],
                           return_stats=s["stats"])
    return dict(zip("olm", y)) if s["stats"] else dict(o=y)


def _plain_plan(s):
    page, n, dev = s["page"], s["rows"], s["table"].device
    table, free, state = s["table"], s["free"], s["state"].long()
    b, width = table.shape
    old, counts = s["lengths"].long(), s["counts"].long()
    new = (old + counts).clamp_min(0)
    pold, pnew = (old + page - 1) // page, (new + page - 1) // page
    give, take = (pold - pnew).clamp_min(0), (pnew - pold).clamp_min(0)
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), counts.clamp_min(0).cumsum(0)])
    top = state[0] + give.sum()
    left = top - take.sum()
    error = torch.where(state[0] < 0, 5, 0) + torch.where(state[0] > free.numel(), 5, 0)
    error = torch.where(top > free.numel(), 5, error)
    error = torch.where(left < 0, 4, error)
    error = torch.where(starts[-1] > n, 3, error)
    error = torch.where((new > width * page).any(), 2, error)
    error = torch.where(((old < 0) | (old > width * page)).any(), 1, error)
    error = torch.where(state[1] != 0, state[1], error)
    ok = error == 0
    j = torch.arange(width, device=dev)[None]
    # the pages given back go on top of the free list, the first of them topmost; then pages are taken from the top
    to = top - 1 - ((give.cumsum(0) - give)[:, None] + j - pnew[:, None])
    mask = (j >= pnew[:, None]) & (j < pold[:, None]) & ok
    spare = torch.cat([free, free.new_zeros(1)])
    spare.scatter_(0, torch.where(mask, to, free.numel()).reshape(-1), table.reshape(-1))
    free.copy_(spare[:-1])
    at = top - 1 - ((take.cumsum(0) - take)[:, None] + j - pold[:, None])
    mask = (j >= pold[:, None]) & (j < pnew[:, None]) & ok
    table.copy_(torch.where(mask, free[torch.where(mask, at, 0)], table))
    i = torch.arange(n, device=dev)
    r = torch.searchsorted(starts[1:], i, right=True).clamp_max(b - 1)
    real = (i < starts[-1]) & ok
    pos = torch.where(real, old[r] + i - starts[r], 0)
    slots = torch.where(real, table[r, pos // page].long() * page + pos % page, -1)
    return dict(table=table, free=free, lengths=torch.where(ok, new, old).int(),
                state=torch.stack([torch.where(ok, left, state[0]), error]).int(),
                starts=torch.where(ok, starts, 0).int(), slots=slots, positions=pos)


def _put(pages, rows, slots):
    """rows [N, Hkv, d] into their slots; rows without one repeat the first row's write."""
    page = pages.shape[2]
    live = slots >= 0
    at = torch.where(live, slots, slots[0])
    pages[at // page, :, at % page] = torch.where(live[:, None, None], rows, rows[:1])


def _plain_append(s):
    _put(s["kp"], s["k"], s["slots"])
    _put(s["vp"], s["v"], s["slots"])
    return dict(k_pages=s["kp"], v_pages=s["vp"])


def _plain_rope(s):
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    rot = cos.shape[-1]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.float()
        y = x[..., :rot]
        half = torch.cat([-y[..., rot // 2:], y[..., :rot // 2]], -1)
        return torch.cat([y * cos + half * sin, x[..., rot:]], -1).to(s["q"].dtype)

    q = turn(s["q"], s["qw"])
    _put(s["kp"], turn(s["k"], s["kw"]), s["slots"])
    _put(s["vp"], s["v"], s["slots"])
    return dict(q=q, k_pages=s["kp"], v_pages=s["vp"])


def _plain_attention(s):
    q, table = s["q"], s["table"].long()
    b, hq, _, d = q.shape
    hkv = s["kp"].shape[1]
    ids = table.clamp_min(0)
    # [B, pages, Hkv, page, d] -> [B, Hkv, T, d]
    k = s["kp"][ids].transpose(1, 2).reshape(b, hkv, -1, d).float()
    v = s["vp"][ids].transpose(1, 2).reshape(b, hkv, -1, d).float()
    t, n = torch.arange(k.shape[2], device=q.device), s["lengths"].long()[:, None]
    seen = t < n
    if s["window"]:
        seen &= t >= n - s["window"]
    seen = seen[:, None, None]
    x = torch.matmul(q.float().view(b, hkv, hq // hkv, d), k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    some = seen.any(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - m), 0.0)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, torch.where(seen.transpose(2, 3), v, 0.0)) / l
    o = torch.where(some, o, 0.0).to(q.dtype).view(b, hq, 1, d)
    if not s["stats"]:
        return dict(o=o)
    m = torch.where(some, m, -1e30).view(b, hq, 1, 1)
    return dict(o=o, l=l.view(b, hq, 1, 1), m=m)


# --------------------------------------------------------------------------- 64 bits, by another route
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "plan":
        return _exact_plan(s)
    if c["op"] == "attention":
        return _exact_attention(s)
    kp, vp = s["kp"].double(), s["vp"].double()
    k, v, q = s["k"].double(), s["v"].double(), None
    if c["op"] == "rope_append":
        q, k = (_exact_rope(s[x].double(), s[w], s) for x, w in (("q", "qw"), ("k", "kw")))
    live = (s["slots"] >= 0).nonzero()[:, 0]
    at = s["slots"][live]
    for pages, rows in ((kp, k), (vp, v)):
        flat = pages.transpose(1, 2).reshape(-1, *rows.shape[1:]).clone()
        flat[at] = rows[live]
        pages.copy_(flat.view(pages.shape[0], pages.shape[2], pages.shape[1], -1).transpose(1, 2))
    return dict(k_pages=kp, v_pages=vp) if q is None else dict(q=q, k_pages=kp, v_pages=vp)


def _exact_rope(x, w, s):
    if w is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
    half = s["rot"] // 2
    turn = torch.complex(s["cos"][:, :half].double(), s["sin"][:, :half].double())[s["positions"]][:, None]
    z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _exact_plan(s):
    page, table, free = s["page"], s["table"].tolist(), s["free"].tolist()
    top, err = s["state"].tolist()
    old, counts = s["lengths"].tolist(), s["counts"].tolist()
    new = [max(0, a + n) for a, n in zip(old, counts)]
    use = [(-(-a // page), -(-n // page)) for a, n in zip(old, new)]
    given = [table[b][j] for b, (a, n) in enumerate(use) for j in range(n, a)]
    stack = free[:top] + given[::-1]
    free[top:len(stack)] = stack[top:]
    for b, (a, n) in enumerate(use):
        for j in range(a, n):
            table[b][j] = stack.pop()
    slots, positions, starts = [], [], [0]
    for b, (a, n) in enumerate(zip(old, counts)):
        for p in range(a, a + n):
            slots.append(table[b][p // page] * page + p % page)
            positions.append(p)
        starts.append(len(slots))
    pad = s["rows"] - len(slots)
    out = dict(table=table, free=free, lengths=new, state=[len(stack), err], starts=starts, slots=slots + [-1] * pad,
               positions=positions + [0] * pad)
    return {k: torch.tensor(v, dtype=torch.long) for k, v in out.items()}


def _exact_attention(s):
    b, hq, _, d = s["q"].shape
    hkv, page = s["kp"].shape[1:3]
    o = torch.zeros(b, hq, 1, d, dtype=torch.float64, device="cuda")
    l, m = torch.zeros_like(o[..., :1]), torch.full_like(o[..., :1], -1e30)
    for i, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - s["window"]) if s["window"] else 0
        if n == lo:
            continue
        ids = s["table"][i, :-(-n // page)].long()
        for h in range(hkv):
            k, v = (x[ids, h].reshape(-1, d)[lo:n].double() for x in (s["kp"], s["vp"]))
            rows = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            x = s["q"][i, rows, 0].double() @ k.t() / math.sqrt(d)
            m[i, rows, 0] = x.amax(-1, keepdim=True)
            p = (x - m[i, rows, 0]).exp()
            l[i, rows, 0] = p.sum(-1, keepdim=True)
            o[i, rows, 0] = p @ v / l[i, rows, 0]
    return dict(o=o, l=l, m=m) if s["stats"] else dict(o=o)
