"""The 4-bit paged cache in plain torch operations and 64 bits, for tests (any device)."""
from __future__ import annotations

import math

import torch


def quantise(x: torch.Tensor, group: int):
    """Rows [..., d] -> codes [..., d] (int64), scale and bias [..., d / group] (float64 values of bf16)."""
    g = x.double().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    bias = lo.float().bfloat16()
    scale = ((hi - lo) / 15).clamp_min(1e-8).float().bfloat16()
    ok = torch.isfinite(g).all(-1) & torch.isfinite(bias) & torch.isfinite(scale)
    nan = torch.tensor(float("nan"), dtype=torch.float64, device=x.device)
    bias, scale = torch.where(ok, bias.double(), nan), torch.where(ok, scale.double(), nan)
    t = (g - bias[..., None]) / scale[..., None]
    codes = torch.where(ok[..., None], torch.round(t).clamp(0, 15), 0.0).long()
    return codes.flatten(-2), scale, bias


def place(d: int, group: int):
    """Where element e's code lies: its byte of the row and its shift in there."""
    per, groups = group // 16, d // group
    out = []
    for e in range(d):
        g, i = divmod(e, group)
        piece, within = divmod(i, per)
        n = (piece * groups + g) * per + within
        out.append((n // 2, 4 * (n % 2)))
    return out


def pack(codes: torch.Tensor, group: int) -> torch.Tensor:
    out = torch.zeros(*codes.shape[:-1], codes.shape[-1] // 2, dtype=torch.long, device=codes.device)
    for e, (byte, shift) in enumerate(place(codes.shape[-1], group)):
        out[..., byte] |= codes[..., e] << shift
    return out.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What packed codes [..., d / 2] and scales [..., d / group, 2] stand for, in 64 bits."""
    d, groups = 2 * codes.shape[-1], scales.shape[-2]
    at = place(d, d // groups)
    byte = torch.tensor([b for b, _ in at], device=codes.device)
    shift = torch.tensor([s for _, s in at], device=codes.device)
    q = (codes.long()[..., byte] >> shift) & 15
    sc = scales.double().repeat_interleave(d // groups, -2)
    return q.double() * sc[..., 0] + sc[..., 1]


def packed(x: torch.Tensor, group: int):
    """Rows [..., d] as packed codes and bf16 scales [..., d / group, 2]."""
    codes, scale, bias = quantise(x, group)
    return pack(codes, group), torch.stack([scale, bias], -1).bfloat16()


def rope(x, weight, cos, sin, positions, eps):
    """Norm and rotate-half RoPE of rows [N, H, d] in 64 bits; NaN for positions outside the tables."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    r = cos.shape[-1]
    inside = (positions >= 0) & (positions < cos.shape[0])
    at = positions.clamp(0, cos.shape[0] - 1)
    c, s = (torch.where(inside[:, None], t.double()[at], math.nan)[:, None] for t in (cos, sin))
    y = x[..., :r]
    y = y * c + torch.cat([-y[..., r // 2:], y[..., :r // 2]], -1) * s
    rest = torch.where(inside[:, None, None], x[..., r:], math.nan)
    return torch.cat([y, rest], -1)


def attention(q, kc, ks, vc, vs, table, lengths, *, scale=None, window=0):
    """(out, l, m) in 64 bits, and the bound of each row's weighted values max (31 scale + |bias|) of v."""
    b, hq, _, d = q.shape
    hkv, page = kc.shape[1], kc.shape[2]
    g = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    o = torch.zeros(b, hq, 1, d, dtype=torch.float64, device=q.device)
    l, m = torch.zeros_like(o[..., :1]), torch.full_like(o[..., :1], -1e30)
    for i, n in enumerate(lengths.tolist()):
        if n > table.shape[1] * page:
            o[i], l[i], m[i] = math.nan, math.nan, math.nan
            continue
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        ids = table[i, :-(-n // page)].long()
        for h in range(hkv):
            k, v = (values(c[ids, h], s[ids, h]).reshape(-1, d)[lo:n] for c, s in ((kc, ks), (vc, vs)))
            rows = slice(h * g, (h + 1) * g)
            x = q[i, rows, 0].double() @ k.t() * scale
            m[i, rows, 0] = x.amax(-1, keepdim=True)
            p = (x - m[i, rows, 0]).exp()
            l[i, rows, 0] = p.sum(-1, keepdim=True)
            o[i, rows, 0] = p @ v / l[i, rows, 0]
    return o, l, m


# --------------------------------------------------------------------------- in the place of the native ones
def append(k, v, pages, slots):
    size, group = pages.k_codes.shape[2], 2 * pages.k_codes.shape[3] // pages.k_scales.shape[3]
    for x, codes, scales in ((k, pages.k_codes, pages.k_scales), (v, pages.v_codes, pages.v_scales)):
        c, s = packed(x, group)
        for i, slot in enumerate(slots.tolist()):
            if slot >= 0:
                codes[slot // size, :, slot % size] = c[i]
                scales[slot // size, :, slot % size] = s[i]


def read(pages, table, tokens, *, dtype=torch.bfloat16):
    return tuple(values(c[table.long().clamp_min(0)], s[table.long().clamp_min(0)]).transpose(1, 2).flatten(2, 3)[:, :, :tokens]
                 .to(dtype) for c, s in ((pages.k_codes, pages.k_scales), (pages.v_codes, pages.v_scales)))


def paged_attention(q, pages, table, lengths, *, scale=None, window=0, return_stats=False):
    assert not window and not return_stats
    return attention(q, *pages, table, lengths, scale=scale)[0].to(q.dtype)


def install(monkeypatch):
    """Puts them in the place of the native ones behind ``PagedKVCache(..., quant_bits=4)``."""
    from butterfly_amd import paged_q4

    for name, f in (("paged_q4_append", append), ("paged_q4_read", read), ("paged_q4_attention", paged_attention)):
        monkeypatch.setattr(paged_q4, name, f)
