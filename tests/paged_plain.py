"""The paged operators in plain torch operations on the CPU, for tests of what calls them."""
from __future__ import annotations

import torch

from butterfly_amd.paged import PagedPlan


def plan(table, lengths, counts, free, state, *, page_size, num_rows, rows_each=0, in_place=False):
    assert in_place
    old, add = lengths.tolist(), counts.tolist()
    new = [max(0, n + c) for n, c in zip(old, add)]
    top, error = state.tolist()
    up = lambda n: -(-n // page_size)
    stack = free[:top].tolist() + [int(table[b, j]) for b, (a, n) in enumerate(zip(old, new))
                                   for j in range(up(n), up(a))][::-1]
    need = sum(max(0, up(n) - up(a)) for a, n in zip(old, new))
    if not error:
        error = (2 if any(up(n) > table.shape[1] for n in new) else 3 if rows_each and max(add) > rows_each
                 else 4 if need > len(stack) else 0)
    slots, positions, starts = [-1] * num_rows, [0] * num_rows, [0] * (len(old) + 1)
    if not error:
        for b, (a, n) in enumerate(zip(old, new)):
            for j in range(up(a), up(n)):
                table[b, j] = stack.pop()
            at = starts[b]
            for i, p in enumerate(range(a, n)):
                slots[at + i] = int(table[b, p // page_size]) * page_size + p % page_size
                positions[at + i] = p
            starts[b + 1] = at + (rows_each or max(0, add[b]))
        lengths.copy_(torch.tensor(new))
        free[:len(stack)] = torch.tensor(stack, dtype=torch.int32)
        top = len(stack)
    state.copy_(torch.tensor([top, error]))
    return PagedPlan(lengths, state, torch.tensor(starts, dtype=torch.int32), torch.tensor(slots), torch.tensor(positions))


def append(k, v, k_pages, v_pages, slots):
    assert k.shape == v.shape and k.shape[0] == slots.shape[0]
    size = k_pages.shape[2]
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            k_pages[s // size, :, s % size] = k[i]
            v_pages[s // size, :, s % size] = v[i]


def attention(q, k_pages, v_pages, table, lengths, *, scale=None, window=0, return_stats=False):
    assert not window and not return_stats and q.shape[2] == 1
    out = torch.zeros_like(q)
    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            continue
        ids = table[b, :-(-n // k_pages.shape[2])].long()
        k, v = (x[ids].transpose(0, 1).flatten(1, 2)[:, :n].double() for x in (k_pages, v_pages))
        g = q.shape[1] // k.shape[0]
        s = q[b].double() @ k.repeat_interleave(g, 0).transpose(1, 2) * (scale or q.shape[-1] ** -0.5)
        out[b] = (s.softmax(-1) @ v.repeat_interleave(g, 0)).to(q.dtype)
    return out


def install(monkeypatch):
    """Puts them in the place of the native ones behind ``PagedKVCache``."""
    from butterfly_amd import paged

    for name, f in (("paged_plan", plan), ("paged_append", append), ("paged_attention", attention)):
        monkeypatch.setattr(paged, name, f)
