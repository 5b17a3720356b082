"""GPU: the paged operators refuse what a native call would hide itself from."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import butterfly_amd as bf

pytestmark = pytest.mark.gpu


def _calls():
    """Each operator as a function of its floating tensors, and those."""
    pages = [torch.zeros(4, 1, 16, 64, device="cuda") for _ in range(2)]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    slots = torch.arange(2, device="cuda")
    rows = lambda h: torch.randn(2, h, 64, device="cuda")
    tab, w = torch.ones(4, 64, device="cuda"), torch.ones(64, device="cuda")
    return {
        "append": (lambda k, v, kp, vp: (bf.paged_append(k, v, kp, vp, slots), kp)[1], [rows(1), rows(1), *pages]),
        "rope_append": (lambda q, k, v, kp, vp, cos, sin, qw, kw: bf.paged_rope_append(
            q, k, v, kp, vp, slots, slots, cos, sin, q_weight=qw, k_weight=kw),
            [rows(2), rows(1), rows(1), *pages, tab, tab.clone(), w, w.clone()]),
        "attention": (lambda q, kp, vp: bf.paged_attention(q, kp, vp, i32(0, 1).view(2, 1), i32(2, 3)),
                      [rows(2).unsqueeze(2), *pages]),
    }


@pytest.mark.parametrize("name", ["append", "rope_append", "attention"])
def test_tangents_are_refused(name):
    call, tensors = _calls()[name]
    with torch.no_grad():
        want = call(*tensors)
        with forward_ad.dual_level():
            assert torch.equal(call(*tensors), want)           # none here
            for i, t in enumerate(tensors):
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(ValueError, match="tangents"):
                    call(*tensors[:i], dual, *tensors[i + 1:])
        assert torch.equal(call(*tensors), want)


@pytest.mark.parametrize("name", ["append", "rope_append", "attention"])
def test_traces_are_refused(name):
    call, tensors = _calls()[name]
    with torch.no_grad(), pytest.raises(ValueError, match="traced"):
        torch.jit.trace(call, tuple(tensors))


def test_a_traced_plan_is_refused():
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    free, state = i32(0, 1, 2), i32(3, 0)
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda n, c: tuple(bf.paged_plan(table, n, c, free, state, page_size=16, num_rows=2)),
                        (i32(0, 0), i32(1, 1)))
    assert state.tolist() == [3, 0] and free.tolist() == [0, 1, 2]
