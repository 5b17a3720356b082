"""The paged operators' argument checks, at the C ABI and in Python, without a GPU: every refusal comes
before any launch."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd import _native

I = 4096   # stands for an aligned device pointer: never followed, the calls below are refused first


def _pack(name, a, kw):
    """The packed argument struct with some members changed (None: a null pointer)."""
    a = {**a, **kw}
    return _native.PAGED_STRUCTS[name].pack(*[0 if x is None else x for x in a.values()])


PAGES = dict(kp=I, vp=I, pages=4, page=64, a=16384, b=8192, c=128, e=16384, f=8192, g=128)
ARGS = {
    "bfly_paged_plan": dict(table=I, requests=4, width=8, stride=8, lengths=I, counts=I, free=I, cap=32, state=I, page=64,
                            rows=4, each=0, lengths_out=I, state_out=I, starts=I, slots=I, positions=I, ws=I, ws_bytes=60),
    "bfly_paged_append": dict(k=I, v=I, dtype=1, rows=4, hkv=2, d=128, ks=256, kh=128, vs=256, vh=128, slots=I, **PAGES),
    "bfly_paged_rope_append": dict(q=I, k=I, v=I, dtype=1, rows=4, hq=4, hkv=2, d=128, qs=512, qh=128, ks=256, kh=128, vs=256,
                                   vh=128, qw=I, kw=I, eps=1e-6, cos=I, sin=I, table=16, rot=128, pos=I, slots=I, out=I,
                                   **PAGES),
    "bfly_paged_attention": dict(q=I, dtype=1, requests=4, hq=4, hkv=2, d=128, qr=512, qh=128, **PAGES, table=I, width=8,
                                 stride=8, lengths=I, window=0, scale=1.0, out=I, l=None, m=None, ws=I, ws_bytes=1 << 40),
}
_plan, _append, _rope, _attn = ARGS


INVALID, UNSUPPORTED = _native.ERR_INVALID, _native.ERR_UNSUPPORTED


@pytest.mark.parametrize("name,kw,rc,msg", [
    ("bfly_paged_plan", dict(page=48), INVALID, b"power of two"),
    ("bfly_paged_plan", dict(page=8), INVALID, b"power of two"),
    ("bfly_paged_plan", dict(page=2048), INVALID, b"power of two"),
    ("bfly_paged_plan", dict(stride=7), INVALID, b"overlap"),
    ("bfly_paged_plan", dict(requests=-1), INVALID, b"shape"),
    ("bfly_paged_plan", dict(rows=-1), INVALID, b"num_rows"),
    ("bfly_paged_plan", dict(rows=1 << 31), INVALID, b"2^31"),
    ("bfly_paged_plan", dict(cap=1 << 31), INVALID, b"2^31"),
    ("bfly_paged_plan", dict(ws_bytes=56), INVALID, b"workspace"),
    ("bfly_paged_plan", dict(each=2), INVALID, b"rows_each"),
    ("bfly_paged_plan", dict(each=-1), INVALID, b"rows_each"),
    ("bfly_paged_plan", dict(ws=None), INVALID, b"workspace"),
    ("bfly_paged_plan", dict(slots=None), INVALID, b"null"),
    ("bfly_paged_plan", dict(state=None), INVALID, b"null"),
    ("bfly_paged_append", dict(dtype=7), INVALID, b"dtype"),
    ("bfly_paged_append", dict(d=124), INVALID, b"16-byte"),
    ("bfly_paged_append", dict(page=24), INVALID, b"power of two"),
    ("bfly_paged_append", dict(pages=0), INVALID, b"num_pages"),
    ("bfly_paged_append", dict(c=132), INVALID, b"strides"),
    ("bfly_paged_append", dict(ks=-256), INVALID, b"strides"),
    ("bfly_paged_append", dict(k=I + 8), INVALID, b"aligned"),
    ("bfly_paged_append", dict(vp=None), INVALID, b"null"),
    ("bfly_paged_append", dict(c=1 << 30), INVALID, b"row stride"),
    ("bfly_paged_append", dict(hkv=0), INVALID, b"shape"),
    ("bfly_paged_rope_append", dict(d=96), UNSUPPORTED, b"head_dim"),
    ("bfly_paged_rope_append", dict(rot=24), INVALID, b"rotary_dim"),
    ("bfly_paged_rope_append", dict(rot=144), INVALID, b"rotary_dim"),
    ("bfly_paged_rope_append", dict(rot=0), INVALID, b"rotary_dim"),
    ("bfly_paged_rope_append", dict(table=0), INVALID, b"rows"),
    ("bfly_paged_rope_append", dict(qw=None), INVALID, b"neither"),
    ("bfly_paged_rope_append", dict(hq=3), INVALID, b"head counts"),
    ("bfly_paged_rope_append", dict(cos=I + 4), INVALID, b"aligned"),
    ("bfly_paged_rope_append", dict(pos=None), INVALID, b"null"),
    ("bfly_paged_rope_append", dict(rows=1 << 27), INVALID, b"too many"),
    ("bfly_paged_append", dict(rows=1 << 27), INVALID, b"too many"),
    ("bfly_paged_attention", dict(requests=65536), INVALID, b"65535"),
    ("bfly_paged_attention", dict(requests=65535, hq=512, hkv=512), INVALID, b"too many"),
    ("bfly_paged_attention", dict(ws_bytes=100, width=1000), INVALID, b"workspace"),
    ("bfly_paged_attention", dict(d=80), UNSUPPORTED, b"head_dim"),
    ("bfly_paged_attention", dict(hq=5), INVALID, b"head counts"),
    ("bfly_paged_attention", dict(window=-1), INVALID, b"window"),
    ("bfly_paged_attention", dict(l=I), INVALID, b"l and m"),
    ("bfly_paged_attention", dict(q=I + 2), INVALID, b"aligned"),
    ("bfly_paged_attention", dict(qh=4), INVALID, b"q strides"),
    ("bfly_paged_attention", dict(table=None), INVALID, b"null"),
    ("bfly_paged_attention", dict(page=100), INVALID, b"power of two"),
])
def test_c_abi_refuses_before_launch(name, kw, rc, msg):
    lib = _native.lib()
    assert set(kw) <= set(ARGS[name])
    assert getattr(lib, name)(_pack(name, ARGS[name], kw), None) == rc
    assert msg in lib.bfly_last_error()


def test_null_argument_structs_are_refused():
    lib = _native.lib()
    for name in ARGS:
        assert getattr(lib, name)(None, None) == INVALID and b"null" in lib.bfly_last_error()


def test_the_packed_formats_are_the_headers_structs():
    """Members of each struct in include/butterfly_amd_paged.h, in order: eight bytes each, doubles where the
    format has one."""
    text = (Path(__file__).resolve().parents[1] / "include" / "butterfly_amd_paged.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    structs = {}
    for name, body in re.findall(r"typedef struct (\w+) \{(.*?)\}", text, flags=re.S):
        kinds = []
        for decl in filter(None, (x.strip() for x in body.split(";"))):
            if decl.startswith("bfly_pages_t "):
                kinds += structs["bfly_pages"]
                continue
            assert "*" in decl or decl.startswith(("int64_t ", "double ")), decl
            kinds += ["d" if decl.startswith("double ") else "q"] * (decl.count(",") + 1)
        structs[name] = kinds
    for name, fmt in _native.PAGED_STRUCTS.items():
        kinds = structs[name + "_args"]
        assert fmt.size == 8 * len(kinds)
        values = [float(i) if k == "d" else i for i, k in enumerate(kinds)]
        assert list(fmt.unpack(fmt.pack(*values))) == values
        assert len(ARGS[name]) == len(kinds)


def test_nothing_to_do_returns_without_a_launch():
    lib = _native.lib()
    for name, kw in [(_append, dict(rows=0, k=None, v=None, slots=None)), (_rope, dict(rows=0, q=None)),
                     (_attn, dict(requests=0, q=None))]:
        assert getattr(lib, name)(_pack(name, ARGS[name], kw), None) == 0


def test_operators_refuse_cpu_tensors():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    pages = torch.zeros(4, 2, 16, 64)
    slots = torch.zeros(3, dtype=torch.int64)
    rows = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        bf.paged_plan(i32(2, 4), i32(2), i32(2), i32(4), i32(2), page_size=16, num_rows=2)
    with pytest.raises(ValueError, match="GPU"):
        bf.paged_append(rows, rows, pages, pages, slots)
    with pytest.raises(ValueError, match="GPU"):
        bf.paged_rope_append(rows, rows, rows, pages, pages, slots, slots, torch.zeros(4, 64), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="GPU"):
        bf.paged_attention(torch.zeros(2, 2, 1, 64), pages, pages, i32(2, 4), i32(2))
