"""The 4-bit paged operators' argument checks, at the C ABI and in Python, without a GPU: every refusal comes before any
launch; and the plain forms that the GPU tests compare with, by hand."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

import butterfly_amd as bf
from butterfly_amd import _native
from tests import q4_plain

I = 4096   # stands for an aligned device pointer: never followed, the calls below are refused first
INVALID, UNSUPPORTED = _native.ERR_INVALID, _native.ERR_UNSUPPORTED

PAGES = dict(kc=I, ks=I, vc=I, vs=I, pages=4, page=64, group=64, kcp=8192, kch=4096, kcr=64, ksp=1024, ksh=512, ksr=8,
             vcp=8192, vch=4096, vcr=64, vsp=1024, vsh=512, vsr=8)
ARGS = {
    "bfly_paged_q4_append": dict(k=I, v=I, dtype=1, rows=4, hkv=2, d=128, krs=256, khs=128, vrs=256, vhs=128, slots=I, **PAGES),
    "bfly_paged_q4_rope_append": dict(q=I, k=I, v=I, dtype=1, rows=4, hq=4, hkv=2, d=128, qs=512, qh=128, krs=256, khs=128,
                                      vrs=256, vhs=128, qw=I, kw=I, eps=1e-6, cos=I, sin=I, table=16, rot=128, pos=I, slots=I,
                                      out=I, **PAGES),
    "bfly_paged_q4_read": dict(dtype=1, requests=4, hkv=2, d=128, tokens=100, table=I, width=8, stride=8, k=I, v=I, **PAGES),
    "bfly_paged_q4_attention": dict(q=I, dtype=1, requests=4, hq=4, hkv=2, d=128, qr=512, qh=128, **PAGES, table=I, width=8,
                                    stride=8, lengths=I, window=0, scale=1.0, out=I, l=None, m=None, ws=I, ws_bytes=1 << 40),
}
_append, _rope, _read, _attn = ARGS


def _pack(name, kw):
    a = {**ARGS[name], **kw}
    return _native.PAGED_Q4_STRUCTS[name].pack(*[0 if x is None else x for x in a.values()])


@pytest.mark.parametrize("kw,rc,msg", [
    (dict(dtype=2), INVALID, b"dtype"),
    (dict(d=96), UNSUPPORTED, b"head_dim"),
    (dict(group=16), INVALID, b"group"),
    (dict(group=128), INVALID, b"group"),
    (dict(page=48), INVALID, b"power of two"),
    (dict(page=2048), INVALID, b"power of two"),
    (dict(pages=0), INVALID, b"num_pages"),
    (dict(pages=1 << 31), INVALID, b"num_pages"),
    (dict(kcr=68), INVALID, b"codes must be multiples of 16"),
    (dict(vch=-4096), INVALID, b"codes must be multiples of 16"),
    (dict(ksr=12), INVALID, b"scales must be multiples of 8"),
    (dict(vsp=1 << 48), INVALID, b"scales must be multiples of 8"),
    (dict(group=32, vsr=24), INVALID, b"scales must be multiples of 16"),
    (dict(kcr=1 << 30), INVALID, b"row stride"),
    (dict(vs=None), INVALID, b"null"),
    (dict(kc=I + 8), INVALID, b"aligned"),
    (dict(ks=I + 8), INVALID, b"aligned"),
])
@pytest.mark.parametrize("name", list(ARGS))
def test_c_abi_refuses_pages(name, kw, rc, msg):
    lib = _native.lib()
    assert getattr(lib, name)(_pack(name, kw), None) == rc
    assert msg in lib.bfly_last_error(), lib.bfly_last_error()


@pytest.mark.parametrize("name,kw,rc,msg", [
    (_append, dict(rows=-1), INVALID, b"shape"),
    (_append, dict(hkv=0), INVALID, b"shape"),
    (_append, dict(krs=-256), INVALID, b"strides"),
    (_append, dict(krs=260), INVALID, b"strides"),
    (_append, dict(k=I + 8), INVALID, b"aligned"),
    (_append, dict(slots=None), INVALID, b"null"),
    (_append, dict(rows=1 << 29), INVALID, b"too many"),
    (_append, dict(rows=1 << 27, d=256, ksr=16, vsr=16), INVALID, b"too many"),
    (_rope, dict(rot=24), INVALID, b"rotary_dim"),
    (_rope, dict(rot=144), INVALID, b"rotary_dim"),
    (_rope, dict(table=0), INVALID, b"rows"),
    (_rope, dict(kw=None), INVALID, b"neither"),
    (_rope, dict(hq=3), INVALID, b"head counts"),
    (_rope, dict(qh=100), INVALID, b"strides"),
    (_rope, dict(sin=I + 4), INVALID, b"aligned"),
    (_rope, dict(pos=None), INVALID, b"null"),
    (_rope, dict(rows=1 << 27), INVALID, b"too many"),
    (_read, dict(tokens=513), INVALID, b"beyond"),
    (_read, dict(tokens=-1), INVALID, b"beyond"),
    (_read, dict(requests=(1 << 24) + 1), INVALID, b"shape"),
    (_read, dict(requests=1 << 24, tokens=512), INVALID, b"too many"),
    (_read, dict(k=None), INVALID, b"null"),
    (_read, dict(table=None), INVALID, b"null"),
    (_attn, dict(requests=65536), INVALID, b"65535"),
    (_attn, dict(requests=65535, hq=512, hkv=512), INVALID, b"too many"),
    (_attn, dict(requests=1, hq=1 << 20, hkv=1 << 20), INVALID, b"too many heads"),
    (_attn, dict(ws_bytes=100, width=1000), INVALID, b"workspace"),
    (_attn, dict(ws=None, width=1000), INVALID, b"workspace"),
    (_attn, dict(hq=5), INVALID, b"head counts"),
    (_attn, dict(window=-1), INVALID, b"window"),
    (_attn, dict(window=1 << 31), INVALID, b"window"),
    (_attn, dict(m=I), INVALID, b"l and m"),
    (_attn, dict(q=I + 2), INVALID, b"aligned"),
    (_attn, dict(qh=4), INVALID, b"q strides"),
    (_attn, dict(table=None), INVALID, b"null"),
    (_attn, dict(width=-1), INVALID, b"table"),
])
def test_c_abi_refuses_before_launch(name, kw, rc, msg):
    lib = _native.lib()
    assert set(kw) <= set(ARGS[name])
    assert getattr(lib, name)(_pack(name, kw), None) == rc
    assert msg in lib.bfly_last_error(), lib.bfly_last_error()


def test_null_structs_and_nothing_to_do():
    lib = _native.lib()
    for name in ARGS:
        assert getattr(lib, name)(None, None) == INVALID and b"null" in lib.bfly_last_error()
    for name, kw in [(_append, dict(rows=0, k=None, slots=None)), (_rope, dict(rows=0, q=None)),
                     (_read, dict(requests=0, k=None)), (_read, dict(tokens=0, k=None)), (_attn, dict(requests=0, q=None))]:
        assert getattr(lib, name)(_pack(name, kw), None) == 0


def test_the_packed_formats_are_the_headers_structs():
    text = (Path(__file__).resolve().parents[1] / "include" / "butterfly_amd_paged_q4.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    structs = {}
    for name, body in re.findall(r"typedef struct (\w+) \{(.*?)\}", text, flags=re.S):
        kinds = []
        for decl in filter(None, (x.strip() for x in body.split(";"))):
            if decl.startswith("bfly_q4_pages_t "):
                kinds += structs["bfly_q4_pages"]
                continue
            assert "*" in decl or decl.startswith(("int64_t ", "double ")), decl
            kinds += ["d" if decl.startswith("double ") else "q"] * (decl.count(",") + 1)
        structs[name] = kinds
    assert set(_native.PAGED_Q4_STRUCTS) == set(ARGS)
    for name, fmt in _native.PAGED_Q4_STRUCTS.items():
        kinds = structs[name + "_args"]
        assert fmt.size == 8 * len(kinds) and len(ARGS[name]) == len(kinds)
        values = [float(i) if k == "d" else i for i, k in enumerate(kinds)]
        assert list(fmt.unpack(fmt.pack(*values))) == values


def test_workspace_only_where_requests_can_be_split():
    need = _native.lib().bfly_paged_q4_attention_workspace_bytes
    assert need(1, 1, 8, 2, 128, 1, 128, 0) == 0 and need(1, 0, 8, 2, 128, 1000, 128, 0) == 0 and need(0, 1, 8, 3, 128, 1000, 128, 0) == 0
    big = need(1, 1, 8, 2, 128, 1000, 128, 0)
    assert big > 0 and need(1, 1, 8, 2, 128, 1000, 128, 100) == 0
    assert need(0, 1, 64, 2, 256, 1000, 128, 0) > big


def test_operators_refuse_cpu_tensors():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    pages = bf.empty_q4_pages(4, 2, 16, 64, device="cpu")
    slots = torch.zeros(3, dtype=torch.int64)
    rows = torch.zeros(3, 2, 64)
    for f in (lambda: bf.paged_q4_append(rows, rows, pages, slots),
              lambda: bf.paged_q4_rope_append(rows, rows, rows, pages, slots, slots, torch.zeros(4, 64), torch.zeros(4, 64)),
              lambda: bf.paged_q4_read(pages, i32(2, 4), 3),
              lambda: bf.paged_q4_attention(torch.zeros(2, 2, 1, 64), pages, i32(2, 4), i32(2))):
        with pytest.raises(ValueError, match="GPU"):
            f()


def test_the_layout_by_hand():
    """d 128 in groups of 64: piece n is two bytes of group 0 (codes 4n..4n + 3), then two of group 1."""
    codes = torch.arange(128) % 16
    row = q4_plain.pack(codes[None], 64)[0]
    assert row.shape == (64,)
    assert row[4 * 3] == (codes[12] | codes[13] << 4) and row[4 * 3 + 1] == (codes[14] | codes[15] << 4)
    assert row[4 * 3 + 2] == (codes[64 + 12] | codes[64 + 13] << 4)
    row = q4_plain.pack(codes[None], 32)[0]            # four groups: a byte (codes 2n, 2n + 1) of each
    assert [int(x) for x in row[4 * 5:4 * 5 + 4]] == [int(codes[32 * g + 10] | codes[32 * g + 11] << 4) for g in range(4)]
    assert q4_plain.place(64, 64) == [(e // 2, 4 * (e % 2)) for e in range(64)]
    x = torch.randn(3, 256)
    for group in (32, 64):
        c, s = q4_plain.packed(x, group)
        step = s[..., 0].double().repeat_interleave(group, -1)
        lo = x.double().unflatten(-1, (-1, group)).amin(-1).abs().repeat_interleave(group, -1)
        # half a step, and where the roundings of scale (15 times) and bias hold the last code within 15
        assert bool(((q4_plain.values(c, s) - x.double()).abs() <= 0.5 * step + 2.0 ** -8 * (15 * step + lo)).all())
    c, s, b = q4_plain.quantise(torch.tensor([[0.0] * 16 + [15.0] * 16 + [0.5, 1.5, 2.5, 14.5] * 8] ).repeat(1, 1), 64)
    assert s.item() == 1.0 and b.item() == 0.0 and c[0, 32:36].tolist() == [0, 2, 2, 14]
