"""Host-side checks of the paged-cache entry points (no GPU): the pages struct and the refusals that come
before any CUDA call."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from sisa_b200 import _lib


def test_pages_struct_matches_the_c_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not found")
    root = Path(__file__).resolve().parents[1]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "sisa_b200.h"', 'int main(void) {',
             'printf("size %zu\\n", sizeof(sisa_pages));']
    lines += [f'printf("{f} %zu\\n", offsetof(sisa_pages, {f}));' for f, _ in _lib.Pages._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run([gcc, "-I", str(root / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                                              text=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(_lib.Pages)
    for f, _ in _lib.Pages._fields_:
        assert int(got[f]) == getattr(_lib.Pages, f).offset, f


A = 0x10000          # a fake 16-byte aligned address: no call here reaches the device


def pages(**kw):
    H, S = 2, 64
    d = dict(k=A, v=A, b=A, g=A, f=A, weight=A, token=A, k_sp=64 * S * H, k_sh=64 * S, v_sp=64 * S * H, v_sh=64 * S,
             b_sp=32 * S * H, b_sh=32 * S, s_sp=S * H, s_sh=S, n_pages=8, page_size=S)
    d.update(kw)
    return _lib.Pages(**d)


def attn(pg, **kw):
    a = dict(q=_lib.View4(A, 128, 64, 64), c=_lib.View4(A, 64, 32, 32), gq=A, fq=A, table=A, tsb=4, mp=4, lengths=A, lam=A,
             B=3, H=2, dtype=_lib.BF16, y=_lib.View4(A, 128, 64, 64), lse=None, wo=None, ws=A)
    a.update(kw)
    return _lib.load().sisa_paged_attn(_lib.vref(a["q"]), _lib.vref(a["c"]), a["gq"], a["fq"], ctypes.byref(pg), a["table"],
                                       a["tsb"], a["mp"], a["lengths"], a["lam"], a["B"], a["H"], a["dtype"],
                                       _lib.vref(a["y"]), a["lse"], a["wo"], a["ws"], None, None)


def test_pages_and_attention_refusals():
    V, T, AL = _lib.ERR_VALUE, _lib.ERR_TYPE, _lib.ERR_ALIGN
    for kw, rc in ((dict(page_size=48), V), (dict(page_size=8), V), (dict(page_size=512), V), (dict(n_pages=0), V), (dict(k=None), V),
                   (dict(g=None), V), (dict(k=A + 8), AL), (dict(weight=A + 4), AL), (dict(k_sp=68), AL), (dict(k_sh=32 * 64), V),
                   (dict(b_sh=16 * 64), V), (dict(s_sh=32), V), (dict(s_sp=130), AL), (dict(f=None), V), (dict(v_sp=-8192), V)):
        assert attn(pages(**kw)) == rc, kw
    for kw, rc in ((dict(dtype=_lib.F32), T), (dict(B=0), V), (dict(B=65536), V), (dict(table=None), V), (dict(tsb=3), V),
                   (dict(mp=0), V), (dict(lengths=None), V), (dict(ws=None, mp=16, tsb=16), V), (dict(ws=A + 4), AL), (dict(wo=A + 4), AL),
                   (dict(gq=None), V), (dict(lam=None), V), (dict(q=_lib.View4(A + 8, 128, 64, 64)), AL),
                   (dict(y=_lib.View4(None, 128, 64, 64)), V)):
        assert attn(pages(), **kw) == rc, kw
    assert attn(pages(weight=None), wo=A) == V and "weight" in _lib.last_error()


def test_cache_refusals():
    lib, V, AL = _lib.load(), _lib.ERR_VALUE, _lib.ERR_ALIGN

    def evict(pg, **kw):
        a = dict(table=A, mp=4, pos=A, budget=100, recent=8, slots=A)
        a.update(kw)
        return lib.sisa_paged_evict(ctypes.byref(pg), a["table"], 4, a["mp"], a["pos"], 3, 2, a["budget"], a["recent"],
                                    a["slots"], None, None)

    for kw in (dict(budget=0), dict(budget=257), dict(recent=100), dict(recent=-1), dict(pos=None), dict(slots=None)):
        assert evict(pages(), **kw) == V, kw
    assert evict(pages(token=None)) == V and evict(pages(weight=None)) == V

    def append(pg, **kw):
        a = dict(proj=A, psb=560, z=A, pos=A, slots=None, budget=0, ci=A, co=A, c=A, g=A, f=A)
        a.update(kw)
        return lib.sisa_paged_append(a["proj"], a["psb"], a["z"], 2, ctypes.byref(pg), A, 4, 4, a["pos"], a["slots"],
                                     a["budget"], 3, 2, _lib.BF16, a["ci"], a["co"], a["c"], a["g"], a["f"], None, None, None)

    for kw, rc in ((dict(proj=None), V), (dict(psb=540), AL), (dict(psb=561), AL), (dict(z=None), V), (dict(f=None), V),
                   (dict(pos=None), V), (dict(budget=257), V), (dict(budget=-1), V), (dict(ci=None), V), (dict(c=A + 2), AL)):
        assert append(pages(), **kw) == rc, kw
    assert append(pages(f=None)) == V

    view = lambda w: _lib.View4(A, 200 * w * 2, w, 2 * w)  # noqa: E731

    def fill(pg, **kw):
        a = dict(k=view(64), v=view(64), b=view(32), g=A, f=A, w=A, L=200, keep=100, recent=10, ws=A)
        a.update(kw)
        return lib.sisa_paged_fill(ctypes.byref(pg), A, 4, 4, _lib.vref(a["k"]), _lib.vref(a["v"]), _lib.vref(a["b"]), a["g"],
                                   400, 200, a["f"], 400, 200, a["w"], 3, 2, a["L"], a["keep"], a["recent"], a["ws"], None, None)

    for kw, rc in ((dict(keep=0), V), (dict(keep=201), V), (dict(L=400, keep=300), V), (dict(recent=101), V), (dict(recent=-1), V),
                   (dict(w=None), V), (dict(g=None), V), (dict(ws=None), V), (dict(ws=A + 4), AL), (dict(L=0), V),
                   (dict(k=_lib.View4(A + 2, 64, 64, 64)), AL)):
        assert fill(pages(), **kw) == rc, kw

    def weights(**kw):
        a = dict(pos=A, lam=A, lse=A, first=0, w=A, dtype=_lib.BF16)
        a.update(kw)
        return lib.sisa_attn_key_weights(*(_lib.vref(view(x)) for x in (64, 64, 32, 32)), a["pos"], a["lam"], a["lse"], 3, 2, 200,
                                         a["first"], a["dtype"], a["w"], None, None)

    for kw, rc in ((dict(pos=None), V), (dict(pos=A + 4), AL), (dict(lse=None), V), (dict(w=None), V), (dict(first=200), V),
                   (dict(first=-1), V), (dict(dtype=_lib.F32), _lib.ERR_TYPE)):
        assert weights(**kw) == rc, kw


def test_launches_report_a_refused_shared_memory_size():
    """Every opt-in to more shared memory in the paged cache's sources hands its result on."""
    import re

    csrc = Path(__file__).resolve().parents[1] / "sisa_b200" / "csrc"
    for name in ("paged_attn.cu", "paged_cache.cu", "key_weights.cu"):
        text = (csrc / name).read_text()
        calls = re.findall(r"^(.*)\bcudaFuncSetAttribute\(", text, flags=re.M)
        assert calls and all(head.rstrip().endswith("=") for head in calls), name
        assert len(re.findall(r"if \(e != cudaSuccess\) return e;", text)) >= len(calls), name
