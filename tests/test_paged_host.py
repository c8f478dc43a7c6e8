"""The paged cache on the host: the C ABI's argument checks, the wrappers' refusals, how attention is laid out, and the loads that go to LDS.  Nothing is
launched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from polarquant_amd import _ffi, build, paged

A, ODD = 0x10000, 0x10004              # stand-in addresses; nothing is launched by the validators
OK, NUL, SHAPE, BITS, DTYPE, ALIGN, STRIDE, WS = 0, -1, -2, -3, -4, -5, -6, -7
LAYOUT = (32768, 16384, 32768, 16384, 16384, 8192, 128, 64, 10, 20, 20)


def layout(**kw):
    v = list(LAYOUT)
    for i, x in kw.items():
        v[int(i[1:])] = x
    return (ctypes.c_int64 * 11)(*v)


@pytest.fixture(scope="module")
def lib():
    return _ffi.paged_lib()


def caller(fn, names, defaults):
    def call(**kw):
        d = dict(defaults)
        d.update(kw)
        return fn(*[d[n] for n in names.split()])
    return call


CACHE = dict(keys=A, values=A, codes=A, rs=A, rm=A, ts=A, tm=A, lay=None, qs=A, kv=A, ns=A, pages=A, vp=A, op=A, W=8, Wo=4, T=20, B=2, N=8, Nk=2, mq=16, mkv=1000,
             rb=4, tb=4, dt=1, flags=0)


def test_header_and_signatures_name_the_same_symbols(lib):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "polarquant_paged.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    found = re.findall(r"\b(pq_\w+)\s*\(([^)]*)\)\s*;", text)
    assert {n for n, _ in found} == set(_ffi.PAGED_SIGNATURES)
    for n, args in found:
        assert len(args.split(",")) == len(_ffi.PAGED_SIGNATURES[n][1]), n
    assert "PQ_EVICT_MAX_PAGES %d" % _ffi.PQ_EVICT_MAX_PAGES in text and "PQ_PAGE %d" % paged.PAGE in text


def test_attention_arguments(lib):
    call = caller(lib.pq_validate_paged_attn, "q qr keys values codes rs rm ts tm lay qs kv ns pages vp op W Wo mask mr out lse T B N Nk mq mkv rb tb sp ws wb dt flags",
                  dict(CACHE, q=A, qr=1024, lay=layout(), mask=None, mr=0, out=A, lse=None, sp=0, ws=None, wb=0))
    assert call() == OK and call(codes=None, pages=None, rs=None) == OK and call(lse=A, mask=A, mr=1000) == OK and call(ns=None) == OK
    assert call(Wo=0, op=None) == OK and call(N=34, Nk=2, qr=34 * 128) == OK and call(dt=0) == OK
    for k in ("q", "keys", "values", "out", "qs", "kv", "vp", "op", "pages", "rs", "tm", "lay"):
        assert call(**{k: None}) == NUL, k
    for kw in (dict(B=0), dict(N=9), dict(Nk=0), dict(mq=0), dict(mq=21), dict(mkv=0), dict(mkv=1025), dict(W=0), dict(T=0), dict(Wo=-1), dict(flags=8), dict(sp=-1),
               dict(sp=70000), dict(lay=layout(_8=-1)), dict(lay=layout(_10=1 << 31)), dict(T=1 << 28, N=8), dict(B=65536)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(rb=0), dict(tb=0), dict(rb=5), dict(rb=1, tb=8), dict(flags=4), dict(flags=4, rb=4, tb=3)):
        assert call(**kw) == BITS, kw
    assert call(flags=4, rb=3, tb=3) == OK and call(rb=1, tb=7) == OK
    assert call(dt=2) == DTYPE
    for kw in (dict(qr=1020), dict(qr=512), dict(qr=-1024), dict(qr=1 << 25), dict(lay=layout(_0=4)), dict(lay=layout(_5=8)), dict(lay=layout(_3=-16384)), dict(mask=A, mr=999)):
        assert call(**kw) == STRIDE, kw
    for k in ("q", "keys", "values", "codes", "rm", "out"):
        assert call(**{k: ODD}) == ALIGN, k
    assert call(qs=A + 2) == ALIGN and call(pages=A + 1) == ALIGN
    size = lib.pq_paged_attn_workspace_bytes
    need = size(2, 8, 2, 16, 5)
    assert need == 5 * 2 * 256 * 130 * 4 + 16 and size(2, 8, 2, 4, 5) == 5 * 2 * 16 * 130 * 4 + 16 and size(2, 8, 2, 16, 0) == 0
    assert call(sp=5, ws=A, wb=need) == OK and call(sp=5, ws=A, wb=need - 1) == WS and call(sp=5) == NUL and call(sp=5, ws=ODD, wb=need) == ALIGN
    assert call(sp=1, ws=A, wb=1 << 30) == WS           # fewer than row tiles


def test_weights_arguments(lib):
    call = caller(lib.pq_validate_paged_weights, "q qr lse keys codes rs rm ts tm lay qs kv ns pages vp op W Wo mask mr onto out T B N Nk mq mkv rb tb dt flags",
                  dict(CACHE, q=A, qr=1024, lay=layout(), lse=A, mask=None, mr=0, onto=None, out=A))
    assert call() == OK and call(onto=A, codes=None, pages=None) == OK
    for k in ("q", "lse", "keys", "out", "qs", "kv", "vp"):
        assert call(**{k: None}) == NUL, k
    assert call(W=65536) == SHAPE and call(N=7) == SHAPE and call(dt=2) == DTYPE and call(tb=5) == BITS and call(lse=A + 2) == ALIGN and call(qr=8) == STRIDE


def test_append_arguments(lib):
    names = "q qr k kr v vr cos sin ar pos qn kn qo keys values lay qs kv ns vp op W Wo T B N Nk mq mkv dt"
    call = caller(lib.pq_validate_paged_append, names,
                  dict(CACHE, q=A, qr=1536, k=A, kr=1536, v=A, vr=1536, cos=A, sin=A, ar=100, pos=None, qn=None, kn=None, qo=A, lay=layout()))
    assert call() == OK and call(pos=A, qn=A, kn=A, ns=None) == OK
    for k in ("q", "k", "v", "cos", "sin", "qo", "keys", "values", "vp", "qs"):
        assert call(**{k: None}) == NUL, k
    assert call(ar=0) == SHAPE and call(mq=21) == SHAPE and call(kr=128) == STRIDE and call(vr=260) == STRIDE and call(qn=ODD) == ALIGN and call(dt=2) == DTYPE


def test_evict_arguments(lib):
    names = "w p ns kv B Nk W keep sinks po no ko wo fr"
    call = caller(lib.pq_validate_evict_pages, names, dict(w=A, p=A, ns=A, kv=A, B=2, Nk=2, W=8, keep=4, sinks=1, po=A + 64, no=A + 64, ko=A + 64, wo=A + 64, fr=A + 128))
    assert call() == OK and call(sinks=4) == OK and call(keep=100) == OK and call(W=16384) == OK
    for k in names.split():
        if k not in ("B", "Nk", "W", "keep", "sinks"):
            assert call(**{k: None}) == NUL, k
    for kw in (dict(B=0), dict(Nk=0), dict(W=0), dict(W=16385), dict(keep=0, sinks=0), dict(sinks=5), dict(sinks=-1), dict(po=A), dict(wo=A), dict(fr=A + 64), dict(ko=A)):
        assert call(**kw) == SHAPE, kw


def test_seal_arguments():
    call = caller(_ffi.lib().pq_validate_seal_pages, "keys lay codes rs rm ts tm kv ns pages op W Wo B Nk rb tb dt flags", dict(CACHE, lay=layout()))
    assert call() == OK and call(ns=None) == OK and call(flags=9) == OK and call(flags=4, rb=3, tb=3) == OK
    for k in ("keys", "codes", "rs", "kv", "pages", "op", "lay"):
        assert call(**{k: None}) == NUL, k
    assert call(W=0) == SHAPE and call(Wo=0) == SHAPE and call(flags=2) == SHAPE and call(B=65536) == SHAPE and call(rb=5) == BITS and call(flags=4) == BITS
    assert call(dt=2) == DTYPE and call(lay=layout(_4=8)) == STRIDE and call(keys=ODD) == ALIGN


def test_units(lib):
    plan = lib.pq_paged_attn_plan
    assert plan(1, 32, 8, 1, 128, 256) == 0                             # a page is not cut
    assert plan(1, 32, 8, 1, 2000, 256) == 16                           # as many workgroups a KV head as pages
    assert plan(1, 32, 8, 1, 131072, 256) == 64 and plan(16, 32, 8, 1, 32769, 256) == 64     # two on every unit
    assert plan(64, 32, 8, 1, 32769, 256) == 0 and plan(1, 32, 8, 2048, 40000, 256) == 0     # the row tiles fill the device
    assert plan(0, 1, 1, 1, 1, 256) == 0 and plan(1, 3, 2, 1, 1, 256) == 0


def test_refusals():
    cpu = torch.zeros(3, 2, 128, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged.PagePool(cpu, cpu)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged.PageBatch(None, torch.zeros(1, dtype=torch.int32), None, torch.zeros(1, 1, dtype=torch.int32), None, 1, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged.evict_pages(torch.zeros(1, 1, 1), None, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged.paged_attention(cpu[:, :, 0], None, None)


@pytest.mark.parametrize("src", [u[0] for u in build.LAYER_UNITS["paged"] if "capi" not in u[0]])
def test_a_wait_state_before_every_load_to_lds(src):
    """Loads that go to LDS directly read M0 one wait state after a scalar write at the earliest, which inside an asm statement nobody sees to."""
    cmd = [build._hipcc()] + build.FLAGS + ["--cuda-device-only", "-S", os.path.join(build.CSRC, src), "-o", "-"]
    run = subprocess.run(cmd, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    loads, previous = 0, ""
    for line in run.stdout.splitlines():
        line = line.split(";")[0].strip()
        if not line or line.startswith(".") or line.endswith(":"):
            continue
        if re.match(r"buffer_load\S* .*\blds\b", line):
            loads += 1
            assert not re.match(r"s_\S+ m0\b", previous), (previous, line)
        previous = line
    assert (loads > 0) == ("chunk" in src or "weights" in src)
