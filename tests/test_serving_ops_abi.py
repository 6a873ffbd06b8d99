"""Refusals of the serving operators' C entry points: every one is made before a HIP call, so they run on the CPU."""
import ctypes
import os

import pytest

from heterocache_amd import _lib

FAKE = 4096  # 16-byte aligned, never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libhc.so not built")
    return _lib.load()


def _s(*v):
    return (ctypes.c_int64 * 3)(*v)


def _refused(lib, rc, text):
    assert rc == _lib.HC_ERR_INVALID and text in lib.hc_last_error(), (rc, lib.hc_last_error())


def _append(lib, **kw):
    a = dict(dtype=2, tdtype=2, q=FAKE, qs=_s(1024, 128, 1024), qo=FAKE, qos=_s(1024, 128, 1024), k=FAKE,
             ks=_s(256, 128, 256), v=FAKE, vs=_s(256, 128, 256), cos=FAKE, sin=FAKE, tb=0, tt=128, kst=FAKE, vst=FAKE,
             off=FAKE, len=FAKE, cap=FAKE, lo=FAKE, counts=None, b=1, hq=8, hkv=2, t=1, status=None)
    a.update(kw)
    return lib.hc_append_rotated(a["dtype"], a["tdtype"], a["q"], a["qs"], a["qo"], a["qos"], a["k"], a["ks"], a["v"],
                                 a["vs"], a["cos"], a["sin"], a["tb"], a["tt"], a["kst"], a["vst"], a["off"], a["len"],
                                 a["cap"], a["lo"], a["counts"], a["b"], a["hq"], a["hkv"], a["t"], a["status"], None)


def test_append_rotated(lib):
    _refused(lib, _append(lib, hq=7), b"q_heads=7")
    _refused(lib, _append(lib, hkv=0), b"kv_heads=0")
    _refused(lib, _append(lib, t=-1), b"tokens=-1")
    _refused(lib, _append(lib, t=2 ** 31 - 1), b"tokens=")
    _refused(lib, _append(lib, dtype=5), b"dtype")
    _refused(lib, _append(lib, tdtype=1), b"tables")
    _refused(lib, _append(lib, len=None), b"null")
    _refused(lib, _append(lib, cap=None), b"null")
    _refused(lib, _append(lib, cos=None), b"null")
    _refused(lib, _append(lib, ks=None), b"strides")
    _refused(lib, _append(lib, ks=_s(256, 128, 260)), b"strides")
    _refused(lib, _append(lib, tt=132), b"table strides")
    _refused(lib, _append(lib, v=FAKE + 2), b"aligned")
    _refused(lib, _append(lib, b=1 << 20, t=1 << 20), b"rows")
    _refused(lib, _append(lib, off=None, t=0, lo=FAKE + 64), b"null")
    _refused(lib, _append(lib, lo=FAKE + 4), b"overlaps")
    _refused(lib, _append(lib, lo=FAKE - 4), b"overlaps")
    assert _append(lib, b=0) == 0 and _append(lib, t=0, q=None, lo=None) == 0


def _shared(lib, **kw):
    a = dict(dtype=2, q=FAKE, qs=_s(1024, 128, 1024), pk=FAKE, pv=FAKE, po=FAKE, pl=FAKE, pt=4, k=FAKE, v=FAKE, off=FAKE,
             len=FAKE, rt=4, out=FAKE, os=_s(1024, 128, 1024), b=1, hq=8, hkv=2, n=1, scale=0.1, ws=FAKE, wb=0)
    a.update(kw)
    return lib.hc_shared_attn(a["dtype"], a["q"], a["qs"], a["pk"], a["pv"], a["po"], a["pl"], a["pt"], a["k"], a["v"],
                              a["off"], a["len"], None, a["rt"], a["out"], a["os"], a["b"], a["hq"], a["hkv"], a["n"],
                              a["scale"], a["ws"], a["wb"], None)


def test_shared_attn(lib):
    _refused(lib, _shared(lib), b"workspace too small")
    _refused(lib, _shared(lib, wb=lib.hc_shared_workspace_size(2, 1, 8, 2, 1, 4, 4) - 1), b"workspace too small")
    _refused(lib, _shared(lib, ws=None, wb=1 << 30), b"workspace too small")
    _refused(lib, _shared(lib, hq=9), b"q_heads=9")
    _refused(lib, _shared(lib, hq=34), b"at most 16")
    _refused(lib, _shared(lib, dtype=3), b"dtype=3")
    _refused(lib, _shared(lib, b=1 << 23), b"2^24")
    _refused(lib, _shared(lib, pt=-1), b"hc_shared_attn")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _refused(lib, _shared(lib, scale=scale), b"scale")
    _refused(lib, _shared(lib, pl=None, len=None), b"neither")
    _refused(lib, _shared(lib, pk=None), b"null")
    _refused(lib, _shared(lib, off=None), b"null")
    _refused(lib, _shared(lib, qs=_s(1024, 128, 1028)), b"strides")
    _refused(lib, _shared(lib, k=FAKE + 8), b"aligned")
    assert _shared(lib, b=0) == 0 and _shared(lib, n=0) == 0
    assert lib.hc_shared_workspace_size(2, 1, 34, 2, 1, 4, 4) == 0


def test_shared_workspace_is_bounded(lib):
    """Partials grow with the work of one round of workgroups, not with the prefix."""
    for tiles in (1 << 12, 1 << 16, 1 << 22):
        assert 0 < lib.hc_shared_workspace_size(2, 32, 32, 8, 1, tiles, 16) < 100 << 20


def test_block_bounds(lib):
    def call(dtype=2, ks=FAKE, off=FAKE, rows=2, block=32, span=1, fresh=0, bounds=FAKE, exps=FAKE):
        return lib.hc_block_bounds(dtype, ks, off, FAKE, FAKE, rows, block, span, fresh, bounds, exps, None)
    _refused(lib, call(dtype=9), b"dtype")
    for block in (0, 16, 33, -32, 1 << 21):
        _refused(lib, call(block=block), b"block=")
    _refused(lib, call(span=-1), b"span=-1")
    _refused(lib, call(fresh=-2), b"fresh=-2")
    _refused(lib, call(ks=None), b"null")
    _refused(lib, call(bounds=FAKE + 1), b"aligned")
    _refused(lib, call(rows=1 << 20, span=1 << 20), b"blocks")
    assert call(rows=0) == 0 and call(span=0) == 0


def test_block_select(lib):
    def call(dtype=2, q=FAKE, qs=_s(1024, 128, 1024), b=1, hq=8, hkv=2, n=1, block=32, mb=20000, keep=8, sink=1, local=2,
             idx=FAKE, scratch=FAKE, sb=None):
        sb = lib.hc_block_select_scratch_size(b, hkv, n, mb) - 1 if sb is None else sb
        return lib.hc_block_select(dtype, q, qs, FAKE, FAKE, FAKE, FAKE, None, b, hq, hkv, n, block, mb, keep, sink, local, idx,
                                   FAKE, scratch, sb, None)
    _refused(lib, call(), b"scratch too small")
    _refused(lib, call(scratch=None, sb=1 << 30), b"scratch too small")
    _refused(lib, call(scratch=FAKE + 8, sb=1 << 30), b"aligned")
    _refused(lib, call(hq=9), b"q_heads=9")
    _refused(lib, call(block=40), b"block=40")
    for kw in (dict(keep=0), dict(local=0), dict(sink=-1), dict(keep=2), dict(sink=7), dict(mb=-1), dict(keep=1 << 25)):
        _refused(lib, call(**kw), b"hc_block_select")
    _refused(lib, call(idx=None), b"null")
    _refused(lib, call(qs=_s(1024, 4, 1024)), b"strides")
    _refused(lib, call(q=FAKE + 4), b"aligned")
    assert call(b=0) == 0 and call(n=0) == 0


def test_block_attn(lib):
    def call(dtype=2, q=FAKE, qs=_s(1024, 128, 1024), ks=FAKE, idx=FAKE, keep=4096, block=32, b=1, hq=8, hkv=2, n=1,
             scale=0.1, ws=FAKE, wb=0):
        return lib.hc_block_attn(dtype, q, qs, ks, FAKE, FAKE, FAKE, None, idx, FAKE, keep, block, FAKE,
                                 _s(1024, 128, 1024), b, hq, hkv, n, scale, ws, wb, None)
    assert lib.hc_block_attn_workspace_size(1, 8, 2, 1, 32, 4096) > 0  # the kept blocks are split
    _refused(lib, call(), b"workspace too small")
    _refused(lib, call(hq=34), b"at most 16")
    _refused(lib, call(keep=0), b"keep=0")
    _refused(lib, call(block=48), b"block=48")
    _refused(lib, call(scale=-0.5), b"scale")
    _refused(lib, call(keep=1 << 24, block=1 << 12), b"keep=")
    _refused(lib, call(idx=None), b"null")
    _refused(lib, call(ks=FAKE + 8), b"aligned")
    assert call(b=0) == 0 and call(n=0) == 0
    assert lib.hc_block_attn_workspace_size(1, 8, 2, 1, 33, 8) == 0


def test_block_step(lib):
    def call(dtype=2, q=FAKE, ks=FAKE, bounds=FAKE, b=1, hq=8, hkv=2, n=1, block=32, mb=20000, keep=4096, sink=1, local=2,
             scale=0.1, idx=FAKE, out=FAKE, ws=FAKE, wb=0):
        return lib.hc_block_step(dtype, q, _s(1024, 128, 1024), ks, FAKE, FAKE, FAKE, None, bounds, FAKE, FAKE, b, hq,
                                 hkv, n, block, mb, keep, sink, local, scale, idx, FAKE, out, _s(1024, 128, 1024), ws, wb, None)
    size = lib.hc_block_step_workspace_size(1, 8, 2, 1, 32, 20000, 4096)
    assert size >= lib.hc_block_select_scratch_size(1, 2, 1, 20000) + lib.hc_block_attn_workspace_size(1, 8, 2, 1, 32, 4096)
    _refused(lib, call(), b"workspace too small")
    _refused(lib, call(wb=size, ws=FAKE + 8), b"workspace")
    _refused(lib, call(hq=9), b"q_heads=9")
    _refused(lib, call(block=31), b"block=31")
    _refused(lib, call(sink=4095), b"keep=4096")
    _refused(lib, call(local=0), b"local")
    _refused(lib, call(scale=0.0), b"scale")
    _refused(lib, call(idx=None), b"null")
    _refused(lib, call(out=None), b"null")
    _refused(lib, call(ks=FAKE + 8), b"aligned")
    _refused(lib, call(bounds=FAKE + 8), b"aligned")
    assert call(b=0) == 0 and call(n=0) == 0
    assert lib.hc_block_step_workspace_size(1, 8, 2, 1, 32, 128, 16) == 0  # one launch
