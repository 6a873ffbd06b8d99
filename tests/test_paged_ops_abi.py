"""Refusals of the paged cache's C entry points: every one is made before a HIP call, so they run on the CPU."""
import ctypes
import os
import re

import pytest

from heterocache_amd import _lib

FAKE = 4096  # 16-byte aligned, never dereferenced: validation fails first
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libhc.so not built")
    return _lib.load()


def _s(*v):
    return (ctypes.c_int64 * 3)(*v)


def _refused(lib, rc, text):
    assert rc == _lib.HC_ERR_INVALID and text in lib.hc_last_error(), (rc, lib.hc_last_error())


def _cache(**kw):
    a = dict(dtype=2, batch=2, kv_heads=2, heads=1, pages=9, page_tokens=16, table_pages=4, k=FAKE, v=FAKE,
             k_strides=_s(2048, 128, 0), v_strides=_s(2048, 128, 0), table=FAKE, table_stride=4, row_len=FAKE,
             weights=FAKE, weight_stride=64, pos=FAKE, pos_stride=64, dropped=FAKE, status=None)
    a.update(kw)
    return _lib.PagedCache(**a)


def test_structure_matches_the_header():
    text = open(os.path.join(ROOT, "include", "hc.h")).read()
    body = re.search(r"typedef struct hc_paged_cache \{(.*?)\} hc_paged_cache;", text, re.S).group(1)
    names = [re.sub(r"\[\d\]", "", n).strip(" *\n") for line in body.split(";") if line.strip()
             for n in re.sub(r"^\s*(const )?\w+\s*", "", line).split(",")]
    assert names == [n for n, _ in _lib.PagedCache._fields_]


BAD_CACHES = [
    (dict(dtype=3), b"dtype 3"), (dict(batch=-1), b"batch=-1"), (dict(kv_heads=0), b"kv_heads=0"),
    (dict(kv_heads=4, heads=2), b"heads=2"), (dict(batch=1 << 24), b"2^24"), (dict(pages=0), b"pages=0"),
    (dict(page_tokens=0), b"page_tokens=0"), (dict(table_pages=0), b"table_pages=0"),
    (dict(page_tokens=1 << 20, table_pages=1 << 20), b"2^30 tokens"),
    (dict(batch=1 << 20, page_tokens=1 << 10, table_pages=1 << 10, table_stride=1 << 10), b"2^30 tiles"),
    (dict(k=None), b"null"), (dict(table=None), b"null"), (dict(row_len=None), b"null"),
    (dict(k_strides=_s(2048, 129, 0)), b"strides"), (dict(v_strides=_s(-2048, 128, 0)), b"strides"),
    (dict(k_strides=_s(2048, 1 << 26, 0)), b"token stride"), (dict(v=FAKE + 8), b"aligned"),
    (dict(table_stride=3), b"table rows 3 apart"), (dict(weight_stride=63), b"weights need"),
    (dict(pos=None), b"weights need"), (dict(dropped=None), b"weights need"), (dict(pos_stride=0), b"weights need"),
]


def _append(lib, c, k=FAKE, ks=_s(256, 128, 256), v=FAKE, vs=_s(256, 128, 256), t=1, lo=FAKE):
    return lib.hc_paged_append(ctypes.byref(c) if c else None, k, ks, v, vs, None, t, lo, None)


def _attn(lib, c, q=FAKE, qs=_s(1024, 128, 1024), hq=8, n=1, k=FAKE, ks=_s(256, 128, 256), v=FAKE, vs=_s(256, 128, 256),
          scale=0.1, weigh=0, wo=None, lo=None, out=FAKE, os_=_s(1024, 128, 1024), ws=FAKE, wb=0):
    return lib.hc_paged_attn(ctypes.byref(c) if c else None, q, qs, hq, n, k, ks, v, vs, None, scale, weigh, wo, lo, out,
                             os_, ws, wb, None)


def _evict(lib, c, keep=None, every=8, sink=2, recent=2, ws=FAKE, wb=None):
    ref = ctypes.byref(c) if c else None
    wb = lib.hc_paged_evict_scratch_size(ref) - 1 if wb is None else wb
    return lib.hc_paged_evict(ref, keep, every, sink, recent, None, None, None, None, ws, wb, None)


@pytest.mark.parametrize("kw,text", BAD_CACHES)
def test_caches(lib, kw, text):
    c = _cache(**kw)
    _refused(lib, _append(lib, c), text)
    _refused(lib, _attn(lib, c), text)
    _refused(lib, _evict(lib, c, wb=1 << 40), text)


def test_no_cache(lib):
    _refused(lib, _append(lib, None), b"null cache")
    _refused(lib, _attn(lib, None), b"null cache")
    _refused(lib, lib.hc_paged_evict(None, None, 8, 0, 0, None, None, None, None, FAKE, 1 << 30, None), b"null cache")
    assert lib.hc_paged_workspace_size(None, 8, 1, 1, 0) == 0 and lib.hc_paged_evict_scratch_size(None) == 0


def test_append(lib):
    c = _cache()
    _refused(lib, _append(lib, c, t=-1), b"tokens=-1")
    _refused(lib, _append(lib, c, k=None), b"null")
    _refused(lib, _append(lib, c, vs=None), b"null")
    _refused(lib, _append(lib, c, ks=_s(256, 128, 260)), b"strides")
    _refused(lib, _append(lib, c, v=FAKE + 2), b"aligned")
    _refused(lib, _append(lib, c, lo=FAKE + 4), b"overlaps")
    _refused(lib, _append(lib, c, lo=FAKE - 12), b"overlaps")
    _refused(lib, _append(lib, _cache(batch=1 << 20, table_pages=1, table_stride=1), t=1 << 20), b"rows x")
    assert _append(lib, _cache(batch=0)) == 0 and _append(lib, c, t=0, lo=None) == 0


def test_attn(lib):
    c = _cache()
    for n in (1, 40):
        for weigh in (0, 1):
            size = lib.hc_paged_workspace_size(ctypes.byref(c), 8, n, 0, weigh)
            assert size > 0
            _refused(lib, _attn(lib, c, n=n, weigh=weigh, wb=size - 1), b"workspace too small")
            _refused(lib, _attn(lib, c, n=n, weigh=weigh, wb=size, ws=FAKE + 8), b"workspace")
            _refused(lib, _attn(lib, c, n=n, weigh=weigh, wb=size, ws=None), b"workspace")
    _refused(lib, _attn(lib, c, hq=9), b"q_heads=9")
    _refused(lib, _attn(lib, c, hq=0), b"q_heads=0")
    _refused(lib, _attn(lib, c, n=-1), b"queries=-1")
    _refused(lib, _attn(lib, c, n=1 << 23), b"2^26")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _refused(lib, _attn(lib, c, scale=scale), b"scale")
    _refused(lib, _attn(lib, _cache(weights=None), weigh=1), b"no weights")
    _refused(lib, _attn(lib, c, wo=FAKE), b"weights_out without")
    _refused(lib, _attn(lib, c, k=None, v=None, lo=FAKE), b"len_out without")
    _refused(lib, _attn(lib, c, k=None), b"null")
    _refused(lib, _attn(lib, c, q=None), b"null")
    _refused(lib, _attn(lib, c, os_=None), b"null")
    _refused(lib, _attn(lib, c, qs=_s(1024, 128, 1028)), b"strides")
    _refused(lib, _attn(lib, c, os_=_s(1024, 4, 1024)), b"strides")
    _refused(lib, _attn(lib, c, ks=_s(1, 128, 128)), b"strides")
    _refused(lib, _attn(lib, c, out=FAKE + 8), b"aligned")
    assert _attn(lib, _cache(batch=0)) == 0 and _attn(lib, c, n=0) == 0
    assert lib.hc_paged_workspace_size(ctypes.byref(c), 9, 1, 1, 0) == 0


def test_evict(lib):
    c = _cache()
    _refused(lib, _evict(lib, c), b"scratch too small")
    _refused(lib, _evict(lib, c, wb=1 << 30, ws=None), b"scratch")
    _refused(lib, _evict(lib, c, wb=1 << 30, ws=FAKE + 4), b"scratch")
    _refused(lib, _evict(lib, c, every=-1), b"keep=-1")
    _refused(lib, _evict(lib, c, sink=-1), b"sink=-1")
    _refused(lib, _evict(lib, c, recent=-2), b"recent=-2")
    _refused(lib, _evict(lib, c, recent=7), b"exceed keep=8")
    _refused(lib, _evict(lib, _cache(weights=None)), b"no weights")
    assert _evict(lib, _cache(batch=0)) == 0


def test_query_rows_past_64_bits(lib):
    c = _cache(batch=16)
    _refused(lib, _attn(lib, c, hq=1 << 30, n=1 << 30), b"2^26")
    _refused(lib, _attn(lib, c, hq=1 << 24, n=1 << 30), b"2^26")
    assert lib.hc_paged_workspace_size(ctypes.byref(c), 1 << 30, 1 << 30, 0, 0) == 0
    assert lib.hc_paged_workspace_size(ctypes.byref(c), 8, 1 << 20, 0, 0) == 0
    assert lib.hc_paged_workspace_size(ctypes.byref(c), 8, 1 << 19, 0, 0) > 0
