"""Sizes at the ends of their types in the serving operators' plans, on the CPU."""
import os

import pytest

from heterocache_amd import _lib


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libhc.so not built")
    return _lib.load()


@pytest.mark.parametrize("batch,q_heads,kv_heads,queries", [(1, 8, 2, 1), (128, 32, 8, 1), (3, 14, 2, 4)])
def test_largest_tile_counts(lib, batch, q_heads, kv_heads, queries):
    """Tile counts are sizes to cut for and no limits: 'as many as you like' plans as a very long prefix or row does."""
    def size(prefix, rows):
        return lib.hc_shared_workspace_size(2, batch, q_heads, kv_heads, queries, prefix, rows)
    long = 1 << 36
    for most in (1 << 40, 1 << 62, (1 << 63) - 9, (1 << 63) - 3, (1 << 63) - 1):
        assert size(most, 4) == size(long, 4)
        assert size(1000, most) == size(1000, long)
        assert size(most, most) == size(long, long)
    assert size(long, 4) >= size(1 << 20, 4) > 0


def test_workspace_of_one_part_alone(lib):
    """No partials are kept for a prefix or rows that the call does not have, nor for rows that write their output."""
    size = lib.hc_shared_workspace_size
    assert size(2, 1, 40, 8, 32768, -1, 1025) == 0
    for args in ((2, 1, 32, 8, 1), (1, 4, 14, 2, 3), (0, 1, 4, 4, 1)):
        # The rows' cut does not depend on the prefix; the prefix's is the one
        # beside rows of no tiles.
        assert 0 < size(*args, -1, 500) < size(*args, 2000, 500)
        assert 0 < size(*args, 2000, -1) < size(*args, 2000, 0)
    assert size(2, 1, 8, 2, 1, -1, -1) == 0


def test_negative_tile_counts(lib):
    """Refused of a prefix or rows that are there, before anything is read."""
    import ctypes
    st = (ctypes.c_int64 * 3)(1024, 128, 1024)
    fake = 4096
    for pre, rows, pt, rt in ((fake, fake, -1, 4), (fake, fake, 4, -1), (None, fake, 4, -2), (fake, None, -1, 4)):
        rc = lib.hc_shared_attn(2, fake, st, fake, fake, fake, pre, pt, fake, fake, fake, rows, None, rt, fake, st, 1,
                                8, 2, 1, 0.1, fake, 1 << 40, None)
        assert rc == _lib.HC_ERR_INVALID and b"tiles=-" in lib.hc_last_error()
