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
