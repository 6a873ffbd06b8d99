"""The paged cache at the edges of what its calls allow."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import _lib, ops
from tests.paged_util import Cache, queries
from tests.serving_util import D

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
SCALE = 1 / math.sqrt(D)


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("page,dtype,apart", [(16, BF, False), (24, BF, True), (16, FL, True)])
@pytest.mark.parametrize("wide", [False, True])
def test_new_tokens_without_a_page(dev, wide, page, dtype, apart, weigh):
    """A padded batch of which one row's table names no page for some of its new tokens: the queries that see them get
    NaN, and so does every weight that they add to; the other sequences and all stored pages are as in a call without the
    fault.  Tables as wide as their rows, and far wider, take the batch in one launch and in several."""
    T, lens, counts = 40, [60, 48, 47], [40, 1, 17]
    width = -(-(24000 if wide else 112) // page)
    for b, value in ((0, -1), (0, 1 << 30), (1, -1), (2, -(1 << 31))):
        good, c = (Cache(np.random.default_rng(10 * page + b), 3, 2, [n for n in lens for _ in range(2 if apart else 1)], page, dtype,
                         dev, apart=apart, room=T, stale=0.0, ledger=True, width=width) for _ in range(2))
        n = lens[b] + counts[b]
        entry = (n - 1) // page
        assert entry * page >= lens[b]  # its tokens are new
        rows = [2 * b, 2 * b + 1] if apart else [b]
        c.pages.table[rows, entry] = value
        rng = np.random.default_rng(b)
        q, kn, vn = (queries(rng, 3, h, T, dtype, dev) for h in (8, 2, 2))
        dc = torch.tensor(counts, dtype=torch.int32, device=dev)
        want = ops.paged_attn(q, good.pages, SCALE, kn, vn, counts=dc, weigh=weigh)
        got = ops.paged_attn(q, c.pages, SCALE, kn, vn, counts=dc, weigh=weigh)
        others = [x for x in range(3) if x != b]
        assert torch.isfinite(want.float()).all() and torch.equal(got[others], want[others])
        assert torch.isnan(got[b, entry * page - lens[b]:counts[b]].float()).all(), (b, value)
        assert not got[b, counts[b]:].any()
        with pytest.raises(_lib.HCError, match="names no page"):
            ops.read_status(c.status)
        assert torch.equal(c.pages.row_len, good.pages.row_len)
        if weigh:
            mine = torch.arange(6, device=dev) // 2 == b
            assert torch.isnan(c.pages.weights[mine, :n]).all(), (b, value)
            assert torch.equal(c.pages.weights[~mine], good.pages.weights[~mine])
        # The entry's tokens are left out, and nothing else.
        left = torch.ones(len(good.k), dtype=torch.bool, device=dev)
        left[torch.as_tensor(good.table[rows, entry].astype(np.int64)).to(dev)] = False
        assert torch.equal(c.k[left], good.k[left]) and torch.equal(c.v[left], good.v[left])


@pytest.mark.parametrize("apart", [True, False])
@pytest.mark.parametrize("counts", [False, True])
def test_no_tokens(dev, apart, counts):
    """A call of no tokens has no outputs, but lengths and weights: the old ones, also in memory of their own."""
    c = Cache(np.random.default_rng(1), 2, 3, [70, 0, 33], 16, BF, dev, apart=apart, ledger=True)
    p = c.pages
    lens, w0 = p.row_len.clone(), p.weights.clone()
    q, kn, vn = (torch.zeros((2, h, 0, D), dtype=BF, device=dev) for h in (6, 3, 3))
    dc = torch.zeros(2, dtype=torch.int32, device=dev) if counts else None
    len_out, w_out = torch.full_like(lens, -9), torch.full_like(w0, -9.0)
    for weigh in (True, False):
        len_out.fill_(-9), w_out.fill_(-9.0)
        got = ops.paged_attn(q, p, SCALE, kn, vn, counts=dc, weigh=weigh, len_out=len_out, weights_out=w_out if weigh else None)
        assert got.shape == (2, 0, 6, D) and torch.equal(len_out, lens)
        for x in range(6):
            n = int(lens[c.row(x // 3, x % 3)[0]])
            if weigh:
                assert torch.equal(w_out[x, :n], w0[x, :n]) and (w_out[x, n:] == -9.0).all()
    w_out.fill_(-9.0)
    ops.paged_attn(q, p, SCALE, counts=dc, weigh=True, weights_out=w_out)  # of tokens that are stored
    assert all(torch.equal(w_out[x, :n], w0[x, :n]) for x in range(6) for n in [int(lens[c.row(x // 3, x % 3)[0]])])
    ops.paged_attn(q, p, SCALE, kn, vn, counts=dc, weigh=True)             # in place
    len_out.fill_(-9)
    ops.paged_append(kn, vn, p, counts=dc, len_out=len_out)
    assert torch.equal(len_out, lens) and torch.equal(p.row_len, lens) and torch.equal(p.weights, w0) and c.status.item() == 0


def _table(rows, entries, row_pages, dev):
    """A table of -1 but for the rows given."""
    table = torch.full((rows, entries), -1, dtype=torch.int32, device=dev)
    for r, page in row_pages.items():
        table[r] = page
    return table


def _pool(rng, pages, page, dtype, dev):
    return (torch.as_tensor(rng.standard_normal((pages, page, 1, D)), dtype=torch.float32).to(dtype).to(dev) for _ in range(2))


def _i32(a, dev):
    return torch.as_tensor(a, dtype=torch.int32).to(dev)


def test_as_many_columns_as_a_launch_holds_threads(dev):
    """2^20 rows of 16 columns are folded by 2^24 workgroups, 2^32 threads: every 64 rows as in a call of 64."""
    rng = np.random.default_rng(20)
    k, v = _pool(rng, 1, 16, BF, dev)
    q = queries(rng, 64, 16, 1, BF, dev)
    lens = _i32(np.arange(64) % 17, dev)
    want = ops.paged_attn(q, ops.Pages(k, v, torch.zeros((64, 1), dtype=torch.int32, device=dev), lens, 1), SCALE)
    n = 1 << 14
    p = ops.Pages(k, v, torch.zeros((64 * n, 1), dtype=torch.int32, device=dev), lens.repeat(n), 1)
    got = ops.paged_attn(q.repeat(n, 1, 1, 1), p, SCALE)
    assert torch.isfinite(want.float()).all()
    assert all(torch.equal(x.view(-1, 64, 1, 16, D), want.expand(x.shape[0] // 64, -1, -1, -1, -1)) for x in got.split(1 << 16))


def test_as_many_weights_as_a_launch_holds_threads(dev):
    """2^16 rows of wide tables take 2^24 workgroups to weigh in fp32."""
    rng = np.random.default_rng(21)
    T, page, n = 5, 1 << 14, 1 << 10
    k, v = _pool(rng, 1, page, FL, dev)
    q = queries(rng, 64, 4, T, FL, dev)
    lens = _i32(1 + 7 * np.arange(64) % 73, dev)

    def call(times):
        rows = 64 * times
        led = {"weights": torch.zeros((rows, page), device=dev), "pos": torch.zeros((rows, page), dtype=torch.int32, device=dev),
               "dropped": torch.zeros(rows, dtype=torch.int32, device=dev)}
        p = ops.Pages(k, v, torch.zeros((rows, 1), dtype=torch.int32, device=dev), lens.repeat(times), 1, **led)
        return ops.paged_attn(q.repeat(times, 1, 1, 1), p, SCALE, weigh=True), p.weights

    (out, w), (outs, ws) = call(1), call(n)
    assert torch.isfinite(out).all() and (w.sum(1) > 0).all()
    assert torch.equal(outs.view(n, *out.shape), out.expand(n, *out.shape))
    assert torch.equal(ws.view(n, 64, page)[:, :, :128], w[:, :128].expand(n, -1, -1)) and not ws[:, 128:].any()


def test_as_many_rows_as_a_cache_holds(dev):
    """2^24 table rows: an append and an eviction reach the last ones."""
    rng = np.random.default_rng(22)
    rows, page = 1 << 24, 4
    some = {0: 0, 1 << 23: 1, rows - 1: 2}
    k, v = _pool(rng, 4, page, BF, dev)
    table = _table(rows, 1, some, dev)
    row_len, status = torch.zeros(rows, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    led = {"weights": torch.full((rows, page), -1.0, device=dev), "pos": torch.full((rows, page), -1, dtype=torch.int32, device=dev),
           "dropped": torch.zeros(rows, dtype=torch.int32, device=dev)}
    p = ops.Pages(k, v, table, row_len, 1, status=status, **led)
    kn, vn = (queries(rng, 1, 1, page, BF, dev) for _ in range(2))
    counts = torch.zeros(rows, dtype=torch.int32, device=dev)
    counts[list(some)] = page
    ops.paged_append(kn.expand(rows, -1, -1, -1), vn.expand(rows, -1, -1, -1), p, counts=counts)
    assert torch.equal(row_len, counts) and status.item() == 0
    for r, pg in some.items():
        assert torch.equal(k[pg, :, 0], kn[0, 0]) and torch.equal(v[pg, :, 0], vn[0, 0])
        assert p.pos[r].tolist() == [0, 1, 2, 3] and p.weights[r].tolist() == [0.0] * page
        p.weights[r] = torch.tensor([2.0, 1.0, 4.0, 3.0], device=dev)
    ops.paged_evict(p, 2)
    assert torch.equal(row_len, counts // 2) and torch.equal(p.dropped, counts // 2) and status.item() == 0
    for r, pg in some.items():
        assert p.pos[r, :2].tolist() == [2, 3] and p.weights[r, :2].tolist() == [4.0, 3.0]
        assert torch.equal(k[pg, :2, 0], kn[0, 0, 2:]) and torch.equal(v[pg, :2, 0], vn[0, 0, 2:])
