"""Eviction from a paged cache by accumulated weight (ops.paged_evict): exact against its plain form."""
import numpy as np
import pytest
import torch

from heterocache_amd import ops
from tests.paged_util import Cache, evict_order

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32


def _evict(c, keep, sink, recent, apart_outputs=False):
    """One eviction of cache c, checked slot by slot; keep: an integer or one a row."""
    p = c.pages
    w, pos, dropped = p.weights.cpu().numpy().copy(), p.pos.cpu().numpy().copy(), p.dropped.cpu().numpy().copy()
    lens = p.row_len.cpu().numpy().astype(int)
    old = {(b, h): c.read(b, h, int(lens[c.row(b, h)[0]])) for b in range(c.batch) for h in range(c.kv_heads)}
    arg = keep if isinstance(keep, int) else torch.tensor(keep, dtype=torch.int32, device=c.k.device)
    res = {}
    if apart_outputs:
        res = {"len_out": torch.full_like(p.row_len, -9), "weights_out": torch.full_like(p.weights, -9.0),
               "pos_out": torch.full_like(p.pos, -9), "dropped_out": torch.full_like(p.dropped, -9)}
    ops.paged_evict(p, arg, sink=sink, recent=recent, **res)
    new_len, new_w, new_pos, new_dropped = (res.get(x + "_out", t) for x, t in (
        ("len", p.row_len), ("weights", p.weights), ("pos", p.pos), ("dropped", p.dropped)))
    if apart_outputs:
        assert np.array_equal(p.weights.cpu().numpy(), w, equal_nan=True) and np.array_equal(p.pos.cpu().numpy(), pos)
        assert p.row_len.tolist() == lens.tolist() and p.dropped.tolist() == dropped.tolist()
    hd = c.heads
    for r, n in enumerate(lens.tolist()):
        k_r = keep if isinstance(keep, int) else keep[r]
        m = min(n, k_r)
        assert int(new_len[r]) == m and int(new_dropped[r]) == dropped[r] + n - m
        src = evict_order(w[r * hd:(r + 1) * hd], pos[r], n, k_r, sink, recent, int(dropped[r]))
        assert new_pos[r, :m].tolist() == pos[r, src].tolist()
        got = new_w[r * hd:(r + 1) * hd, :m].cpu().numpy()
        assert np.array_equal(got, w[r * hd:(r + 1) * hd][:, src], equal_nan=True)
        behind = -9 if apart_outputs else pos[r, m:]
        assert (new_pos[r, m:].cpu().numpy() == behind).all()
    for (b, h), (k, v) in old.items():
        r, _ = c.row(b, h)
        k_r = keep if isinstance(keep, int) else keep[r]
        src = evict_order(w[r * hd:(r + 1) * hd], pos[r], int(lens[r]), k_r, sink, recent, int(dropped[r]))
        gk, gv = c.read(b, h, len(src))
        src = torch.as_tensor(src).to(k.device)
        assert torch.equal(gk, k[src]) and torch.equal(gv, v[src])
    assert c.status.item() == 0
    c.lens = new_len.cpu().numpy().astype(np.int64)


CASES = [
    # B, Hkv, lengths (cycled), keep, sink, recent, page, dtype, apart, order
    (1, 2, [40, 33], 32, 4, 8, 16, BF, True, "token"), (2, 2, [64], 63, 0, 0, 16, FP, True, "head"),
    (2, 4, [100, 7, 0], 50, 2, 10, 48, BF, False, "token"), (1, 1, [1], 0, 0, 0, 16, BF, True, "token"),
    (3, 2, [1000, 513, 64], 64, 4, 60, 256, FL, True, "head"), (1, 1, [5000], 4999, 4, 100, 16, BF, True, "token"),
    (2, 3, [4097, 300], 2000, 0, 500, 100, BF, False, "head"), (1, 2, [20000, 17000], 1000, 16, 200, 64, FP, True, "token"),
    (1, 2, [70, 65], 1, 0, 1, 7, BF, True, "token"), (1, 1, [12000], 11990, 4, 32, 1, FL, True, "head"),
    (1, 2, [1024, 1025], 1024, 4, 32, 16, BF, True, "token"), (1, 5, [2300], 700, 8, 0, 32, BF, False, "token"),
]


@pytest.mark.parametrize("apart_outputs", [False, True])
@pytest.mark.parametrize("B,H,lens,keep,sink,recent,page,dtype,apart,order", CASES)
def test_keeps_the_heaviest(dev, B, H, lens, keep, sink, recent, page, dtype, apart, order, apart_outputs):
    rng = np.random.default_rng(len(lens) * 7 + keep)
    c = Cache(rng, B, H, lens, page, dtype, dev, apart=apart, order=order, ledger=True)
    _evict(c, keep, sink, recent, apart_outputs)
    if not apart_outputs:
        _evict(c, keep // 2 + (sink + recent) // 2 + 1 if keep else 0, sink // 2, recent // 2)


def test_budgets_a_row_and_more_protected_than_kept(dev):
    rng = np.random.default_rng(1)
    c = Cache(rng, 2, 3, [90, 50, 10, 64, 33, 0], 16, BF, dev, apart=True, ledger=True)
    _evict(c, [30, 50, 12, 0, 1, 5], 3, 4)  # rows of fewer kept than protected: the lower slots of these


def test_ties_infinities_and_nan(dev):
    """Equal weights go to the lower slots; NaN ranks below everything, also below -inf; protected above inf."""
    rng = np.random.default_rng(2)
    for value in (0.0, 1.5, float("inf")):
        c = Cache(rng, 1, 2, [300], 16, BF, dev, apart=True, ledger=True)
        c.pages.weights.fill_(value)
        _evict(c, 200, 4, 20)
    c = Cache(rng, 1, 2, [3000, 200], 16, BF, dev, apart=True, ledger=True)
    w = torch.as_tensor(rng.choice([0.0, -0.0, 1.0, float("inf"), float("-inf"), float("nan"), 1e-40, 3e38], c.pages.weights.shape),
                        dtype=torch.float32)
    c.pages.weights.copy_(w)
    _evict(c, 150, 2, 30)
    c = Cache(rng, 1, 4, [500], 16, BF, dev, apart=False, ledger=True)
    c.pages.weights.copy_(torch.as_tensor(rng.choice([0.25, 0.5, 2.0 ** -30], c.pages.weights.shape), dtype=torch.float32))
    _evict(c, 333, 0, 16)


@pytest.mark.parametrize("apart", [True, False])
def test_long_tables(dev, apart):
    """Tables of more than 16384 tokens: short rows among long ones, sums over heads, every weight equal, nothing kept."""
    rng = np.random.default_rng(3)
    heads = 2
    lens = [20000, 500, 17001, 0] if apart else [18000, 40]
    c = Cache(rng, 2, heads, lens, 64, BF, dev, apart=apart, ledger=True)
    keep = [15000, 1000, 0, 7] if apart else [900, 39]
    _evict(c, keep, 0, 0, apart_outputs=True)
    _evict(c, keep, 0, 0)
    for value in (0.0, 3.5):
        c = Cache(rng, 1, heads, [18000], 256, FP, dev, apart=apart, ledger=True)
        c.pages.weights.fill_(value)
        _evict(c, 7000, 4, 300)
        _evict(c, 6999, 4, 300)
    c = Cache(rng, 1, heads, [50], 64, FP, dev, apart=apart, ledger=True, width=400)  # little in a large table
    _evict(c, 33, 2, 9)


def test_many_rows(dev):
    rng = np.random.default_rng(4)
    c = Cache(rng, 700, 4, [20, 33, 7], 16, BF, dev, apart=True, ledger=True)
    _evict(c, 16, 1, 4)


def test_counters_past_32_bits(dev):
    """Long table rows with more than 2^31 counters: the rows at both ends are evicted from, the others are
    empty."""
    rows, cap, n, keep = (1 << 19) + 5, 16385, 16384, 9000
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 210 * 10 ** 9:
        pytest.skip("needs 182 GB of free device memory")
    rng = np.random.default_rng(5)
    k, v = (torch.as_tensor(rng.standard_normal((2, cap, 1, 128)), dtype=torch.float32).to(BF).to(dev) for _ in range(2))
    table = torch.full((rows, 1), -1, dtype=torch.int32, device=dev)
    row_len, dropped, status = (torch.zeros(x, dtype=torch.int32, device=dev) for x in (rows, rows, 1))
    weights, pos = (torch.empty((rows, cap), dtype=t, device=dev) for t in (FL, torch.int32))
    want = {}
    for r, page in ((0, 0), (rows - 1, 1)):
        table[r, 0], row_len[r] = page, n
        w = rng.exponential(size=(1, cap)).astype(np.float32)
        weights[r], pos[r] = torch.as_tensor(w[0]).to(dev), torch.arange(cap, dtype=torch.int32, device=dev)
        src = evict_order(w, np.arange(cap), n, keep, 4, 100, 0)
        want[r] = [src, k[page, :n, 0].cpu()[src], v[page, :n, 0].cpu()[src], w[0, src]]
    p = ops.Pages(k, v, table, row_len, 1, weights=weights, pos=pos, dropped=dropped, status=status)
    ops.paged_evict(p, keep, sink=4, recent=100)
    for r, page in ((0, 0), (rows - 1, 1)):
        src, wk, wv, ww = want[r]
        assert int(row_len[r]) == keep and int(dropped[r]) == n - keep
        assert pos[r, :keep].tolist() == src.tolist() and np.array_equal(weights[r, :keep].cpu().numpy(), ww)
        assert torch.equal(k[page, :keep, 0].cpu(), wk) and torch.equal(v[page, :keep, 0].cpu(), wv)
    assert int(row_len.sum()) == 2 * keep and status.item() == 0
    del weights, pos, p
    torch.cuda.empty_cache()
