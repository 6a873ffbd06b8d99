"""Attention over a paged cache (ops.paged_append, ops.paged_attn) against its plain 64-bit form."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import _lib, ops
from tests.paged_util import Cache, attend_causal, queries
from tests.serving_util import D, close

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
SCALE = 1 / math.sqrt(D)


def _step(rng, c, G, T, dtype, dev, counts=None, fresh=True, weigh=False):
    """One call on cache c and its checks: outputs, stored tokens, lengths, weights."""
    B, H = c.batch, c.kv_heads
    q = queries(rng, B, H * G, T, dtype, dev)
    kn, vn = queries(rng, B, H, T, dtype, dev), queries(rng, B, H, T, dtype, dev)
    before = c.pages.weights.double().clone() if weigh else None
    dc = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
    got = ops.paged_attn(q, c.pages, SCALE, *((kn, vn) if fresh else (None, None)), counts=dc, weigh=weigh)
    assert got.shape == (B, T, H * G, D)
    lens = c.pages.row_len.tolist()
    for b in range(B):
        n = T if counts is None else min(max(counts[b], 0), T)
        for h in range(H):
            r, _ = c.row(b, h)
            old = int(c.lens[r])
            k, v = c.kv[b * H + h]
            if fresh:
                k, v = torch.cat([k, kn[b, h, :n]]), torch.cat([v, vn[b, h, :n]])
                sk, sv = c.read(b, h, old + n)
                assert torch.equal(sk, k) and torch.equal(sv, v), (b, h)
            assert lens[r] == len(k)
            c.kv[b * H + h] = (k, v)
            heads = slice(h * G, (h + 1) * G)
            out, tol, w, wtol = attend_causal(q[b, heads, :n].transpose(0, 1), k, v, len(k) - n, SCALE, dtype)
            close(got[b, :n, heads], out, tol, f"sequence {b} KV head {h}")
            assert not got[b, n:, heads].any()
            if weigh:
                want = w.clone()
                want[:old] += before[b * H + h, :old]
                if not fresh:
                    want = w + before[b * H + h, :len(k)]
                close(c.pages.weights[b * H + h, :len(k)], want, wtol + 2.0 ** -23 * want, f"weights of {b}, {h}")
                assert torch.equal(c.pages.weights[b * H + h, len(k):].double(), before[b * H + h, len(k):])
                if fresh:
                    pos = np.arange(old, old + n) + int(c.pages.dropped[r])
                    assert c.pages.pos[r, old:old + n].tolist() == pos.tolist()
    for r in range(len(c.lens)):
        c.lens[r] = lens[r]
    assert c.status.item() == 0


CASES = [
    # B, Hkv, G, T, lengths (cycled), page, dtype, apart, order
    (1, 2, 4, 1, [1], 16, BF, False, "token"), (1, 1, 1, 1, [0], 16, BF, True, "token"),
    (3, 2, 4, 1, [5, 32, 0, 64, 31], 16, BF, True, "head"), (2, 4, 7, 1, [333, 18], 64, FP, False, "token"),
    (5, 2, 16, 1, [129, 1], 48, BF, False, "head"), (2, 2, 5, 1, [95, 96], 32, FL, True, "token"),
    (2, 1, 4, 4, [3, 40], 16, FP, False, "token"), (3, 2, 3, 5, [100, 0, 7], 5, BF, True, "token"),
    (2, 2, 8, 2, [257], 1, FL, False, "head"), (70, 2, 4, 1, [20, 33, 1], 256, BF, True, "token"),
    (1, 8, 4, 1, [9000], 16, BF, False, "head"), (2, 2, 2, 8, [5000, 31], 100, FP, True, "token"),
    (1, 2, 4, 5, [0], 16, BF, False, "token"), (2, 2, 4, 33, [8, 100], 64, BF, False, "head"),
    (1, 1, 1, 17, [3], 16, FP, True, "token"), (2, 2, 7, 20, [64, 1], 16, FL, False, "token"),
    (1, 2, 4, 130, [300], 48, BF, True, "token"), (3, 1, 4, 65, [1000, 0, 63], 7, BF, False, "token"),
    (1, 2, 1, 200, [57], 256, FP, False, "head"), (1, 1, 16, 9, [4000], 32, BF, True, "head"),
    (2, 1, 5, 77, [2500, 129], 16, FL, True, "head"), (1, 1, 24, 3, [90], 16, BF, False, "token"),
]


@pytest.mark.parametrize("B,H,G,T,lens,page,dtype,apart,order", CASES)
def test_matches_the_plain_form(dev, B, H, G, T, lens, page, dtype, apart, order):
    """New tokens stored and attended, twice; stale slots hold NaN."""
    rng = np.random.default_rng(B * 100 + T)
    c = Cache(rng, B, H, lens, page, dtype, dev, apart=apart, order=order, room=2 * T)
    _step(rng, c, G, T, dtype, dev)
    _step(rng, c, G, T, dtype, dev)


@pytest.mark.parametrize("B,H,G,T,lens,page,dtype,apart,order", CASES)
def test_accumulates_weights(dev, B, H, G, T, lens, page, dtype, apart, order):
    rng = np.random.default_rng(B * 101 + T)
    c = Cache(rng, B, H, lens, page, dtype, dev, apart=apart, order=order, room=2 * T, ledger=True)
    _step(rng, c, G, T, dtype, dev, weigh=True)
    _step(rng, c, G, T, dtype, dev, weigh=True)


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("T,counts", [(1, [1, 0, 1, 0]), (3, [0, 3, 2, 1]), (40, [0, 1, 40, 17]), (130, [130, 0, 7, 129]),
                                      (4, [-3, 9, 4, 0])])
@pytest.mark.parametrize("fresh", [True, False])
def test_padded_batches(dev, T, counts, fresh, weigh):
    """Counts of each sequence, clamped to 0 .. T; rows shorter than their queries where nothing is appended."""
    rng = np.random.default_rng(T)
    c = Cache(rng, 4, 2, [50, 3, 0, 200], 16, BF, dev, room=T, ledger=True)
    _step(rng, c, 4, T, BF, dev, counts=counts, fresh=fresh, weigh=weigh)


def test_append_alone(dev):
    rng = np.random.default_rng(5)
    for T, dtype, apart in ((1, BF, True), (37, FP, False), (64, FL, True)):
        c = Cache(rng, 3, 2, [5, 0, 31], 16, dtype, dev, apart=apart, room=T, ledger=True)
        kn, vn = queries(rng, 3, 2, T, dtype, dev), queries(rng, 3, 2, T, dtype, dev)
        counts = [T, 0, max(T - 1, 0)]
        ops.paged_append(kn, vn, c.pages, counts=counts)
        for b in range(3):
            for h in range(2):
                r, _ = c.row(b, h)
                n = int(c.lens[r])
                k, v = c.read(b, h, n + counts[b])
                assert torch.equal(k, torch.cat([c.kv[b * 2 + h][0], kn[b, h, :counts[b]]]))
                assert torch.equal(v, torch.cat([c.kv[b * 2 + h][1], vn[b, h, :counts[b]]]))
                assert int(c.pages.row_len[r]) == n + counts[b]
                assert not c.pages.weights[b * 2 + h, n:n + counts[b]].any()
                assert c.pages.pos[r, n:n + counts[b]].tolist() == [n + i + int(c.pages.dropped[r]) for i in range(counts[b])]


@pytest.mark.parametrize("dtype", [BF, FP, FL])
@pytest.mark.parametrize("T,n", [(4, 60), (40, 100)])
def test_values_that_are_no_numbers_reach_those_who_see_them(dev, dtype, T, n):
    """An infinite or NaN key or value of a later token does not reach the queries before it."""
    rng = np.random.default_rng(T)
    for what in ("v", "k"):
        for value in (float("inf"), float("-inf"), float("nan")):
            c = Cache(rng, 1, 1, [n], 16, dtype, dev, room=T)
            q, kn, vn = (queries(rng, 1, h, T, dtype, dev) for h in (4, 1, 1))
            at = T // 2
            (vn if what == "v" else kn)[0, 0, at, 5] = value
            got = ops.paged_attn(q, c.pages, SCALE, kn, vn)
            k, v = torch.cat([c.kv[0][0], kn[0, 0]]), torch.cat([c.kv[0][1], vn[0, 0]])
            out, tol, _, _ = attend_causal(q[0, :, :at].transpose(0, 1), k[:n + at], v[:n + at], n, SCALE, dtype)
            close(got[0, :at], out, tol, f"{what} {value}")
            late = got[0, at:].float()
            if what == "v":
                assert (torch.isnan(late[..., 5]).all() if value != value else (late[..., 5] == value).all())
                keep = [d for d in range(D) if d != 5]
                assert torch.isfinite(late[..., keep]).all()
            elif value != value:
                assert torch.isnan(late).all()
            else:
                # The score is +-inf by the query's sign there: no softmax, or a token of no weight.
                bad = q[0, :, at:, 5].transpose(0, 1).float() * value == float("inf")
                assert torch.isnan(late[bad]).all() and torch.isfinite(late[~bad]).all()


@pytest.mark.parametrize("T", [1, 30])
def test_no_visible_number(dev, T):
    """All scores -inf: NaN, and NaN weights; no token: zeros."""
    rng = np.random.default_rng(3)
    c = Cache(rng, 2, 1, [5, 0], 16, BF, dev, room=T, ledger=True)
    q, kn, vn = (queries(rng, 2, h, T, BF, dev) for h in (4, 1, 1))
    q[0].fill_(1.0)
    kn[0].fill_(float("-inf"))
    for t in range(5):
        pg, sl = c.slots(0, [t])
        c.k[pg, sl, 0] = float("-inf")
    got = ops.paged_attn(q, c.pages, SCALE, kn, vn, weigh=True, counts=[T, 0])
    assert torch.isnan(got[0]).all() and not got[1].any()
    assert torch.isnan(c.pages.weights[0, :5]).all() and torch.isfinite(c.pages.weights[1]).all()


def test_small_weights_behind_a_dominant_token(dev):
    """fp16: a long flat tail e^-17 below one token counts in the product with V as it does in the sum."""
    n = 6000
    for T in (1, 20):
        rng = np.random.default_rng(T)
        c = Cache(rng, 1, 1, [n], 64, FP, dev, room=T)
        q, kn, vn = (queries(rng, 1, h, T, FP, dev) for h in (2, 1, 1))
        q.zero_(), kn.zero_()
        q[..., 0] = 16.0
        pg, sl = c.slots(0, np.arange(n))
        c.k[:] = 0.0
        c.k[pg[:1], sl[:1], 0, 0] = 12.0
        c.v[pg, sl] = 1.0
        vn.fill_(1.0)
        c.v[pg[:1], sl[:1]] = 0.0
        c.kv[0] = (c.k[pg, sl, 0], c.v[pg, sl, 0])
        got = ops.paged_attn(q, c.pages, SCALE, kn, vn)
        k, v = torch.cat([c.kv[0][0], kn[0, 0]]), torch.cat([c.kv[0][1], vn[0, 0]])
        out, tol, _, _ = attend_causal(q[0].transpose(0, 1), k, v, n, SCALE, FP)
        close(got[0], out, tol, f"{T} queries")


def test_rows_without_room(dev):
    """They keep what they hold, attend NaN, and set the status word; the others go on."""
    rng = np.random.default_rng(6)
    for T in (2, 40):
        c = Cache(rng, 3, 2, [60, 64 - T, 63], 16, BF, dev, width=4, room=0, ledger=True, spare=12)
        for r in range(3):  # every entry of the tables names a page
            free = sorted(set(range(c.k.shape[0])) - set(c.table.reshape(-1).tolist()))
            hole = np.nonzero(c.table[r] < 0)[0]
            c.table[r, hole] = free[:len(hole)]
        c.pages.table.copy_(torch.as_tensor(c.table))
        k0, w0 = c.k.clone(), c.pages.weights.clone()
        q, kn, vn = (queries(rng, 3, h, T, BF, dev) for h in (4, 2, 2))
        got = ops.paged_attn(q, c.pages, SCALE, kn, vn, weigh=True)
        full = [64 - T < n for n in (60, 64 - T, 63)]
        assert c.pages.row_len.tolist() == [n + (0 if f else T) for n, f in zip((60, 64 - T, 63), full)]
        for b in range(3):
            assert torch.isnan(got[b]).all() == full[b]
            if full[b]:
                assert torch.equal(c.pages.weights[2 * b:2 * b + 2], w0[2 * b:2 * b + 2])
                pg = torch.as_tensor(c.table[b].astype(np.int64)).to(dev)
                a, z = c.k[pg], k0[pg]
                assert torch.equal(torch.isnan(a), torch.isnan(z)) and torch.equal(a.nan_to_num(), z.nan_to_num())
        with pytest.raises(_lib.HCError, match="capacity"):
            ops.read_status(c.status)


def test_bad_pages(dev):
    """Entries outside of the pool are not followed: NaN for the rows that need them, and the status word."""
    rng = np.random.default_rng(7)
    for T, page in ((1, 16), (1, 24), (40, 16), (40, 24)):
        for value in (-1, 1 << 30, -(1 << 31)):
            c = Cache(rng, 2, 2, [100, 90], page, BF, dev, room=T, ledger=True)
            c.pages.table[1, 2] = value
            q, kn, vn = (queries(rng, 2, h, T, BF, dev) for h in (4, 2, 2))
            got = ops.paged_attn(q, c.pages, SCALE, kn, vn)
            assert torch.isfinite(got[0].float()).all() and torch.isnan(got[1]).all()
            with pytest.raises(_lib.HCError, match="names no page"):
                ops.read_status(c.status)
            ops.paged_evict(c.pages, 20)
            with pytest.raises(_lib.HCError, match="names no page"):
                ops.read_status(c.status)
            assert c.pages.row_len.tolist() == [20, 20]


def test_offsets_past_32_bits(dev):
    """Pools of more than 2^31 elements, read and written at their end."""
    rng = np.random.default_rng(8)
    page, heads = 64, 2
    total = (1 << 31) // (page * heads * D) + 300
    k, v = (torch.empty((total, page, heads, D), dtype=BF, device=dev) for _ in range(2))
    ids = (total - 1 - rng.permutation(200)).astype(np.int32)
    for T in (1, 40):
        n = 500
        table = torch.as_tensor(ids[:10].reshape(1, 10)).to(dev)
        p = ops.Pages(k, v, table, torch.tensor([n], dtype=torch.int32, device=dev), heads)
        rows = torch.as_tensor(ids[:10].astype(np.int64)).to(dev)
        k[rows], v[rows] = (torch.as_tensor(rng.standard_normal((10, page, heads, D)), dtype=torch.float32).to(BF).to(dev)
                            for _ in range(2))
        q, kn, vn = (queries(rng, 1, h, T, BF, dev) for h in (8, 2, 2))
        got = ops.paged_attn(q, p, SCALE, kn, vn)
        for h in range(2):
            kk, vv = (torch.cat([x[rows].reshape(-1, heads, D)[:n, h], y[0, h]]) for x, y in ((k, kn), (v, vn)))
            out, tol, _, _ = attend_causal(q[0, 4 * h:4 * h + 4].transpose(0, 1), kk, vv, n, SCALE, BF)
            close(got[0, :, 4 * h:4 * h + 4], out, tol, f"{T} queries head {h}")
            assert torch.equal(k[rows].reshape(-1, heads, D)[n:n + T, h], kn[0, h])


def test_layouts_outputs_and_lengths_apart(dev):
    """Contiguous [B, H, T, 128] inputs, an output slice of a larger tensor, a table and a ledger that are slices, lengths
    and weights written elsewhere."""
    rng = np.random.default_rng(9)
    for T in (1, 40):
        c = Cache(rng, 2, 2, [70, 33], 16, BF, dev, room=T, ledger=True)
        p = c.pages
        wide = torch.full((2, p.table.shape[1] + 3), -1, dtype=torch.int32, device=dev)
        wide[:, :p.table.shape[1]] = p.table
        ledger = torch.zeros((4, p.capacity + 37), device=dev)
        ledger[:, :p.capacity] = p.weights
        p2 = ops.Pages(c.k, c.v, wide[:, :p.table.shape[1]], p.row_len, 2, weights=ledger[:, :p.capacity], pos=p.pos,
                       dropped=p.dropped)
        q, kn, vn = (queries(rng, 2, h, T, BF, dev).contiguous() for h in (8, 2, 2))
        big = torch.full((2, T + 2, 8, D + 8), 7.0, dtype=BF, device=dev)
        lens, weights = torch.zeros_like(p.row_len), torch.full((4, p.capacity + 37), -1.0, device=dev)[:, :p.capacity]
        got = ops.paged_attn(q, p2, SCALE, kn, vn, out=big[:, 1:T + 1, :, :D], weigh=True, len_out=lens, weights_out=weights)
        want = ops.paged_attn(q, p, SCALE, kn, vn, weigh=True)
        assert torch.equal(got, want)
        assert (big[:, 0] == 7).all() and (big[:, T + 1] == 7).all() and (big[..., D:] == 7).all()
        assert lens.tolist() == p.row_len.tolist() == [70 + T, 33 + T]
        for r, n in ((0, 70 + T), (1, 70 + T), (2, 33 + T), (3, 33 + T)):
            assert torch.equal(weights[r, :n], p.weights[r, :n]) and (weights[r, n:] == -1).all()


def test_repeats_bit_for_bit(dev):
    rng = np.random.default_rng(10)
    for T in (1, 60):
        c = Cache(rng, 3, 2, [700, 20, 333], 16, BF, dev, room=T, ledger=True)
        q, kn, vn = (queries(rng, 3, h, T, BF, dev) for h in (8, 2, 2))
        runs = []
        for _ in range(3):
            w, lens = torch.zeros_like(c.pages.weights), torch.zeros_like(c.pages.row_len)
            runs.append((ops.paged_attn(q, c.pages, SCALE, kn, vn, weigh=True, weights_out=w, len_out=lens), w, lens))
        for x in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(x, runs[0]))


def test_python_refusals(dev):
    rng = np.random.default_rng(11)
    c = Cache(rng, 2, 2, [20], 16, BF, dev, room=4, ledger=True)
    p = c.pages
    q, kn, vn = (queries(rng, 2, h, 1, BF, dev) for h in (4, 2, 2))
    bad = [
        (TypeError, lambda: ops.paged_attn(q.half(), p, SCALE, kn, vn)), (TypeError, lambda: ops.paged_attn(q, p, SCALE, kn.half(), vn)),
        (ValueError, lambda: ops.paged_attn(q, p, SCALE, kn)), (ValueError, lambda: ops.paged_attn(q[:1], p, SCALE, kn, vn)),
        (ValueError, lambda: ops.paged_attn(q[:, :3], p, SCALE, kn, vn)), (ValueError, lambda: ops.paged_attn(q, p, SCALE, kn[:, :1], vn[:, :1])),
        (ValueError, lambda: ops.paged_attn(q, p, SCALE, kn.expand(2, 2, 3, D), vn.expand(2, 2, 3, D))),
        (ValueError, lambda: ops.paged_attn(q.cpu(), p, SCALE)), (ValueError, lambda: ops.paged_attn(q, p, SCALE, weights_out=p.weights)),
        (ValueError, lambda: ops.paged_attn(q, p, SCALE, weigh=True, weights_out=p.weights[:, :5])),
        (ValueError, lambda: ops.paged_attn(q, p, SCALE, kn, vn, counts=[1])), (ValueError, lambda: ops.paged_attn(q, p, SCALE, out=q)),
        (ValueError, lambda: ops.paged_attn(q, p, SCALE, kn, vn, len_out=p.row_len.long())),
        (_lib.HCError, lambda: ops.paged_attn(q, p, 0.0, kn, vn)), (_lib.HCError, lambda: ops.paged_attn(q, p, SCALE, len_out=p.row_len)),
        (ValueError, lambda: ops.paged_append(kn, vn[..., :64], p)), (ValueError, lambda: ops.paged_evict(p, torch.ones(3, dtype=torch.int32, device=dev))),
        (_lib.HCError, lambda: ops.paged_evict(p, 3, sink=2, recent=2)), (ValueError, lambda: ops.paged_evict(p, 8, pos_out=p.pos[:, :4])),
        (ValueError, lambda: ops.Pages(c.k, c.v, p.table, p.row_len, 3)), (ValueError, lambda: ops.Pages(c.k, c.v, p.table.long(), p.row_len, 2)),
        (ValueError, lambda: ops.Pages(c.k, c.v[:, :8], p.table, p.row_len, 2)), (ValueError, lambda: ops.Pages(c.k, c.v, p.table, p.row_len[:1], 2)),
        (ValueError, lambda: ops.Pages(c.k, c.v, p.table, p.row_len, 2, weights=p.weights)),
        (ValueError, lambda: ops.Pages(c.k, c.v, p.table, p.row_len, 2, weights=p.weights[:, :9], pos=p.pos, dropped=p.dropped)),
        (ValueError, lambda: ops.Pages(c.k[:1].expand(9, -1, -1, -1), c.v[:1].expand(9, -1, -1, -1), p.table, p.row_len, 2)),
        (TypeError, lambda: ops.Pages(c.k.double(), c.v.double(), p.table, p.row_len, 2)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("dtype", [BF, FP, FL])
@pytest.mark.parametrize("page,apart,order", [(16, False, "token"), (5, True, "head"), (24, False, "head")])
@pytest.mark.parametrize("fresh", [True, False])
def test_padded_batches_of_other_pages_and_types(dev, dtype, page, apart, order, fresh):
    rng = np.random.default_rng(page)
    c = Cache(rng, 4, 2, [70, 3, 0, 210], page, dtype, dev, apart=apart, order=order, room=40, ledger=True)
    _step(rng, c, 4, 40, dtype, dev, counts=[1, 40, 17, 4], fresh=fresh, weigh=True)


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("page,fresh", [(64, True), (64, False), (20, True)])
def test_padded_batches_over_long_rows(dev, page, fresh, weigh):
    """Chunks with much to do, which are launched apart from the single tokens."""
    rng = np.random.default_rng(page)
    c = Cache(rng, 4, 2, [20000, 30, 0, 7001], page, BF, dev, room=70, ledger=weigh)
    _step(rng, c, 4, 70, BF, dev, counts=[70, 1, 9, 1], fresh=fresh, weigh=weigh)


@pytest.mark.parametrize("counts", [None, "some"])
@pytest.mark.parametrize("T,G", [(2, 8), (9, 3), (40, 4), (3, 24)])
def test_more_rows_than_a_wave_scans_at_once(dev, T, G, counts):
    rng = np.random.default_rng(T)
    B = 45
    c = Cache(rng, B, 2, [0, 40, 3, 17, 90], 16, BF, dev, room=T, ledger=True)
    some = None if counts is None else [int(x) for x in rng.integers(0, T + 1, B)]
    _step(rng, c, G, T, BF, dev, counts=some, weigh=True)


def test_a_long_row_beside_short_ones(dev):
    """One row's keys are cut although there are blocks enough."""
    rng = np.random.default_rng(12)
    c = Cache(rng, 40, 1, [30] * 39 + [30000], 64, BF, dev, room=150)
    _step(rng, c, 8, 150, BF, dev, counts=[150] * 40)


def test_thousands_of_rows(dev):
    rng = np.random.default_rng(13)
    c = Cache(rng, 700, 4, [5, 33, 0], 16, BF, dev, room=2, apart=True, ledger=True)
    _step(rng, c, 2, 1, BF, dev, weigh=True)
    _step(rng, c, 2, 1, BF, dev, counts=[b % 2 for b in range(700)])


@pytest.mark.parametrize("T", [1, 30])
def test_rows_that_share_pages(dev, T):
    """A prefix whose whole pages stand in every sequence's table, each with pages of its own behind it."""
    rng = np.random.default_rng(T)
    c = Cache(rng, 3, 2, [64], 16, BF, dev, room=T, spare=9)
    for b in (1, 2):
        c.pages.table[b, :4] = c.pages.table[0, :4]
        c.table[b, :4] = c.table[0, :4]
        for h in range(2):
            c.kv[b * 2 + h] = c.kv[h]
    _step(rng, c, 4, T, BF, dev)


@pytest.mark.parametrize("n,T", [(100, 9), (20000, 40)])
def test_padded_batches_captured(dev, n, T):
    """A padded chunk with weights, captured once: three replays beside eager calls on a twin, with other counts each."""
    caches = [Cache(np.random.default_rng(1), 3, 2, [n, 5, 60], 16, BF, dev, room=3 * T, ledger=True) for _ in range(2)]
    rng = np.random.default_rng(2)
    new = lambda: [queries(rng, 3, h, T, BF, dev) for h in (8, 2, 2)]
    static, counts = new(), torch.zeros(3, dtype=torch.int32, device=dev)
    ops.paged_attn(static[0], caches[0].pages, SCALE, *static[1:], counts=counts, weigh=True)  # nothing is appended
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.paged_attn(static[0], caches[0].pages, SCALE, *static[1:], counts=counts, weigh=True)
    for some in ([T, 1, 0], [2, T, T], [T, 0, 3]):
        args = new()
        counts.copy_(torch.tensor(some, dtype=torch.int32))
        for x, y in zip(static, args):
            x.copy_(y)
        graph.replay()
        want = ops.paged_attn(args[0], caches[1].pages, SCALE, *args[1:], counts=some, weigh=True)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and caches[0].pages.row_len.tolist() == caches[1].pages.row_len.tolist()
        for r, m in enumerate(caches[1].pages.row_len.tolist()):
            assert torch.equal(caches[0].pages.weights[2 * r:2 * r + 2, :m], caches[1].pages.weights[2 * r:2 * r + 2, :m])
            assert torch.equal(caches[0].pages.pos[r, :m], caches[1].pages.pos[r, :m])


@pytest.mark.parametrize("dtype", [BF, FP, FL])
@pytest.mark.parametrize("T", [1, 20])
def test_infinite_values_that_all_queries_see(dev, dtype, T):
    """An infinite value of an earlier token is the output's channel; the others are as without it."""
    rng = np.random.default_rng(T)
    c = Cache(rng, 1, 1, [300], 16, dtype, dev, room=T)
    pg, sl = c.slots(0, [100, 170])
    c.v[pg[0], sl[0], 0, 3], c.v[pg[1], sl[1], 0, 9] = float("inf"), float("-inf")
    q, kn, vn = (queries(rng, 1, h, T, dtype, dev) for h in (4, 1, 1))
    got = ops.paged_attn(q, c.pages, SCALE, kn, vn)[0]
    k, v = torch.cat([c.kv[0][0], kn[0, 0]]), torch.cat([c.kv[0][1], vn[0, 0]]).clone()
    v[100, 3] = v[170, 9] = 0.0
    out, tol, _, _ = attend_causal(q[0].transpose(0, 1), k, v, 300, SCALE, dtype)
    assert (got[..., 3] == float("inf")).all() and (got[..., 9] == float("-inf")).all()
    rest = [d for d in range(D) if d not in (3, 9)]
    close(got[..., rest], out[..., rest], tol[..., rest], "the other channels")
