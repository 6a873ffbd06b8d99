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
