"""PagedStore: prompts, steps, evictions and sequences that come and go, together as a server runs them."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import _lib, ops
from heterocache_amd.paged import PagedStore
from tests.paged_util import attend_causal, evict_order, queries
from tests.serving_util import D, close

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
SCALE = 1 / math.sqrt(D)


class Plain:
    """What the store should hold: per (sequence, head) keys, values and positions, per table row what was given up."""

    def __init__(self, store):
        self.s = store
        dev = store.device
        self.kv = {(b, h): tuple(torch.zeros((0, D), dtype=store.dtype, device=dev) for _ in range(2))
                   for b in range(store.batch) for h in range(store.kv_heads)}
        self.pos = [[] for _ in range(store.rows)]
        self.dropped = [0] * store.rows

    def row(self, b, h):
        return b * self.s.per_sequence + (h if self.s.per_sequence > 1 else 0)

    def extend(self, out, q, kn, vn, counts, dtype, before):
        """Checks a call's outputs, lengths and weights; the tokens join."""
        s, G = self.s, q.shape[1] // self.s.kv_heads
        for b in range(s.batch):
            n = counts[b]
            for r in range(b * s.per_sequence, (b + 1) * s.per_sequence):
                self.pos[r] += [len(self.pos[r]) + self.dropped[r] + i for i in range(n)]
            for h in range(s.kv_heads):
                k, v = (torch.cat([x, y[b, h, :n]]) for x, y in zip(self.kv[b, h], (kn, vn)))
                self.kv[b, h] = (k, v)
                heads = slice(h * G, (h + 1) * G)
                want, tol, w, wtol = attend_causal(q[b, heads, :n].transpose(0, 1), k, v, len(k) - n, SCALE, dtype)
                close(out[b, :n, heads], want, tol, f"sequence {b} KV head {h}")
                assert not out[b, n:, heads].any()
                if before is not None:
                    x = b * s.kv_heads + h
                    w[:len(k) - n] += before[x, :len(k) - n].double()
                    close(s.pages.weights[x, :len(k)], w, wtol + 2.0 ** -23 * w, f"weights of {b}, {h}")

    def evict(self, keep, sink, recent, weights):
        s = self.s
        hd = s.kv_heads // s.per_sequence
        for r in range(s.rows):
            n = len(self.pos[r])
            w = weights[r * hd:(r + 1) * hd]
            src = evict_order(w, np.asarray(self.pos[r]), n, keep[r], sink, recent, self.dropped[r])
            self.pos[r] = [self.pos[r][i] for i in src]
            self.dropped[r] += n - len(src)
            for h in range(s.kv_heads):
                b = r // s.per_sequence
                if self.row(b, h) == r:
                    at = torch.as_tensor(src).to(s.device)
                    self.kv[b, h] = tuple(x[at] for x in self.kv[b, h])

    def check(self):
        s = self.s
        lens = s.row_len.tolist()
        assert lens == [len(p) for p in self.pos]
        table = s.table.cpu().numpy()
        for (b, h), (k, v) in self.kv.items():
            r = self.row(b, h)
            at = np.arange(len(k))
            pg = torch.as_tensor(table[r, at // s.page_tokens].astype(np.int64)).to(s.device)
            sl = torch.as_tensor(at % s.page_tokens).to(s.device)
            hd = 0 if s.per_sequence > 1 else h
            assert torch.equal(s.k[pg, sl, hd], k) and torch.equal(s.v[pg, sl, hd], v)
        if s.pages.pos is not None:
            for r in range(s.rows):
                assert s.pages.pos[r, :lens[r]].tolist() == self.pos[r] and int(s.pages.dropped[r]) == self.dropped[r]
        # Every page belongs to one row, or is free.
        held = [x for r in range(s.rows) for x in table[r, :s.held[r]].tolist()]
        assert sorted(held + s._free) == list(range(s.k.shape[0]))
        assert all((table[r, s.held[r]:] == -1).all() for r in range(s.rows))


def _new(rng, s, G, T, dtype):
    q = queries(rng, s.batch, s.kv_heads * G, T, dtype, s.device)
    return q, *(queries(rng, s.batch, s.kv_heads, T, dtype, s.device) for _ in range(2))


def _extend(rng, s, plain, G, T, dtype, counts=None, weigh=None):
    q, kn, vn = _new(rng, s, G, T, dtype)
    before = s.pages.weights.clone() if s.pages.weights is not None and weigh is not False else None
    out = s.extend(q, kn, vn, SCALE, counts=counts, weigh=weigh)
    plain.extend(out, q, kn, vn, [T] * s.batch if counts is None else counts, dtype, before)


@pytest.mark.parametrize("dtype,per_head,page,G", [(BF, True, 16, 4), (FP, False, 32, 2), (FL, True, 8, 5), (BF, False, 5, 8)])
def test_prompts_steps_evictions_and_sequences_that_end(dev, dtype, per_head, page, G):
    rng = np.random.default_rng(page)
    s = PagedStore(3, 2, 200 if page > 8 else 500, dtype, dev, max_tokens=160, page_tokens=page, per_head=per_head, track=True)
    plain = Plain(s)
    _extend(rng, s, plain, G, 40, dtype, counts=[40, 17, 0])
    for step in range(3):
        _extend(rng, s, plain, G, 1, dtype)
    keep = [20 + 3 * r for r in range(s.rows)]
    weights = s.pages.weights.cpu().numpy()
    s.evict(keep, sink=2, recent=5)
    plain.evict(keep, 2, 5, weights)
    plain.check()
    _extend(rng, s, plain, G, 9, dtype, counts=[1, 9, 4])       # drafts beside a decode step
    _extend(rng, s, plain, G, 33, dtype, counts=[0, 1, 33])
    weights = s.pages.weights.cpu().numpy()
    s.evict(24, sink=1, recent=8)
    plain.evict([24] * s.rows, 1, 8, weights)
    plain.check()
    s.release([1])
    for h in range(2):
        plain.kv[1, h] = tuple(x[:0] for x in plain.kv[1, h])
    for r in range(s.per_sequence, 2 * s.per_sequence):
        plain.pos[r], plain.dropped[r] = [], 0
    plain.check()
    _extend(rng, s, plain, G, 50, dtype, counts=[2, 50, 1])
    plain.check()
    assert s.attend(_new(rng, s, G, 1, dtype)[0], SCALE).shape == (3, 1, 2 * G, D)
    s.check_status()
    assert (s.host_len == s.row_len.cpu().numpy()).all()


def test_append_beside_another_attention_and_no_ledger(dev):
    """A prompt that ops.prefill_attn attends, stored, and the steps behind it."""
    rng = np.random.default_rng(3)
    s = PagedStore(2, 2, 60, BF, dev, max_tokens=300, page_tokens=16)
    plain = Plain(s)
    q, kn, vn = _new(rng, s, 4, 70, BF)
    out = ops.prefill_attn(q, kn, vn, SCALE)
    s.append(kn, vn)
    plain.extend(out, q, kn, vn, [70, 70], BF, None)
    again = s.attend(q, SCALE)
    fresh = Plain(s)
    fresh.extend(again, q, kn, vn, [70, 70], BF, None)
    for _ in range(2):
        _extend(rng, s, plain, 4, 1, BF)
    plain.check()
    with pytest.raises(ValueError, match="no weights"):
        s.evict(8)


def test_refusals(dev):
    rng = np.random.default_rng(4)
    s = PagedStore(2, 2, 4, BF, dev, max_tokens=48, page_tokens=16, track=True, layer_idx=7)
    q, kn, vn = _new(rng, s, 2, 33, BF)
    with pytest.raises(RuntimeError, match="Layer 7 OOM"):
        s.extend(q, kn, vn, SCALE)                      # six pages of four
    assert s.free_pages == 4 and not s.host_len.any()
    s.extend(q, kn, vn, SCALE, counts=[33, 1])
    with pytest.raises(RuntimeError, match="OOM"):
        s.reserve([16, 0])                              # past max_tokens
    for bad in ([34, 0], [-1, 0], [1]):
        with pytest.raises(ValueError):
            s.append(kn, vn, counts=bad)
    with pytest.raises(ValueError):
        s.evict(4, sink=3, recent=2)
    with pytest.raises(ValueError):
        s.release([2])
    with pytest.raises(RuntimeError):
        s.sync_host_lengths([64, 1])
    for kw in (dict(pages=0), dict(max_tokens=0), dict(page_tokens=0)):
        with pytest.raises(ValueError):
            PagedStore(**{**dict(batch=1, kv_heads=1, pages=1, dtype=BF, device=dev, max_tokens=16), **kw})
    s.check_status()


def test_captured_steps(dev):
    """A step with its eviction captured once and replayed between eager work, against an eager twin."""
    rng = np.random.default_rng(5)
    stores = [PagedStore(2, 2, 120, BF, dev, max_tokens=128, page_tokens=16, per_head=True, track=True) for _ in range(2)]
    first = [_new(np.random.default_rng(6), s, 4, 40, BF) for s in stores]
    for s, (q, kn, vn) in zip(stores, first):
        s.extend(q, kn, vn, SCALE, counts=[40, 30])
        s.reserve(8)
    a, b = stores
    q, kn, vn = (torch.empty_like(x) for x in _new(rng, a, 4, 1, BF))
    counts = torch.ones(2, dtype=torch.int32, device=dev)

    def step(s, args):
        out = s.extend(*args, SCALE, counts=counts)
        s.evict(36, sink=2, recent=6)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    held = a.held.copy()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(a, (q, kn, vn))
    torch.cuda.current_stream().wait_stream(side)
    assert (a.held == held).all()
    for i in range(6):
        args = _new(rng, a, 4, 1, BF)
        counts.copy_(torch.tensor([1, i % 2], dtype=torch.int32))
        for x, y in zip((q, kn, vn), args):
            x.copy_(y)
        graph.replay()
        want = step(b, args)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        n = b.row_len.tolist()
        assert a.row_len.tolist() == n
        for r, m in enumerate(n):
            assert torch.equal(a.pages.weights[r, :m], b.pages.weights[r, :m])
            assert torch.equal(a.pages.pos[r, :m], b.pages.pos[r, :m])
    a.sync_host_lengths(a.row_len.cpu().numpy())
    a.check_status()
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="reserved before"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                a.extend(*_static(rng, a, 100), SCALE)


def _static(rng, s, T):
    z = lambda h: torch.zeros((s.batch, h, T, D), dtype=s.dtype, device=s.device)
    return z(s.kv_heads * 4), z(s.kv_heads), z(s.kv_heads)


def test_replays_past_the_reserved_pages_are_told(dev):
    """A replay that outgrows its pages touches no other row's: NaN out, and an error from the status word."""
    s = PagedStore(1, 1, 10, BF, dev, max_tokens=64, page_tokens=16)
    rng = np.random.default_rng(8)
    args = _new(rng, s, 4, 1, BF)
    s.extend(*_new(rng, s, 4, 15, BF), SCALE)
    pool = s.k.clone()
    for i in range(3):
        out = ops.paged_attn(args[0], s.pages, SCALE, args[1], args[2])  # behind the host's back
    assert torch.isnan(out.float()).all()
    at = int(s.table[0, 0])
    pool[at, 15] = args[1][0, :, 0]
    assert torch.equal(s.k, pool)
    with pytest.raises(_lib.HCError, match="names no page"):
        s.check_status()
    s.check_status()


def test_two_streams(dev):
    """Two stores at work on two streams at once."""
    rng = np.random.default_rng(9)
    stores = [PagedStore(2, 2, 100, BF, dev, max_tokens=400, page_tokens=32, track=True) for _ in range(2)]
    plains = [Plain(s) for s in stores]
    streams = [torch.cuda.Stream() for _ in stores]
    calls = []
    for T in (120, 1, 30, 1):
        args = [_new(rng, s, 4, T, BF) for s in stores]
        torch.cuda.synchronize()
        before = [s.pages.weights.clone() for s in stores]
        torch.cuda.synchronize()
        outs = [s.extend(*x, SCALE, stream=st) for s, x, st in zip(stores, args, streams)]
        torch.cuda.synchronize()
        for s, p, o, x, w in zip(stores, plains, outs, args, before):
            p.extend(o, *x, [T, T], BF, w)
    for p in plains:
        p.check()


def test_an_eviction_that_is_captured_and_not_replayed(dev):
    """Capturing runs nothing: the rows keep their tokens, and what the host knows of them still bounds their lengths."""
    rng = np.random.default_rng(10)
    s = PagedStore(2, 2, 60, BF, dev, max_tokens=128, page_tokens=16, per_head=True, track=True)
    plain = Plain(s)
    _extend(rng, s, plain, 4, 32, BF)                        # full pages
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            s.evict(20, sink=2, recent=6)
    torch.cuda.current_stream().wait_stream(side)
    assert (s.host_len >= s.row_len.cpu().numpy()).all()
    _extend(rng, s, plain, 4, 1, BF)                         # into a page that is not reserved yet
    plain.check()
    s.check_status()
    weights = s.pages.weights.cpu().numpy()
    graph.replay()
    plain.evict([20] * s.rows, 2, 6, weights)
    torch.cuda.synchronize()
    s.sync_host_lengths(s.row_len.cpu().numpy())
    plain.check()
    _extend(rng, s, plain, 4, 5, BF)
    weights = s.pages.weights.cpu().numpy()
    s.evict(9, sink=2, recent=6)                             # the pages behind come back now
    plain.evict([9] * s.rows, 2, 6, weights)
    plain.check()
    assert (s.held == 1).all()


def test_steps_and_evictions_in_one_graph(dev):
    """A graph of more steps than its evictions leave pages for: what the first replay needs is known along the graph,
    while the host's bound holds for the rows as they are before it."""
    rng = np.random.default_rng(11)
    s = PagedStore(1, 2, 40, BF, dev, max_tokens=64, page_tokens=4, per_head=True, track=True)
    plain = Plain(s)
    _extend(rng, s, plain, 4, 32, BF)
    s.reserve(1)                                             # room for 36 tokens a row, and the graph appends 6
    args = [_new(rng, s, 4, 1, BF) for _ in range(6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph, outs, before = torch.cuda.CUDAGraph(), [], []
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            for a in args:
                before.append(s.pages.weights.clone())
                outs.append((s.extend(*a, SCALE), s.pages.weights.clone()))
                s.evict(32, sink=1, recent=4)
    torch.cuda.current_stream().wait_stream(side)
    assert (s.host_len >= 32).all() and (s.host_len <= 36).all()
    for _ in range(3):                                       # the graph runs when it is replayed, not before
        _extend(rng, s, plain, 4, 1, BF)
    weights = s.pages.weights.cpu().numpy()
    s.evict(32, sink=1, recent=4)
    plain.evict([32] * s.rows, 1, 4, weights)
    s.reserve(1)
    graph.replay()
    torch.cuda.synchronize()
    kept = s.pages.weights
    for a, b, (out, w) in zip(args, before, outs):
        kept.copy_(w)                                        # (as it was behind the step, for its check)
        plain.extend(out, *a, [1], BF, b)
        plain.evict([32] * s.rows, 1, 4, w.cpu().numpy())
    s.sync_host_lengths(s.row_len.cpu().numpy())
    plain.check()
    s.check_status()
