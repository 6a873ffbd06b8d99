"""The serving operators as they are used: chunks appended with their rotation,
then attended behind a shared prefix or over selected blocks, padded batches,
captured steps, against the plain 64-bit forms."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import ops
from heterocache_amd.store import KVStore
from tests.serving_util import D, attend, bounds, close, rotate, rounding, select, unpack

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
SCALE = 1 / math.sqrt(D)


class Feed:
    """Random new tokens of a batch at given positions."""

    def __init__(self, seed, Hkv, G, dtype, dev):
        self.rng, self.Hkv, self.G, self.dtype, self.dev = np.random.default_rng(seed), Hkv, G, dtype, dev

    def _draw(self, *shape):
        return torch.as_tensor(self.rng.standard_normal(shape), dtype=torch.float32).to(self.dtype).to(self.dev)

    def __call__(self, start, T):
        """start: first position of each sequence.  q, k, v, cos, sin."""
        B = len(start)
        q = self._draw(B, T, self.Hkv * self.G, D).transpose(1, 2)
        k, v = (self._draw(B, T, self.Hkv, D).transpose(1, 2) for _ in range(2))
        pos = torch.as_tensor(start, dtype=torch.float64)[:, None] + torch.arange(T, dtype=torch.float64)
        freq = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
        ang = (pos[..., None] * freq).repeat(1, 1, 2)
        return q, k, v, ang.cos().to(self.dtype).to(self.dev), ang.sin().to(self.dtype).to(self.dev)


def _rows_of(store):
    """(k, v) of each row as stored, in natural order."""
    k, v = unpack(store.k, store.v)
    off, n = (store.row_tile_off * 32).tolist(), store.row_len.tolist()
    return [(k[o:o + m], v[o:o + m]) for o, m in zip(off, n)]


def _append(store, fed, counts=None):
    """append_rotated of fed tokens; checks queries, keys, values, lengths."""
    q, k, v, cos, sin = fed
    before = store.row_len.tolist()
    got = store.append_rotated(q, k, v, cos, sin, counts=counts)
    B, Hkv, T, _ = k.shape
    want, tol = rotate(q, cos, sin)
    close(got, want, tol + rounding(want, q.dtype), "queries")
    want, tol = rotate(k, cos, sin)
    tol = tol + rounding(want, k.dtype)
    for r, (rk, rv) in enumerate(_rows_of(store)):
        b, h = divmod(r, Hkv)
        n = T if counts is None else counts[b]
        assert len(rk) == before[r] + n == int(store.host_len[r]), r
        close(rk[before[r]:], want[b, h, :n], tol[b, h, :n], f"keys of row {r}")
        assert torch.equal(rv[before[r]:], v[b, h, :n]), r
    return got


def _seen(n, T, count, i):
    return min(max(n - count + 1 + i, 0), n)


def _check_shared(out, q, prefix, store, counts=None):
    B, Hq, T, _ = q.shape
    rows, pre = _rows_of(store), _rows_of(prefix) if prefix is not None else None
    kv = store.rows // B
    G = Hq // kv
    for r, (k, v) in enumerate(rows):
        b, h = divmod(r, kv)
        for i in range(T):
            n = _seen(len(k), T, T if counts is None else counts[b], i)
            ks, vs = k[:n], v[:n]
            if pre is not None:
                ks, vs = torch.cat([pre[h][0], ks]), torch.cat([pre[h][1], vs])
            want, tol = attend(q[b, h * G:(h + 1) * G, i], ks, vs, SCALE, q.dtype)
            close(out[b, i, h * G:(h + 1) * G], want, tol, f"row {r} query {i}")


def _check_blocks(got, q, store, block, keep, sink, local, counts=None):
    out, idx, kept = got
    B, Hq, T, _ = q.shape
    kv = store.rows // B
    G = Hq // kv
    for r, (k, v) in enumerate(_rows_of(store)):
        b, h = divmod(r, kv)
        table = bounds(k, block)
        for i in range(T):
            n = _seen(len(k), T, T if counts is None else counts[b], i)
            head = q[b, h * G:(h + 1) * G, i]
            want = select(head, *table, n, block, keep, sink, local)
            assert int(kept[r, i]) == len(want) and np.array_equal(idx[r, i, :len(want)].cpu().numpy(), want), (r, i)
            pos = (want[:, None] * block + np.arange(block)).reshape(-1)
            pos = torch.as_tensor(pos[pos < n], dtype=torch.int64).to(k.device)
            ref, tol = attend(head, k[pos], v[pos], SCALE, q.dtype)
            close(out[b, i, h * G:(h + 1) * G], ref, tol, f"row {r} query {i}")


@pytest.mark.parametrize("Hkv,G,dtype,prefix_chunks,prompt,drafts", [
    (2, 4, BF, [100, 33, 7], [5, 40, 0], [3, 1, 2]), (1, 16, FP, [257], [1, 1, 1], [2, 2, 2]),
    (3, 1, FL, [32, 1], [64, 31, 2], [0, 4, 1]), (2, 7, BF, [], [70, 3, 33], [4, 0, 0]),
])
def test_sequences_behind_a_shared_prompt(dev, Hkv, G, dtype, prefix_chunks, prompt, drafts):
    """A prompt appended in chunks (each attending itself), three sequences behind it: padded own prompts, padded
    drafts, single tokens."""
    feed = Feed(1, Hkv, G, dtype, dev)
    prefix = KVStore([300] * Hkv, dtype, dev)
    at = 0
    for n in prefix_chunks:
        q = _append(prefix, feed([at], n))
        _check_shared(prefix.attend_shared(q, None, SCALE), q, None, prefix)
        at += n
    rows = KVStore([200] * (3 * Hkv), dtype, dev)
    pos = np.full(3, at)
    for counts in (prompt, drafts):
        T = max(counts) + 1  # the last query of every sequence is padding
        q = _append(rows, feed(pos, T), counts)
        _check_shared(rows.attend_shared(q, prefix, SCALE, query_counts=counts), q, prefix, rows, counts)
        on_dev = torch.tensor(counts, dtype=torch.int32, device=dev)
        again = rows.attend_shared(q, prefix, SCALE, query_counts=on_dev)
        _check_shared(again, q, prefix, rows, counts)
        pos = pos + counts
    for _ in range(3):
        q = _append(rows, feed(pos, 1))
        _check_shared(rows.attend_shared(q, prefix, SCALE), q, prefix, rows)
        pos = pos + 1


@pytest.mark.parametrize("Hkv,G,dtype,block,keep,sink,local", [
    (2, 4, BF, 32, 6, 1, 2), (1, 9, FP, 64, 4, 1, 1), (2, 1, FL, 32, 3, 0, 1), (1, 16, BF, 96, 3, 1, 2),
])
def test_blocks_of_growing_rows(dev, Hkv, G, dtype, block, keep, sink, local):
    """Padded prompts, padded drafts and single tokens appended, indexed and attended over their selected blocks."""
    feed = Feed(2, Hkv, G, dtype, dev)
    rows = KVStore([900] * (2 * Hkv), dtype, dev)
    index = rows.block_index(block)
    pos = np.zeros(2, dtype=np.int64)
    for counts in ([400, 63], [300, 0], [2, 5], [0, 3]):
        T = max(counts)
        q = _append(rows, feed(pos, T), counts)
        index.update(T)
        take = q[:, :, -8:] if T > 8 else q  # the last queries (of the shorter sequence: padding)
        n = [min(max(c - (T - take.shape[2]), 0), take.shape[2]) for c in counts]
        got = rows.attend_blocks(take, index, keep, SCALE, sink=sink, local=local, query_counts=n)
        _check_blocks(got, take, rows, block, keep, sink, local, n)
        pos = pos + counts
    for _ in range(2 * block // 8):
        q = feed(pos, 8)
        q = _append(rows, q)
        index.update(8)
        pos = pos + 8
        got = rows.attend_blocks(q[:, :, -1:], index, keep, SCALE, sink=sink, local=local)
        _check_blocks(got, q[:, :, -1:], rows, block, keep, sink, local)
    whole = rows.block_index(block)
    whole.update()
    for r in range(rows.rows):
        a, n = int(index.row_block_off[r]), int(rows.host_len[r]) // block
        assert torch.equal(index.bounds[a:a + n], whole.bounds[a:a + n])
        assert torch.equal(index.exps[a:a + n], whole.exps[a:a + n])


@pytest.mark.parametrize("hkv,g,Q,block,blocks,keep", [
    (2, 4, 1, 32, 100, 8), (2, 4, 3, 32, 100, 8), (1, 12, 1, 32, 100, 8), (2, 4, 1, 32, 600, 8), (1, 4, 1, 64, 200, 150),
    (3, 8, 100, 32, 40, 5),
])
def test_one_call_equals_selection_then_attention(dev, hkv, g, Q, block, blocks, keep):
    """block_step's one launch and its several, beside block_select and block_attn."""
    feed = Feed(3, hkv, g, BF, dev)
    n = block * blocks - 5
    rows = KVStore([n + 9] * hkv, BF, dev)
    q = _append(rows, feed([0], n))[:, :, -Q:]
    index = rows.block_index(block)
    index.update()
    out, idx, counts = rows.attend_blocks(q, index, keep, SCALE)
    idx2, counts2 = ops.block_select(q, index.bounds, index.exps, index.row_block_off, rows.row_len, block,
                                     index.max_blocks, keep, sink=1, local=2)
    assert torch.equal(idx, idx2) and torch.equal(counts, counts2)
    if Q == 1:
        _check_blocks((out, idx, counts), q, rows, block, keep, 1, 2)
    out2 = ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, idx2, counts2, block, SCALE)
    # Both within their bound of the same sum.
    k, v = _rows_of(rows)[0]
    lim = 2 * float(attend(q[0, :g, 0], k, v, SCALE, BF)[1].max()) + 2 ** -8 * float(out2.abs().max())
    assert float((out.float() - out2.float()).abs().max()) <= lim


def test_captured_steps_of_padded_batches(dev):
    """Two graphs, replayed in turn: padded drafts appended with counts on the device, indexed, attended both ways; every
    replay equals the eager calls on a store of its own."""
    Hkv, G, T = 2, 4, 3
    feed = Feed(4, Hkv, G, BF, dev)
    prefix = KVStore([150] * Hkv, BF, dev)
    _append(prefix, feed([0], 150))
    lens = np.array([300, 70])

    def fresh():
        f = Feed(5, Hkv, G, BF, dev)
        s = KVStore([500] * (2 * Hkv), BF, dev)
        _append(s, f([150, 150], 300), lens.tolist())
        ix = s.block_index(32)
        ix.update()
        return s, ix

    def step(s, ix, q, k, v, cos, sin, counts):
        q = ops.append_rotated(q, k, v, cos, sin, s.k, s.v, s.row_tile_off, s.row_len, s.row_cap, counts=counts,
                               len_out=s.row_len, status=s.status)
        ix.update(T)
        out, idx, kept = s.attend_blocks(q, ix, 5, SCALE, query_counts=counts)
        return s.attend_shared(q, prefix, SCALE, query_counts=counts), out, idx, kept

    eager, captured = fresh(), fresh()
    ins = [[t.clone() for t in feed([450, 220], T)] + [torch.ones(2, dtype=torch.int32, device=dev)] for _ in range(2)]
    lengths = captured[0].row_len.clone()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for x in ins:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*captured, *x)
        torch.cuda.current_stream().wait_stream(side)
        captured[0].row_len.copy_(lengths)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*captured, *x))
        graphs.append(g)
    captured[0].row_len.copy_(lengths)
    for turn, counts in enumerate(([3, 1], [0, 2], [1, 3], [2, 0], [3, 3], [1, 1])):
        w = turn % 2
        new = feed((lens + 150).tolist(), T)
        for dst, src in zip(ins[w], list(new) + [torch.tensor(counts, dtype=torch.int32, device=dev)]):
            dst.copy_(src)
        graphs[w].replay()
        want = step(*eager, *[t.clone() for t in ins[w]])
        torch.cuda.synchronize()
        for a, b in zip(outs[w], want):
            assert torch.equal(a, b), turn
        lens = lens + counts
        assert captured[0].row_len.tolist() == np.repeat(lens, Hkv).tolist()
    assert ops.read_status(captured[0].status) == 0


def test_whole_update_in_a_graph_follows_the_rows(dev):
    """update() captured over short rows takes all blocks of the longer ones that its replays find."""
    feed = Feed(6, 1, 4, BF, dev)
    rows = KVStore([700], BF, dev)
    _append(rows, feed([0], 40))
    index = rows.block_index(32)
    index.update()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        index.update()
    for at, n in ((40, 300), (340, 77), (417, 283)):
        _append(rows, feed([at], n))
        index.bounds.zero_()
        g.replay()
        hi, lo, ex = bounds(_rows_of(rows)[0][0], 32)
        assert np.array_equal(index.bounds[:len(ex), 0].cpu().numpy(), hi)
        assert np.array_equal(index.bounds[:len(ex), 1].cpu().numpy(), lo)
        assert np.array_equal(index.exps[:len(ex)].cpu().numpy(), ex)


def test_two_streams_at_once(dev):
    """Calls on two streams over one store share no workspace."""
    feed = Feed(7, 2, 4, BF, dev)
    prefix = KVStore([3000] * 2, BF, dev)
    _append(prefix, feed([0], 3000))
    rows = KVStore([3000] * 8, BF, dev)
    q = _append(rows, feed([3000] * 4, 2500))
    index = rows.block_index(32)
    index.update()
    qs = [q[:, :, -1:].contiguous(), q[:, :, -2:-1].contiguous()]
    want = [(rows.attend_shared(x, prefix, SCALE), rows.attend_blocks(x, index, 70, SCALE)) for x in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [(rows.attend_shared(x, prefix, SCALE, stream=s), rows.attend_blocks(x, index, 70, SCALE, stream=s))
               for x, s in zip(qs, streams)]
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, want):
            assert torch.equal(a, c) and all(torch.equal(x, y) for x, y in zip(b, d))


def test_refusals(dev):
    feed = Feed(8, 2, 4, BF, dev)
    prefix, rows, other = (KVStore([64] * n, BF, dev) for n in (2, 4, 4))
    q, k, v, cos, sin = feed([0, 0], 3)
    index = rows.block_index(32)
    for bad in ([1], [1, 1, 1], torch.ones(3, dtype=torch.int32, device=dev), torch.ones(2, device=dev)):
        with pytest.raises(ValueError, match="query_counts"):
            rows.attend_shared(q, prefix, SCALE, query_counts=bad)
        with pytest.raises(ValueError, match="query_counts"):
            rows.attend_blocks(q, index, 4, SCALE, query_counts=bad)
    for bad in ([4, 0], [-1, 0], [1]):
        with pytest.raises(ValueError, match="counts"):
            rows.append_rotated(q, k, v, cos, sin, counts=bad)
    with pytest.raises(ValueError, match="expanded"):
        rows.attend_shared(q, prefix, SCALE, out=torch.empty((2, 1, 8, D), dtype=BF, device=dev).expand(2, 3, 8, D))
    with pytest.raises(ValueError, match="expanded"):
        rows.append_rotated(q, k, v, cos, sin, out=torch.empty((2, 8, 1, D), dtype=BF, device=dev).expand(2, 8, 3, D))
    with pytest.raises(ValueError, match="rows"):
        ops.shared_attn_stores(q, prefix, rows, 1, SCALE)
    with pytest.raises(ValueError, match="prefix"):
        ops.shared_attn_stores(q, rows, rows, 2, SCALE)
    with pytest.raises(ValueError, match="another store"):
        ops.block_step_store(q, other, index, 4, SCALE)
    mark = torch.zeros(1, device=dev)
    lens = rows.host_len.copy()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mark.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            rows.append_rotated(q, k, v, cos, sin, counts=[1, 2])
        with pytest.raises(RuntimeError, match="captured"):
            rows.attend_shared(q, prefix, SCALE, query_counts=[1, 2])
    g.replay()
    torch.cuda.synchronize()
    assert mark.item() == 1.0 and (rows.host_len == lens).all()


@pytest.mark.parametrize("dtype", [FP, FL])
def test_captured_prefix_of_every_type(dev, dtype):
    """attend_shared captured before the rows grow: replays see the device's lengths."""
    feed = Feed(9, 2, 4, dtype, dev)
    prefix, rows = KVStore([500] * 2, dtype, dev), KVStore([120] * 4, dtype, dev)
    _append(prefix, feed([0], 437))
    q = _append(rows, feed([437] * 2, 9))[:, :, -2:].contiguous()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rows.attend_shared(q, prefix, SCALE)
    for n in (0, 1, 60, 40):
        if n:
            q.copy_(_append(rows, feed([446] * 2, max(n, 2)), [n, n])[:, :, :2])
        g.replay()
        _check_shared(out, q, prefix, rows)
