"""The serving operators where their arithmetic has nothing ordinary to fold: scores without a number, weights far below
the largest, lengths that only the device knows."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import ops
from tests.serving_util import D, attend, bounds, close, make_rows

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
SCALE = 1 / math.sqrt(D)


def _q(rng, B, Hq, Q, dtype, dev):
    q = torch.as_tensor(rng.standard_normal((B, Q, Hq, D)), dtype=torch.float32)
    return q.to(dtype).to(dev).transpose(1, 2)


def _meta(s):
    return s.k, s.v, s.row_tile_off, s.row_len


def _every_way(q, prefix, rows, scale=SCALE):
    """(name, output, tokens of row 0's KV head from) of each way to attend all of a row or prefix: one workgroup a
    row, split rows, few and many prefix parts, both, all blocks in one launch and split."""
    index = rows.block_index(32)
    index.update()
    keep = index.max_blocks
    idx, counts = ops.block_select(q, index.bounds, index.exps, index.row_block_off, rows.row_len, 32, keep, keep)
    kv = prefix.rows
    return [
        ("rows", ops.shared_attn(q, None, _meta(rows), kv, scale, row_tiles=1), False, True),
        ("split rows", ops.shared_attn(q, None, _meta(rows), kv, scale, row_tiles=64), False, True),
        ("prefix", ops.shared_attn(q, _meta(prefix), None, kv, scale, prefix_tiles=0), True, False),
        ("parts", ops.shared_attn(q, _meta(prefix), None, kv, scale, prefix_tiles=64), True, False),
        ("both", rows.attend_shared(q, prefix, scale), True, True),
        ("step", rows.attend_blocks(q, index, keep, scale)[0], False, True),
        ("listed", ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, idx, counts, 32, scale), False,
         True),
    ]


def _cat(pre, own, use_pre, use_own):
    """Keys and values of a row as one way attends them."""
    parts = ([pre] if use_pre else []) + ([own] if use_own else [])
    return torch.cat([k for k, _ in parts]), torch.cat([v for _, v in parts])


@pytest.mark.parametrize("dtype", [BF, FP, FL])
@pytest.mark.parametrize("n", [5, 700])
def test_nan_queries_give_nan(dev, dtype, n):
    """A query with a NaN has no finite score: its output is NaN, not the zeros of a query that sees nothing; the
    other heads of its group keep their results."""
    rng = np.random.default_rng(n)
    prefix, pre = make_rows(rng, [n, n + 1], dtype, dev)
    rows, kv = make_rows(rng, [n + 2, n, 3, n + 70], dtype, dev, room=6)
    q = _q(rng, 2, 8, 1, dtype, dev).contiguous()
    q[0, 1] = math.nan
    q[1, 6, 0, 77] = math.nan
    for name, out, use_pre, use_own in _every_way(q, prefix, rows):
        for b in range(2):
            for h in range(8):
                if (b, h) in ((0, 1), (1, 6)):
                    assert torch.isnan(out[b, 0, h]).all(), (name, b, h)
                    continue
                want, tol = attend(q[b, h, 0], *_cat(pre[h // 4], kv[2 * b + h // 4], use_pre, use_own), SCALE, dtype)
                close(out[b, 0, h], want, tol, f"{name} {b} {h}")


@pytest.mark.parametrize("dtype", [BF, FP, FL])
def test_scores_of_minus_infinity(dev, dtype):
    """Tokens that score -inf weigh nothing beside others; a query that sees only such tokens has no softmax (NaN); one
    that sees no token gets zeros."""
    rng = np.random.default_rng(3)
    prefix, pre = make_rows(rng, [300, 90], dtype, dev)
    rows, kv = make_rows(rng, [400, 0, 200, 64], dtype, dev, room=6)
    q = _q(rng, 2, 2, 1, dtype, dev).abs().contiguous()
    for r, cut in ((0, 300), (2, 200), (3, 0)):  # (3: every token -inf but the last ten of its first tile)
        k, v = kv[r]
        if r == 3:
            k[:22, 5] = k[32:, 5] = -math.inf
        else:
            k[:cut, 5] = -math.inf
        rows.write_rows(k[None, None], v[None, None], [(0, 0)], [r], [len(k)])
    for name, out, use_pre, use_own in _every_way(q, prefix, rows):
        for r in range(4):
            b, h = divmod(r, 2)
            k, v = _cat(pre[h], kv[r], use_pre, use_own)
            live = torch.isfinite(k[:, 5])
            if len(k) and not live.any():
                assert torch.isnan(out[b, 0, h]).all(), (name, r)
                continue
            want, tol = attend(q[b, h, 0], k[live], v[live], SCALE, dtype)
            close(out[b, 0, h], want, tol, f"{name} row {r}")
            if len(k) == 0:
                assert not out[b, 0, h].any(), (name, r)


def test_whole_update_after_replayed_appends(dev):
    """Captured appends advance the lengths on the device and not the host's mirror: an update() outside of the graph, on
    the current stream or on another, still takes every complete block."""
    rng = np.random.default_rng(4)
    rows, kv = make_rows(rng, [40, 95, 0], BF, dev, room=400, stale=0.0)
    index = rows.block_index(32)
    T = 50
    q, k, v = (torch.zeros((1, 3, T, D), dtype=BF, device=dev) for _ in range(3))
    one, zero = torch.ones((T, D), device=dev), torch.zeros((T, D), device=dev)
    ops.append_rotated(q, k, v, one, zero, *_meta(rows), rows.row_cap)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.append_rotated(q, k, v, one, zero, *_meta(rows), rows.row_cap, len_out=rows.row_len)
    side = torch.cuda.Stream(dev)
    for step in range(4):
        for t in (k, v):
            t.copy_(torch.as_tensor(rng.standard_normal(t.shape), dtype=torch.float32))
        kv = [(torch.cat([a, k[0, r]]), torch.cat([b, v[0, r]])) for r, (a, b) in enumerate(kv)]
        g.replay()
        index.bounds.fill_(5)
        index.exps.fill_(77)
        if step % 2:
            side.wait_stream(torch.cuda.current_stream(dev))
            index.update(stream=side)
            torch.cuda.current_stream(dev).wait_stream(side)
        else:
            index.update()
        assert rows.host_len.tolist() == [40, 95, 0]
        off = index.row_block_off.tolist()
        for r, (a, _) in enumerate(kv):
            hi, lo, ex = bounds(a, 32)
            got = index.bounds[off[r]:off[r] + len(ex)].cpu().numpy()
            assert np.array_equal(got[:, 0], hi) and np.array_equal(got[:, 1], lo), (step, r)
            assert np.array_equal(index.exps[off[r]:off[r] + len(ex)].cpu().numpy(), ex), (step, r)


@pytest.mark.parametrize("dtype", [BF, FP, FL])
@pytest.mark.parametrize("drop", [9.0, 17.4, 20.0, 24.0])
def test_flat_tail_behind_a_dominant_token(dev, dtype, drop):
    """One token whose value is zero outweighs each of the others by e^drop: the output is what they weigh together."""
    rng = np.random.default_rng(5)
    n = 6000
    prefix, rows = (make_rows(rng, [n], dtype, dev, room=3)[0] for _ in range(2))
    k = torch.zeros((n, D), dtype=dtype, device=dev)
    v = (1 + 0.25 * torch.as_tensor(rng.random((n, D)), dtype=torch.float32)).to(dtype).to(dev)
    q = torch.zeros((1, 1, 1, D), dtype=dtype, device=dev)
    q[..., 0] = 16.0
    k[3, 0], v[3] = drop / SCALE / 16, 0.0
    for store in (prefix, rows):
        store.write_rows(k[None, None], v[None, None], [(0, 0)], [0], [n])
    # Scores are one exact product each.  An exponent is off by 4 roundings of a
    # number up to 1.45 drop + 10, exp2 by 2 steps; a weight's rounding to the input type
    # is half a step, in fp16 (whose smallest steps are 2^-24, the greatest weight 2^10 or
    # more) at least 2^-35 of the greatest; sums of n terms.
    for name, out, use_pre, use_own in _every_way(q, prefix, rows):
        copies = int(use_pre) + int(use_own)
        s = (q[0, 0].double() @ k.double().t() * SCALE)[0]
        w = torch.exp(s - s.max())
        mass = copies * w.sum()
        want = copies * (w @ v.double()) / mass
        slip = 2.0 ** -24 * (4 * (1.45 * drop + 10) * math.log(2) + 4 + 2 * copies * n + 64)
        step = w * torch.finfo(dtype).eps / 2
        if dtype == FP:
            step = step.clamp(min=2.0 ** -35)
        tol = copies * (step @ v.double().abs()) / mass + 2 * slip * want + want * torch.finfo(dtype).eps / 2 * 1.01
        close(out[0, 0, 0], want, tol * 1.02 + torch.finfo(dtype).tiny * torch.finfo(dtype).eps, f"{name} e^-{drop}")


@pytest.mark.parametrize("dtype", [BF, FP, FL])
@pytest.mark.parametrize("size", [64.0, 700.0, 1024.0, 2048.0])
def test_scores_far_beyond_the_exponent(dev, dtype, size):
    """Scores up to 2^26, whose steps in fp32 are several powers of two: the best token's value comes out."""
    rng = np.random.default_rng(6)
    n = 300
    prefix, rows = (make_rows(rng, [n], dtype, dev, room=3)[0] for _ in range(2))
    sign = torch.as_tensor(rng.choice([-1.0, 1.0], (n, D)), dtype=torch.float32).to(dev)
    v = torch.as_tensor(rng.standard_normal((n, D)), dtype=torch.float32).to(dtype).to(dev)
    k = (sign * size).to(dtype)
    q = k[170].clone().view(1, 1, 1, D)
    for store in (prefix, rows):
        store.write_rows(k[None, None], v[None, None], [(0, 0)], [0], [n])
    want = v[170].double()
    # The others are e^-1000 or less of it.  Its weight is off by half a step of the type, the output by another.
    tol = want.abs() * (torch.finfo(dtype).eps * 1.01 + 64 * 2.0 ** -24)
    for name, out, _, _ in _every_way(q, prefix, rows):
        close(out[0, 0, 0], want, tol, name)


def test_room_without_end(dev):
    """Tile counts and max_blocks of the types' largest values: nothing more is read or kept than of fitting ones."""
    rng = np.random.default_rng(7)
    prefix, pre = make_rows(rng, [700], BF, dev)
    rows, kv = make_rows(rng, [900], BF, dev, room=5)
    q = _q(rng, 1, 4, 1, BF, dev)
    most = (1 << 63) - 1
    for pt, rt in ((most, 30), (22, most), (most, most)):
        got = ops.shared_attn(q, _meta(prefix), _meta(rows), 1, SCALE, prefix_tiles=pt, row_tiles=rt)
        for h in range(4):
            want, tol = attend(q[0, h, 0], *_cat(pre[0], kv[0], True, True), SCALE, BF)
            close(got[0, 0, h], want, tol, f"{pt} {rt}")
    index = rows.block_index(32)
    index.update()
    a, b = (ops.block_select(q, index.bounds, index.exps, index.row_block_off, rows.row_len, 32, n, 9, 1, 2)
            for n in (index.max_blocks, (1 << 31) - 1))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("B,Hkv,G,Q,lens,dtype", [(1, 2, 4, 300, [500, 300], BF), (2, 1, 16, 70, [90, 70], FP),
                                                 (1, 1, 5, 129, [129], FL), (2, 2, 3, 33, [4000, 2, 33, 600], BF)])
def test_chunks_of_queries_over_their_own_rows(dev, B, Hkv, G, Q, lens, dtype):
    """A chunk that attends itself, without a prefix: into a view, without partials where the rows are not split."""
    rng = np.random.default_rng(Q)
    rows, kv = make_rows(rng, lens, dtype, dev, room=4)
    q = _q(rng, B, Hkv * G, Q, dtype, dev)
    wide = torch.full((B, Q + 1, Hkv * G + 1, D), 7.0, dtype=dtype, device=dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(dev)
    held = torch.cuda.memory_allocated(dev)
    rows.attend_shared(q, None, SCALE, out=wide[:, 1:, 1:])
    if max(lens) <= 128:  # four tiles a row are not split
        assert torch.cuda.max_memory_allocated(dev) == held
    assert (wide[:, 0] == 7).all() and (wide[:, :, 0] == 7).all()
    for r, (k, v) in enumerate(kv):
        b, h = divmod(r, Hkv)
        for i in range(Q):
            n = max(len(k) - Q + 1 + i, 0)
            want, tol = attend(q[b, h * G:(h + 1) * G, i], k[:n], v[:n], SCALE, dtype)
            close(wide[b, 1 + i, 1 + h * G:1 + (h + 1) * G], want, tol, f"row {r} query {i}")
