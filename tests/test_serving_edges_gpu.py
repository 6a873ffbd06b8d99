"""The serving operators where their arithmetic has nothing ordinary to fold: scores without a number, weights far below
the largest, lengths that only the device knows."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import _lib, ops
from heterocache_amd.store import KVStore
from tests.serving_util import D, attend, bounds, close, make_rows, rotate, rounding, select, unpack

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
    """Captured appends advance the lengths on the device and not the host's mirror: an update() outside of the graph,
    on the current stream or on another, still takes every complete block."""
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


@pytest.mark.parametrize("what", ["peaked", "huge", "rising", "falling"])
@pytest.mark.parametrize("n", [70, 3000])
def test_fp16_scores_far_apart(dev, what, n):
    """One dominant key late, scores in the thousands, a steady rise or fall over many reference points."""
    rng = np.random.default_rng(n)
    prefix, rows = (make_rows(rng, [n], FP, dev, room=3)[0] for _ in range(2))
    k, v = (torch.as_tensor(rng.standard_normal((n, D)), dtype=torch.float32).to(FP).to(dev) for _ in range(2))
    q = _q(rng, 1, 4, 1, FP, dev)
    if what == "peaked":
        k[n - 5] = 12 * q[0, 0, 0]
    elif what == "huge":
        k *= 60
    else:
        ends = (-4, 4) if what == "rising" else (4, -4)
        k[:] = q[0, 0, 0] * torch.linspace(*ends, n, device=dev)[:, None].to(FP)
    for store in (prefix, rows):
        store.write_rows(k[None, None], v[None, None], [(0, 0)], [0], [n])
    for name, out, use_pre, use_own in _every_way(q, prefix, rows):
        want, tol = attend(q[0, :, 0], *_cat((k, v), (k, v), use_pre, use_own), SCALE, FP)
        # Weights below 2^-24 of the greatest: half of fp16's smallest step, 2^-35 of it, each.
        close(out[0, 0], want, tol + 2 * n * 2.0 ** -35 * v.double().abs().amax(0), f"{name} {what}")


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


def _turned(x, cos, sin):
    """rotate with one table a sequence, and the bound of its result in the type of x."""
    want, tol = rotate(x, cos, sin)
    return want, tol + rounding(want, x.dtype)


@pytest.mark.parametrize("dtype,tdt", [(BF, BF), (BF, FL), (FP, FP), (FP, FL), (FL, FL)])
@pytest.mark.parametrize("B,Hkv,G", [(65, 8, 4), (129, 4, 16), (600, 1, 1), (86, 6, 7)])
@pytest.mark.parametrize("in_place", [True, False])
def test_one_token_of_many_rows(dev, dtype, tdt, B, Hkv, G, in_place):
    """More than 512 rows of one token each: some at a tile's last slot, some full, some sequences with a count of 0."""
    rng = np.random.default_rng(B)
    R = B * Hkv
    draw = lambda *s: torch.as_tensor(rng.standard_normal(s), dtype=torch.float32)
    q, k, v = (draw(B, 1, h, D).to(dtype).to(dev).transpose(1, 2) for h in (Hkv * G, Hkv, Hkv))
    ang = rng.uniform(-3, 3, (B, 1, D))
    cos, sin = (torch.as_tensor(f(ang), dtype=torch.float32).to(tdt).to(dev) for f in (np.cos, np.sin))
    start = rng.integers(0, 64, R)
    start[::7] = 31
    start[3::11] = 64  # full
    counts = (rng.random(B) < 0.8).astype(np.int32)
    counts[0], counts[1] = 1, 0
    store = KVStore([64] * R, dtype, dev)
    store.k.copy_(draw(store.k.numel()).to(dtype))
    store.v.copy_(draw(store.v.numel()).to(dtype))
    store.set_lengths(start)
    before = [x.clone() for x in unpack(store.k, store.v)]
    lens = store.row_len if in_place else torch.full_like(store.row_len, -7)
    got = ops.append_rotated(q, k, v, cos, sin, *_meta(store), store.row_cap, len_out=lens, status=store.status,
                             counts=torch.as_tensor(counts).to(dev))
    want, tol = _turned(q, cos, sin)
    close(got, want, tol, "queries")
    per_row = np.repeat(counts, Hkv)
    stored = torch.as_tensor((per_row > 0) & (start < 64)).to(dev)
    assert lens.tolist() == (start + stored.cpu().numpy()).tolist()
    assert bool(store.status) == bool(((per_row > 0) & (start == 64)).any())
    at = (store.row_tile_off * 32 + torch.as_tensor(start).to(dev))[stored]
    want, tol = _turned(k, cos, sin)
    kn, vn = unpack(store.k, store.v)
    close(kn[at], want.reshape(R, D)[stored], tol.reshape(R, D)[stored], "keys")
    assert torch.equal(vn[at], v.reshape(R, D)[stored])
    rest = torch.ones(len(kn), dtype=torch.bool, device=dev)
    rest[at] = False
    assert torch.equal(kn[rest], before[0][rest]) and torch.equal(vn[rest], before[1][rest])


@pytest.mark.parametrize("Q,dtype", [(1, BF), (3, FP), (5, FL)])
def test_waves_of_many_tiles(dev, Q, dtype):
    """Rows cut for one tile: each of four waves walks more than 64 tiles, and more than 128."""
    rng = np.random.default_rng(Q)
    rows, kv = make_rows(rng, [9001, 17003, 8192, 8193], dtype, dev, room=5)
    q = _q(rng, 2, 6, Q, dtype, dev)
    got = ops.shared_attn(q, None, _meta(rows), 2, SCALE, row_tiles=1)
    for r, (k, v) in enumerate(kv):
        b, h = divmod(r, 2)
        for i in range(Q):
            n = len(k) - Q + 1 + i
            want, tol = attend(q[b, 3 * h:3 * h + 3, i], k[:n], v[:n], SCALE, dtype)
            close(got[b, i, 3 * h:3 * h + 3], want, tol, f"row {r} query {i}")


@pytest.mark.parametrize("G,dtype", [(4, BF), (9, FP), (2, FL)])
def test_lists_of_many_tiles(dev, G, dtype):
    """So many queries that no list is split, each of more than 64 tiles a wave: whole lists, shorter ones, entries in
    any order and some that are no block of the row."""
    rng = np.random.default_rng(G)
    B, Q, block, keep = 2, 260, 64, 400
    n = 64 * 500 - 9
    rows, kv = make_rows(rng, [n, 64 * 300 + 5], dtype, dev)
    q = _q(rng, B, G, Q, dtype, dev)
    idx = np.stack([[rng.permutation(520)[:keep] for _ in range(Q)] for _ in range(B)]).astype(np.int32)
    counts = rng.choice([keep, keep, 399, 130, 129, 128, 1], (B, Q)).astype(np.int32)
    assert _lib.load().hc_block_attn_workspace_size(B, G, 1, Q, block, keep) == 0
    got = ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, torch.as_tensor(idx).to(dev),
                         torch.as_tensor(counts).to(dev), block, SCALE)
    for r, (k, v) in enumerate(kv):
        for i in list(range(0, Q, 37)) + [Q - 1]:
            seen = len(k) - Q + 1 + i
            pos = (np.sort(idx[r, i, :counts[r, i]])[:, None] * block + np.arange(block)).reshape(-1)
            pos = torch.as_tensor(pos[pos < seen], dtype=torch.int64).to(dev)
            want, tol = attend(q[r, :, i], k[pos], v[pos], SCALE, dtype)
            close(got[r, i], want, tol, f"row {r} query {i}")


@pytest.mark.parametrize("block,dtype", [(64, BF), (96, FP), (128, FL), (32, BF)])
def test_bounds_of_many_blocks(dev, block, dtype):
    """So many blocks that a workgroup takes several of a row, the next one's first tiles on their way: all entries, and
    no others."""
    rng = np.random.default_rng(block)
    lens = [block * 300 + 7, block * 299, 5, block * 150 + block - 1] * 8
    store = KVStore([n + 40 for n in lens], dtype, dev)
    gen = torch.Generator(device=dev).manual_seed(block)
    store.k.copy_(torch.randn(store.k.numel(), generator=gen, device=dev).to(dtype))
    store.set_lengths(lens)
    index = store.block_index(block)
    assert len(lens) * (max(lens) // block) > 2 * 8 * torch.cuda.get_device_properties(dev).multi_processor_count
    index.bounds.fill_(5)
    index.exps.fill_(77)
    index.update()
    kn, _ = unpack(store.k, store.v)
    filled = torch.zeros(len(index.exps), dtype=torch.bool, device=dev)
    for r, n in enumerate(lens):
        j, at, off = n // block, int(store.host_tile_off[r]) * 32, int(index.row_block_off[r])
        cut = kn[at:at + j * block].double().view(j, block, D)
        hi, lo = cut.amax(1), cut.amin(1)
        e = torch.ceil(torch.log2(torch.maximum(hi.abs(), lo.abs()).amax(1) / 127))  # (64 bits: no top is on a border)
        unit = torch.exp2(e)[:, None]
        assert torch.equal(index.exps[off:off + j].double(), e), r
        assert torch.equal(index.bounds[off:off + j, 0].double(), torch.ceil(hi / unit)), r
        assert torch.equal(index.bounds[off:off + j, 1].double(), torch.floor(lo / unit)), r
        filled[off:off + j] = True
    assert (index.exps[~filled] == 77).all() and (index.bounds[~filled] == 5).all()


@pytest.mark.parametrize("blocks,keep", [(n, 40) for n in (257, 258, 1023, 1024, 1026, 2051, 4099, 6143, 6146, 12287,
                                                                     12288)] + [(300, 150), (5000, 2500)])
@pytest.mark.parametrize("B,Hkv,Q", [(20, 8, 1), (3, 2, 22)])
def test_selection_that_scores_its_own_rows(dev, blocks, keep, B, Hkv, Q):
    """So many queries that each row is scored where it is picked from, however long (keys in LDS): lengths around each
    change of its workgroups, many equal scores, against sorting."""
    rng = np.random.default_rng(blocks + Q)
    G, R = 2, B * Hkv
    assert _lib.load().hc_block_select_scratch_size(B, Hkv, Q, blocks) == 0
    assert _lib.load().hc_block_select_scratch_size(B, Hkv, Q, 12289) > 0
    lens = [(32 * blocks, 32 * blocks - 7, 32 * (blocks // 2) + Q, 32 * (keep + 1) + Q, 32 * (blocks - 1) + Q)[r % 5]
            for r in range(R)]
    # One table for all rows: pairs of equal blocks in it.
    hi = rng.integers(-127, 128, (blocks, D)).astype(np.int8)
    hi[1::3] = hi[::3][:len(hi[1::3])]
    lo = np.minimum(hi, rng.integers(-127, 128, hi.shape)).astype(np.int8)
    lo[1::3] = lo[::3][:len(lo[1::3])]
    ex = np.full(blocks, -5, np.int8)
    q = _q(rng, B, Hkv * G, Q, BF, dev)
    table = torch.as_tensor(np.stack([hi, lo], 1)).to(dev)
    idx, counts = ops.block_select(q, table, torch.as_tensor(ex).to(dev), torch.zeros(R, dtype=torch.int64, device=dev),
                                   torch.tensor(lens, dtype=torch.int32, device=dev), 32, blocks, keep, sink=1, local=2)
    # Whole numbers below 2^24 times powers of two: exact in 64 bits.
    hd, ld = (torch.as_tensor(x).to(dev).double().t().contiguous() for x in (hi, lo))
    qd = q.double().view(B, Hkv, G, Q, D)
    top = qd.abs().amax(-1, keepdim=True)
    eq = torch.ceil(torch.log2(top / 127)).clamp(-48, 48)
    q8 = torch.round(qd / torch.exp2(eq)).clamp(-127, 127).reshape(-1, D)
    s = (q8.clamp(min=0) @ hd + q8.clamp(max=0) @ ld).view(B, Hkv, G, Q, blocks) * torch.exp2(eq - 5)
    s = s.amax(2).reshape(R, Q, blocks)
    seen = torch.tensor(lens, device=dev)[:, None] - Q + 1 + torch.arange(Q, device=dev)
    have = ((seen + 31) // 32)[..., None]
    j = torch.arange(blocks, device=dev)
    s = torch.where((j < 1) | (j >= have - 2), torch.full_like(s, math.inf), s)
    s = torch.where(j < have, s, torch.full_like(s, -math.inf))
    want = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    assert (have > keep).all() and (counts == keep).all()
    assert torch.equal(idx.long(), want)


@pytest.mark.parametrize("B,Hkv,G,Q,blocks,keep,dtype", [
    (2, 2, 4, 1, 60, 8, BF), (1, 2, 9, 1, 60, 8, FP), (2, 1, 4, 3, 700, 6, BF), (1, 1, 2, 1, 100, 80, FL),
    (5, 4, 1, 1, 300, 6, BF),
])
def test_block_step_of_plain_tensors(dev, B, Hkv, G, Q, blocks, keep, dtype):
    """ops.block_step, on tensors of its own: its output, list and counts against the plain form, with query counts."""
    rng = np.random.default_rng(blocks)
    n = 32 * blocks
    rows, kv = make_rows(rng, [(n - 5, n // 2, 40, n)[r % 4] for r in range(B * Hkv)], dtype, dev, room=6)
    index = rows.block_index(32)
    index.update()
    q = _q(rng, B, Hkv * G, Q, dtype, dev)
    part = torch.as_tensor(rng.integers(0, Q + 1, B), dtype=torch.int32).to(dev)
    for qc in (None, part):
        out, idx, counts = ops.block_step(q, *_meta(rows), index.bounds, index.exps, index.row_block_off, 32,
                                          index.max_blocks, keep, SCALE, sink=1, local=2, query_counts=qc)
        for r in ([0, 1, len(kv) - 1] if len(kv) > 8 else range(len(kv))):
            k, v = kv[r]
            b, h = divmod(r, Hkv)
            table = bounds(k, 32)
            for i in range(Q):
                c = Q if qc is None else int(qc[b])
                seen = min(max(len(k) - c + 1 + i, 0), len(k))
                head = q[b, h * G:(h + 1) * G, i]
                want = select(head, *table, seen, 32, keep, 1, 2)
                assert int(counts[r, i]) == len(want) and idx[r, i, :len(want)].tolist() == want.tolist(), (r, i)
                pos = (want[:, None] * 32 + np.arange(32)).reshape(-1)
                pos = torch.as_tensor(pos[pos < seen], dtype=torch.int64).to(dev)
                ref, tol = attend(head, k[pos], v[pos], SCALE, dtype)
                close(out[b, i, h * G:(h + 1) * G], ref, tol, f"row {r} query {i}")
    meta = (index.bounds, index.exps, index.row_block_off)
    for bad in (dict(bounds=index.bounds[:1]), dict(exps=index.exps.int()), dict(off=index.row_block_off.int())):
        a = dict(bounds=meta[0], exps=meta[1], off=meta[2])
        a.update(bad)
        with pytest.raises(ValueError):
            ops.block_step(q, *_meta(rows), a["bounds"], a["exps"], a["off"], 32, index.max_blocks, keep, SCALE)
    with pytest.raises(TypeError):
        ops.block_step(q, rows.k.to(torch.int16), rows.v, rows.row_tile_off, rows.row_len, *meta, 32, index.max_blocks,
                       keep, SCALE)
    with pytest.raises(_lib.HCError, match="block=40"):
        ops.block_step(q, *_meta(rows), *meta, 40, index.max_blocks, keep, SCALE)
