"""Block-sparse attention (BlockIndex, KVStore.attend_blocks, ops.block_*) against its plain 64-bit form."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import _lib, ops
from heterocache_amd.store import KVStore
from tests.serving_util import D, attend, bounds, close, exponent, make_rows, select

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
SCALE = 1 / math.sqrt(D)


def _q(rng, B, Hq, Q, dtype, dev):
    q = torch.as_tensor(rng.standard_normal((B, Q, Hq, D)), dtype=torch.float32)
    return q.to(dtype).to(dev).transpose(1, 2)


def _check_index(index, kv):
    off = index.row_block_off.tolist()
    for r, (k, _) in enumerate(kv):
        hi, lo, ex = bounds(k, index.block)
        n = len(ex)
        got = index.bounds[off[r]:off[r] + n].cpu().numpy()
        assert np.array_equal(got[:, 0], hi) and np.array_equal(got[:, 1], lo), r
        assert np.array_equal(index.exps[off[r]:off[r] + n].cpu().numpy(), ex), r


def _check(got, q, kv, G, block, keep, sink, local, dtype):
    out, idx, counts = got
    B, Hq, Q, _ = q.shape
    Hkv = Hq // G
    for r, (k, v) in enumerate(kv):
        b, h = divmod(r, Hkv)
        table = bounds(k, block)
        for i in range(Q):
            seen = max(len(k) - Q + 1 + i, 0)
            head = q[b, h * G:(h + 1) * G, i]
            want = select(head, *table, seen, block, keep, sink, local)
            assert int(counts[r, i]) == len(want), (r, i)
            row = idx[r, i].cpu().numpy()
            assert np.array_equal(row[:len(want)], want) and (row[len(want):] == -1).all(), (r, i)
            pos = (want[:, None] * block + np.arange(block)).reshape(-1)
            pos = torch.as_tensor(pos[pos < seen], dtype=torch.int64).to(k.device)
            ref, tol = attend(head, k[pos], v[pos], SCALE, dtype)
            close(out[b, i, h * G:(h + 1) * G], ref, tol, f"row {r} query {i}")


CASES = [
    # B, Hkv, G, Q, lengths (cycled), block, keep, sink, local, dtype
    (1, 2, 4, 1, [1000, 5], 32, 8, 1, 2, BF), (2, 2, 7, 1, [641, 640, 0, 31], 32, 5, 0, 1, FP),
    (2, 1, 16, 1, [2000, 1999], 64, 9, 2, 3, BF), (1, 3, 1, 1, [1500, 33, 64], 96, 4, 1, 1, FL),
    (2, 2, 4, 3, [900, 2, 64, 65], 32, 7, 1, 1, BF), (1, 2, 5, 6, [1300, 700], 64, 6, 2, 2, FP),
    (3, 1, 8, 2, [515, 100, 4000], 128, 6, 1, 1, BF), (1, 1, 4, 1, [9000], 32, 90, 1, 2, FL),
    (5, 4, 4, 1, [300, 400], 32, 6, 0, 2, BF), (1, 2, 4, 1, [700, 500], 32, 3, 1, 2, BF),
    (1, 1, 2, 20, [600], 32, 5, 0, 1, FP), (2, 1, 4, 1, [33, 800], 32, 1, 0, 1, BF),
]


@pytest.mark.parametrize("B,Hkv,G,Q,lens,block,keep,sink,local,dtype", CASES)
def test_matches_the_plain_form(dev, B, Hkv, G, Q, lens, block, keep, sink, local, dtype):
    """Bounds, kept blocks (equal) and outputs; stale slots hold NaN."""
    rng = np.random.default_rng(B * 100 + keep)
    rows, kv = make_rows(rng, [lens[r % len(lens)] for r in range(B * Hkv)], dtype, dev, room=7)
    q = _q(rng, B, Hkv * G, Q, dtype, dev)
    index = rows.block_index(block)
    index.update()
    _check_index(index, kv)
    _check(rows.attend_blocks(q, index, keep, SCALE, sink=sink, local=local), q, kv, G, block, keep, sink, local, dtype)


def test_long_rows_select_past_the_keys_held_on_chip(dev):
    """More middle blocks than the selection keeps in LDS, and many of them with equal scores."""
    rng = np.random.default_rng(1)
    n = 32 * 9000 + 5
    rows, kv = make_rows(rng, [n, 2000], BF, dev, room=3)
    k, v = kv[0]
    k[32 * 10:32 * 6000] = k[32 * 4:32 * 5].repeat(5990, 1)  # equal blocks: ties go to the lower ones
    rows.write_rows(k[None, None], v[None, None], [(0, 0)], [0], [n])
    q = (k[32 * 4].float() * 0.5).to(BF).view(1, 1, 1, D).expand(1, 2, 1, D).contiguous()
    index = rows.block_index(32)
    index.update()
    _check(rows.attend_blocks(q, index, 40, SCALE, sink=1, local=2), q, kv, 1, 32, 40, 1, 2, BF)


@pytest.mark.parametrize("dtype", [BF, FP, FL])
def test_values_at_the_edges_of_the_8_bit_scales(dev, dtype):
    """Zero blocks, tiny and large keys, values just above 127 steps, zero and tiny queries."""
    rng = np.random.default_rng(3)
    rows, kv = make_rows(rng, [32 * 9], dtype, dev, room=0)
    k, v = kv[0]
    k[0:32] = 0
    k[32:64] *= 2.0 ** -14
    k[64:96] *= 2.0 ** 8
    k[96:128, :] = 1.0
    k[96, 0] = 127.5
    k[128:160] = -0.25
    k[160, 5] = 127.0
    if dtype == FL:
        k[192:224] *= 1e-30
        k[224:256] *= 1e25
    rows.write_rows(k[None, None], v[None, None], [(0, 0)], [0], [32 * 9])
    index = rows.block_index(32)
    index.update()
    _check_index(index, kv)
    for scale in (0.0, 1.0, 2.0 ** -12):
        q = (_q(rng, 1, 4, 1, FL, dev) * scale).to(dtype)
        if dtype == FL:
            got = ops.block_select(q, index.bounds, index.exps, index.row_block_off, rows.row_len, 32, 9, 5, 1, 2)
            want = select(q[0, :, 0], *bounds(k, 32), 32 * 9, 32, 5, 1, 2)
            assert got[0][0, 0].tolist() == want.tolist()
        else:
            _check(rows.attend_blocks(q, index, 5, SCALE, sink=1, local=2), q, kv, 4, 32, 5, 1, 2, dtype)


def test_infinite_and_nan_keys_saturate(dev):
    """They neither hang nor misplace a block: NaN is passed over, an infinity takes the largest scale."""
    rows, kv = make_rows(np.random.default_rng(4), [32 * 5], BF, dev)
    k, v = kv[0]
    k[40, 3], k[70, 9], k[100, 9] = math.nan, math.inf, -math.inf
    rows.write_rows(k[None, None], v[None, None], [(0, 0)], [0], [160])
    index = rows.block_index(32)
    index.update()
    fixed = k[32:64].clone()
    fixed[8, 3] = fixed[9, 3]
    hi, lo, ex = bounds(fixed, 32)
    assert np.array_equal(index.bounds[1, 0].cpu().numpy(), hi[0]) and int(index.exps[1]) == ex[0]
    assert index.exps[2:4].tolist() == [48, 48]
    assert int(index.bounds[2, 0, 9]) == 127 and int(index.bounds[3, 1, 9]) == -127


def test_incremental_update_equals_a_whole_one(dev):
    """Blocks completed by appended tokens, one and several at a time; the others are left alone."""
    rng = np.random.default_rng(5)
    rows, kv = make_rows(rng, [30, 64, 95, 0], BF, dev, room=300, stale=0.0)
    index = rows.block_index(32)
    index.update()
    one, zero = torch.ones((1, D), device=dev), torch.zeros((1, D), device=dev)
    for T in (1, 1, 5, 70, 32, 1):
        k, v = (torch.as_tensor(rng.standard_normal((1, 4, T, D)), dtype=torch.float32).to(BF).to(dev) for _ in range(2))
        rows.append_rotated(k, k, v, one.expand(T, D), zero.expand(T, D))
        kv = [(torch.cat([a, k[0, r]]), torch.cat([b, v[0, r]])) for r, (a, b) in enumerate(kv)]
        index.update(T)
        _check_index(index, kv)
    mark = index.exps.clone()
    index.exps.fill_(77)
    index.update(1)  # each row's last token completed no block but where its length says so
    done = [len(k) % 32 == 0 and len(k) > 0 for k, _ in kv]
    off = index.row_block_off.tolist()
    for r, (k, _) in enumerate(kv):
        n = len(k) // 32
        got = index.exps[off[r]:off[r] + n].tolist()
        assert got == [77] * (n - 1) + [int(mark[off[r] + n - 1]) if done[r] else 77]


def test_selection_does_not_depend_on_the_batch(dev):
    rng = np.random.default_rng(6)
    rows, kv = make_rows(rng, [1500] * 8, BF, dev)
    q = _q(rng, 8, 4, 1, BF, dev)
    index = rows.block_index(32)
    index.update()
    out, idx, counts = rows.attend_blocks(q, index, 11, SCALE)
    again = rows.attend_blocks(q, index, 11, SCALE)
    assert torch.equal(out, again[0]) and torch.equal(idx, again[1])
    for r in (0, 5):
        one = KVStore([1500], BF, dev)
        one.write_rows(kv[r][0][None, None], kv[r][1][None, None], [(0, 0)], [0], [1500])
        ix = one.block_index(32)
        ix.update()
        assert torch.equal(one.attend_blocks(q[r:r + 1], ix, 11, SCALE)[1][0], idx[r])


def test_given_blocks_in_any_order_and_past_the_row(dev):
    """block_attn with a caller's list: order does not matter, entries outside the row are passed over."""
    rng = np.random.default_rng(7)
    rows, kv = make_rows(rng, [200, 70], FP, dev, room=9)
    q = _q(rng, 1, 8, 1, FP, dev)
    idx = torch.tensor([[[5, 0, 3, -1]], [[1, 900, 2, 40]]], dtype=torch.int32, device=dev)
    counts = torch.tensor([[3], [3]], dtype=torch.int32, device=dev)
    out = ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, idx, counts, 32, SCALE)
    for r, blocks in enumerate(([0, 3, 5], [1, 2])):
        k, v = kv[r]
        pos = torch.as_tensor([p for b in blocks for p in range(32 * b, 32 * b + 32) if p < len(k)]).to(dev)
        want, tol = attend(q[0, 4 * r:4 * r + 4, 0], k[pos], v[pos], SCALE, FP)
        close(out[0, 0, 4 * r:4 * r + 4], want, tol)
    none = ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, idx, counts * 0, 32, SCALE)
    assert not none.any()


def test_more_blocks_than_the_scratch_has_room_for(dev):
    """The selection says so (-1) and the attention of such a query is NaN; the other rows are served."""
    rng = np.random.default_rng(8)
    rows, kv = make_rows(rng, [640, 200], BF, dev)
    q = _q(rng, 1, 8, 1, BF, dev)
    index = rows.block_index(32)
    index.update()
    idx, counts = ops.block_select(q, index.bounds, index.exps, index.row_block_off, rows.row_len, 32, 10, 4)
    assert counts.view(-1).tolist() == [-1, 4] and (idx[0] == -1).all()
    out = ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, idx, counts, 32, SCALE)
    assert torch.isnan(out[0, 0, :4]).all() and torch.isfinite(out[0, 0, 4:]).all()


def test_captured_decode_steps(dev):
    """Append, index update, selection and attention of a step in one graph, replayed across block ends."""
    rng = np.random.default_rng(9)
    rows, kv = make_rows(rng, [318, 95], BF, dev, room=40, stale=0.0)
    index = rows.block_index(32)
    index.update()
    q = _q(rng, 1, 8, 1, BF, dev)
    kn, vn = (torch.zeros((1, 2, 1, D), dtype=BF, device=dev) for _ in range(2))
    one, zero = torch.ones((1, D), device=dev), torch.zeros((1, D), device=dev)
    rows.attend_blocks(q, index, 5, SCALE)
    ops.append_rotated(q, kn, vn, one, zero, rows.k, rows.v, rows.row_tile_off, rows.row_len, rows.row_cap)
    index.update(1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        turned = rows.append_rotated(q, kn, vn, one, zero)
        index.update(1)
        got = rows.attend_blocks(turned, index, 5, SCALE)
    for step in range(6):
        for t in (q, kn, vn):
            t.copy_(torch.as_tensor(rng.standard_normal(t.shape), dtype=torch.float32))
        kv = [(torch.cat([k, kn[0, r]]), torch.cat([v, vn[0, r]])) for r, (k, v) in enumerate(kv)]
        g.replay()
        torch.cuda.synchronize()
        _check_index(index, kv)
        _check(got, q, kv, 4, 32, 5, 1, 2, BF)


def test_another_stream_and_strided_queries(dev):
    rng = np.random.default_rng(10)
    rows, kv = make_rows(rng, [700, 300, 500, 100], BF, dev)
    wide = torch.as_tensor(rng.standard_normal((2, 2, 12, D)), dtype=torch.float32).to(BF).to(dev)
    q = wide[:, :, 2:10].transpose(1, 2)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    index = rows.block_index(64)
    index.update(stream=side)
    got = rows.attend_blocks(q, index, 4, SCALE, stream=side)
    torch.cuda.current_stream(dev).wait_stream(side)
    _check(got, q, kv, 4, 64, 4, 1, 2, BF)


def test_rows_far_into_a_large_store(dev):
    rng = np.random.default_rng(11)
    far = (1 << 31) // 4096 + 5
    buf = torch.zeros((2, (far + 8) * 4096), dtype=BF, device=dev)
    src, kv = make_rows(rng, [32 * 4, 200], BF, dev, stale=0.0)
    for x, one in zip(buf, (src.k, src.v)):
        x[:4 * 4096] = one[:4 * 4096]
        x[far * 4096:(far + 7) * 4096] = one[4 * 4096:11 * 4096]
    off = torch.tensor([0, far], dtype=torch.int64, device=dev)
    index = src.block_index(32)
    ops.block_bounds(buf[0], off, src.row_len, index.row_block_off, 32, index.bounds, index.exps, 6)
    _check_index(index, kv)
    q = _q(rng, 1, 8, 1, BF, dev)
    idx, counts = ops.block_select(q, index.bounds, index.exps, index.row_block_off, src.row_len, 32, 7, 4)
    out = ops.block_attn(q, buf[0], buf[1], off, src.row_len, idx, counts, 32, SCALE)
    _check((out, idx, counts), q, kv, 4, 32, 4, 1, 1, BF)


def test_refusals(dev):
    rng = np.random.default_rng(12)
    rows, _ = make_rows(rng, [100, 90], BF, dev)
    other, _ = make_rows(rng, [100, 90], BF, dev)
    q = _q(rng, 1, 8, 1, BF, dev)
    index = rows.block_index(32)
    index.update()
    for bad in (16, 0, 33, -32):
        with pytest.raises(ValueError):
            rows.block_index(bad)
    with pytest.raises(ValueError):
        other.attend_blocks(q, index, 4, SCALE)
    for kw in (dict(keep=0), dict(keep=2, sink=1, local=2), dict(keep=4, local=0), dict(keep=4, sink=-1)):
        with pytest.raises((_lib.HCError, RuntimeError)):
            rows.attend_blocks(q, index, kw.pop("keep"), SCALE, **kw)
    with pytest.raises(_lib.HCError, match="scale"):
        rows.attend_blocks(q, index, 4, -SCALE)
    with pytest.raises(TypeError):
        rows.attend_blocks(q.to(FP), index, 4, SCALE)
    with pytest.raises(ValueError):
        rows.attend_blocks(q[:, :7], index, 4, SCALE)
    with pytest.raises(ValueError):
        index.update(-1)
    idx, counts = ops.block_select(q, index.bounds, index.exps, index.row_block_off, rows.row_len, 32, 4, 4)
    with pytest.raises(ValueError):
        ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, idx[:1], counts, 32, SCALE)
    with pytest.raises(_lib.HCError, match="block"):
        ops.block_attn(q, rows.k, rows.v, rows.row_tile_off, rows.row_len, idx, counts, 40, SCALE)


@pytest.mark.parametrize("blocks,keep", [(n, 40) for n in (255, 256, 257, 1023, 1026, 2051, 6140, 6148, 12290, 32765, 32780)]
                         + [(n, 9) for n in (30, 63, 66, 67, 68, 127, 130, 131, 132, 150)])
def test_every_way_to_hold_the_keys(dev, blocks, keep):
    """Row lengths around each change of the selection's launch, with many equal scores, against sorting."""
    rng = np.random.default_rng(blocks)
    B, Hkv, G = 2, 2, 3
    lens = [32 * blocks - 7, 32 * (blocks // 2) + 1, 32 * (keep + 1), 32 * (blocks - 1) + 1]
    hi = rng.integers(-127, 128, (B * Hkv * blocks, D)).astype(np.int8)
    hi[1::3] = hi[::3][:len(hi[1::3])]  # pairs of equal blocks
    lo = np.minimum(hi, rng.integers(-127, 128, hi.shape)).astype(np.int8)
    lo[1::3] = lo[::3][:len(lo[1::3])]
    ex = np.full(len(hi), -5, np.int8)
    table = torch.as_tensor(np.stack([hi, lo], 1)).to(dev)
    off = torch.arange(B * Hkv, device=dev) * blocks
    q = _q(rng, B, Hkv * G, 1, BF, dev)
    idx, counts = ops.block_select(q, table, torch.as_tensor(ex).to(dev), off,
                                   torch.tensor(lens, dtype=torch.int32, device=dev), 32, blocks, keep, sink=1, local=2)
    hi, lo = hi.astype(np.int64), lo.astype(np.int64)
    for r in range(B * Hkv):
        b, h = divmod(r, Hkv)
        have = -(-lens[r] // 32)
        score = np.full(have, -np.inf)
        at = slice(r * blocks + 1, r * blocks + have - 2)
        for row in q[b, h * G:(h + 1) * G, 0].double().cpu().numpy():
            eq = exponent(np.abs(row).max())
            q8 = np.clip(np.rint(row / 2.0 ** eq), -127, 127).astype(np.int64)
            s = np.maximum(q8 * hi[at], q8 * lo[at]).sum(1) * 2.0 ** (eq - 5)
            score[1:have - 2] = np.maximum(score[1:have - 2], s)
        score[:1] = score[have - 2:] = np.inf
        want = np.sort(np.lexsort((np.arange(have), -score))[:keep])
        assert int(counts[r, 0]) == keep and np.array_equal(idx[r, 0].cpu().numpy(), want), r


@pytest.mark.parametrize("blocks", [12, 66, 67, 127, 130, 131, 132, 300])
def test_equal_blocks_go_by_their_place(dev, blocks):
    """Rows of three blocks over and over: most scores are equal, and the lower block wins, in one call as in two."""
    rng = np.random.default_rng(blocks)
    lens, block, keep = [32 * blocks - 3, 32 * (blocks // 2)], 32, 10
    rows, _ = make_rows(rng, lens, BF, dev, room=5)
    kv = []
    src = torch.zeros((2, 1, 2, lens[0], D), dtype=BF, device=dev)
    for r, n in enumerate(lens):
        three = torch.as_tensor(rng.standard_normal((96, D)), dtype=torch.float32).to(BF).to(dev)
        k = three.repeat(-(-n // 96), 1)[:n]
        v = torch.as_tensor(rng.standard_normal((n, D)), dtype=torch.float32).to(BF).to(dev)
        src[0, 0, r, :n], src[1, 0, r, :n] = k, v
        kv.append((k, v))
    rows.write_rows(src[0], src[1], [(0, 0), (0, 1)], [0, 1], lens)
    index = rows.block_index(block)
    index.update()
    q = _q(rng, 1, 8, 1, BF, dev)
    got = rows.attend_blocks(q, index, keep, SCALE)
    _check(got, q, kv, 4, block, keep, 1, 2, BF)
    idx, counts = ops.block_select(q, index.bounds, index.exps, index.row_block_off, rows.row_len, block,
                                   index.max_blocks, keep, sink=1, local=2)
    assert torch.equal(idx, got[1]) and torch.equal(counts, got[2])
