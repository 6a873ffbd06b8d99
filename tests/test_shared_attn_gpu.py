"""Shared-prefix attention (ops.shared_attn, KVStore.attend_shared) against its plain 64-bit form."""
import math

import numpy as np
import pytest
import torch

from heterocache_amd import _lib, ops
from heterocache_amd.store import KVStore
from tests.serving_util import D, attend, close, make_rows

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
SCALE = 1 / math.sqrt(D)


def _q(rng, B, Hq, Q, dtype, dev, heads_first=False):
    q = torch.as_tensor(rng.standard_normal((B, Hq, Q, D) if heads_first else (B, Q, Hq, D)), dtype=torch.float32)
    q = q.to(dtype).to(dev)
    return q if heads_first else q.transpose(1, 2)


def _check(got, q, pre, rows, G, scale, dtype, lens=None):
    """got [B, Q, Hq, 128] against the concatenated keys of each (sequence, head)."""
    B, Hq, Q, _ = q.shape
    Hkv = Hq // G
    for b in range(B):
        for h in range(Hkv):
            pk, pv = pre[h] if pre else (q.new_zeros((0, D)),) * 2
            sk, sv = rows[b * Hkv + h] if rows else (q.new_zeros((0, D)),) * 2
            for i in range(Q):
                seen = max(len(sk) - Q + 1 + i, 0)
                heads = slice(h * G, (h + 1) * G)
                want, tol = attend(q[b, heads, i], torch.cat([pk, sk[:seen]]), torch.cat([pv, sv[:seen]]), scale, dtype)
                close(got[b, i, heads], want, tol, f"sequence {b} KV head {h} query {i}")


CASES = [
    # B, Hkv, G, Q, prefix lengths, own lengths (cycled), dtype
    (1, 2, 4, 1, [1, 0], [1], BF), (3, 2, 4, 1, [40, 33], [5, 32, 0], BF), (2, 1, 1, 1, [64], [33, 1], FP),
    (4, 2, 7, 1, [513, 100], [65, 3], FP), (5, 2, 16, 1, [300, 299], [20, 129], BF), (2, 2, 5, 1, [95, 96], [64, 31], FL),
    (3, 2, 4, 3, [130, 1], [3, 2, 40], BF), (2, 2, 4, 8, [70, 0], [8, 100], FP), (2, 1, 16, 5, [257], [33, 4], BF),
    (2, 1, 3, 4, [129], [200, 7], FL), (20, 1, 4, 1, [1000], [17, 90], BF), (33, 1, 4, 1, [700], [5], FP),
    (9, 1, 4, 20, [100], [25], BF), (3, 2, 2, 1, [5000, 31], [1500, 700], BF), (40, 1, 8, 1, [333], [40], FL),
]


@pytest.mark.parametrize("B,Hkv,G,Q,plen,slen,dtype", CASES)
def test_matches_the_plain_form(dev, B, Hkv, G, Q, plen, slen, dtype):
    """Stale slots of both stores hold NaN."""
    rng = np.random.default_rng(B * 100 + Q)
    prefix, pre = make_rows(rng, plen, dtype, dev, room=5)
    rows, kv = make_rows(rng, [slen[r % len(slen)] for r in range(B * Hkv)], dtype, dev, room=9)
    q = _q(rng, B, Hkv * G, Q, dtype, dev, heads_first=B % 2 == 0)
    got = rows.attend_shared(q, prefix, SCALE)
    assert got.shape == (B, Q, Hkv * G, D)
    _check(got, q, pre, kv, G, SCALE, dtype)


@pytest.mark.parametrize("dtype", [BF, FP, FL])
def test_prefix_alone_rows_alone_and_nothing(dev, dtype):
    rng = np.random.default_rng(2)
    prefix, pre = make_rows(rng, [77, 0], dtype, dev)
    rows, kv = make_rows(rng, [20, 0, 3, 0], dtype, dev, room=4)
    q = _q(rng, 2, 8, 2, dtype, dev)
    meta = lambda s: (s.k, s.v, s.row_tile_off, s.row_len)
    _check(ops.shared_attn(q, meta(prefix), None, 2, SCALE, prefix_tiles=3), q, pre, None, 4, SCALE, dtype)
    _check(rows.attend_shared(q, None, SCALE), q, None, kv, 4, SCALE, dtype)
    got = rows.attend_shared(q, prefix, SCALE)
    _check(got, q, pre, kv, 4, SCALE, dtype)
    assert not got[:, :, 4:].any()  # KV head 1 holds nothing in any sequence
    empty = KVStore([32] * 4, dtype, dev)
    assert not empty.attend_shared(q, None, SCALE).any()


def test_sizes_to_cut_for_are_no_limits(dev):
    """Lengths far above the sizes the call was cut for, and below."""
    rng = np.random.default_rng(3)
    prefix, pre = make_rows(rng, [900, 3, 450], BF, dev)
    rows, kv = make_rows(rng, [300, 1, 2, 500, 64, 65], BF, dev, room=4)
    q = _q(rng, 2, 12, 1, BF, dev)
    meta = lambda s: (s.k, s.v, s.row_tile_off, s.row_len)
    for pt, rt in ((0, 0), (1, 1), (100000, 4000)):
        got = ops.shared_attn(q, meta(prefix), meta(rows), 3, SCALE, prefix_tiles=pt, row_tiles=rt)
        _check(got, q, pre, kv, 4, SCALE, BF)


@pytest.mark.parametrize("what", ["peaked", "huge", "rising"])
@pytest.mark.parametrize("dtype", [BF, FL])
def test_extreme_scores(dev, what, dtype):
    """Scores far apart: one dominant key late, scores in the thousands, and a steady rise that moves the
    reference point again and again."""
    rng = np.random.default_rng(4)
    prefix, pre = make_rows(rng, [400], dtype, dev)
    rows, kv = make_rows(rng, [70, 70], dtype, dev)
    q = _q(rng, 2, 4, 1, dtype, dev)
    for store, parts in ((prefix, pre), (rows, kv)):
        for r, (k, v) in enumerate(parts):
            n = len(k)
            if what == "peaked":
                k[n - 5] = 12 * q[0, 0, 0]
            elif what == "huge":
                k *= 60
            else:
                k[:] = q[0, 0, 0] * torch.linspace(-4, 4, n, device=dev)[:, None].to(dtype)
            store.write_rows(k[None, None], v[None, None], [(0, 0)], [r], [n])
    _check(rows.attend_shared(q, prefix, SCALE), q, pre, kv, 4, SCALE, dtype)


@pytest.mark.parametrize("dtype", [BF, FP, FL])
def test_values_of_unseen_tokens_do_not_reach_a_query(dev, dtype):
    """Infinite and NaN keys and values of tokens that only later queries see."""
    rng = np.random.default_rng(5)
    prefix, pre = make_rows(rng, [50], dtype, dev)
    rows, kv = make_rows(rng, [34, 40], dtype, dev)
    k, v = kv[0]
    v[31, 3], v[32, 7], k[33, 5] = math.inf, math.nan, math.nan
    rows.write_rows(k[None, None], v[None, None], [(0, 0)], [0], [34])
    q = _q(rng, 2, 4, 4, dtype, dev)  # query i of sequence 0 sees 31 + i tokens
    got = rows.attend_shared(q, prefix, SCALE)
    for i in (0,):
        want, tol = attend(q[0, :, i], torch.cat([pre[0][0], k[:31]]), torch.cat([pre[0][1], v[:31]]), SCALE, dtype)
        close(got[0, i], want, tol)
    want, tol = attend(q[0, :, 1], torch.cat([pre[0][0], k[:32]]),
                       torch.cat([pre[0][1], v[:32]]).nan_to_num(0, 0, 0), SCALE, dtype)
    ok = torch.arange(D, device=dev) != 3
    close(got[0, 1][:, ok], want[:, ok], tol[:, ok])
    assert torch.isinf(got[0, 1, :, 3]).all()
    assert torch.isnan(got[0, 2, :, 7]).all() and torch.isfinite(got[0, 2, :, 8]).all()
    assert torch.isnan(got[0, 3]).all()
    _check(got[1:], q[1:], pre, kv[1:], 4, SCALE, dtype)


def test_strides_output_view_and_another_stream(dev):
    rng = np.random.default_rng(6)
    prefix, pre = make_rows(rng, [200, 60], BF, dev)
    rows, kv = make_rows(rng, [10, 20, 30, 40], BF, dev, room=8)
    wide = torch.as_tensor(rng.standard_normal((2, 3, 14, D)), dtype=torch.float32).to(BF).to(dev)
    q = wide[:, 1:, 3:11].transpose(1, 2)
    out = torch.full((2, 5, 9, D), 7.0, dtype=BF, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    rows.attend_shared(q, prefix, SCALE, out=out[:, 1:5:2, :8], stream=side)
    torch.cuda.current_stream(dev).wait_stream(side)
    _check(out[:, 1:5:2, :8], q, pre, kv, 4, SCALE, BF)
    assert (out[:, 0::2] == 7).all() and (out[:, :, 8] == 7).all()


def test_two_graphs_replay_while_rows_grow(dev):
    """Append and attend captured on two stores; replays alternate, with eager work between."""
    rng = np.random.default_rng(8)
    prefix, pre = make_rows(rng, [150], BF, dev)
    sets = []
    one, zero = torch.ones((1, D), device=dev), torch.zeros((1, D), device=dev)  # both graphs read them
    for n in (3, 60):
        rows, kv = make_rows(rng, [n, n + 1], BF, dev, room=8, stale=0.0)
        q = _q(rng, 2, 4, 1, BF, dev)
        kn, vn = (torch.zeros((2, 1, 1, D), dtype=BF, device=dev) for _ in range(2))
        out = torch.empty((2, 1, 4, D), dtype=BF, device=dev)
        rows.attend_shared(q, prefix, SCALE, out=out)
        ops.append_rotated(q, kn, vn, one, zero, rows.k, rows.v, rows.row_tile_off, rows.row_len, rows.row_cap)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            turned = rows.append_rotated(q, kn, vn, one, zero)
            rows.attend_shared(turned, prefix, SCALE, out=out)
        sets.append([rows, kv, q, kn, vn, out, g])
    for step in range(3):
        for rows, kv, q, kn, vn, out, g in sets:
            for t in (q, kn, vn):
                t.copy_(torch.as_tensor(rng.standard_normal(t.shape), dtype=torch.float32))
            for r in range(2):
                kv[r] = (torch.cat([kv[r][0], kn[r, 0]]), torch.cat([kv[r][1], vn[r, 0]]))
            g.replay()
        torch.cuda.synchronize()
        for rows, kv, q, kn, vn, out, g in sets:
            _check(out, q, pre, kv, 4, SCALE, BF)


def test_rows_far_into_a_large_store(dev):
    rng = np.random.default_rng(10)
    far = (1 << 31) // 4096 + 5
    buf = torch.zeros((2, (far + 4) * 4096), dtype=BF, device=dev)
    src, kv = make_rows(rng, [70, 45], BF, dev, stale=0.0)
    for x, one in zip(buf, (src.k, src.v)):
        x[:3 * 4096] = one[:3 * 4096]
        x[far * 4096:(far + 2) * 4096] = one[3 * 4096:5 * 4096]
    off = torch.tensor([0, far], dtype=torch.int64, device=dev)
    part = (buf[0], buf[1], off, src.row_len)
    q = _q(rng, 1, 8, 1, BF, dev)
    _check(ops.shared_attn(q, part, None, 2, SCALE), q, kv, None, 4, SCALE, BF)
    _check(ops.shared_attn(q, None, part, 2, SCALE), q, None, kv, 4, SCALE, BF)


def test_refusals(dev):
    rng = np.random.default_rng(12)
    prefix, _ = make_rows(rng, [10, 10], BF, dev)
    rows, _ = make_rows(rng, [10] * 4, BF, dev)
    q = _q(rng, 2, 8, 1, BF, dev)
    for bad in (q[:, :7], q[..., :64], q.cpu(), q[:1].expand(3, -1, -1, -1)):
        with pytest.raises(ValueError):
            rows.attend_shared(bad, prefix, SCALE)
    with pytest.raises(TypeError):
        rows.attend_shared(q.to(FP), prefix, SCALE)
    with pytest.raises(ValueError):
        rows.attend_shared(q, rows, SCALE)
    with pytest.raises(ValueError):
        rows.attend_shared(q, prefix, SCALE, out=torch.empty((2, 1, 8, D), device=dev))
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(_lib.HCError, match="scale"):
            rows.attend_shared(q, prefix, scale)
    with pytest.raises(_lib.HCError, match="16 of it|at most 16"):
        ops.shared_attn(_q(rng, 2, 34, 1, BF, dev), (prefix.k, prefix.v, prefix.row_tile_off, prefix.row_len), None, 2,
                        SCALE)


@pytest.mark.parametrize("B,Hkv,G,Q,dtype", [(2, 2, 4, 1, BF), (40, 2, 4, 1, BF), (9, 1, 8, 3, FP), (3, 2, 2, 1, FL),
                                             (70, 1, 2, 1, FL)])
@pytest.mark.parametrize("tail", [0, 1, 17])
def test_long_parts(dev, B, Hkv, G, Q, dtype, tail):
    """Parts of many tiles (cut for a short prefix), of every number of tiles at their end."""
    rng = np.random.default_rng(13 + tail)
    for tiles in (33, 36, 39, 42):
        prefix, pre = make_rows(rng, [32 * tiles + tail] + [32 * tiles * 3] * (Hkv - 1), dtype, dev)
        rows, kv = make_rows(rng, [7 + r % 5 for r in range(B * Hkv)], dtype, dev)
        q = _q(rng, B, Hkv * G, Q, dtype, dev)
        meta = lambda s: (s.k, s.v, s.row_tile_off, s.row_len)
        got = ops.shared_attn(q, meta(prefix), meta(rows), Hkv, SCALE, prefix_tiles=0, row_tiles=1)
        _check(got, q, pre, kv, G, SCALE, dtype)


@pytest.mark.parametrize("B,Hkv,G,dtype", [(1, 64, 1, BF), (2, 65, 2, BF), (1, 130, 1, FP), (1, 200, 3, FL)])
def test_many_kv_heads(dev, B, Hkv, G, dtype):
    rng = np.random.default_rng(14)
    prefix, pre = make_rows(rng, [(37 * h) % 300 for h in range(Hkv)], dtype, dev)
    rows, kv = make_rows(rng, [(11 * r) % 70 for r in range(B * Hkv)], dtype, dev)
    q = _q(rng, B, Hkv * G, 1, dtype, dev)
    _check(rows.attend_shared(q, prefix, SCALE), q, pre, kv, G, SCALE, dtype)


@pytest.mark.parametrize("B,Hkv,G,Q,dtype,tiles", [
    (20, 8, 4, 1, BF, 8192), (32, 2, 16, 1, FP, 24000), (32, 8, 4, 1, BF, 5558), (16, 4, 7, 4, FP, 1537),
    (33, 2, 4, 1, BF, 300000), (6, 3, 5, 2, FP, 20000),
])
def test_cut_for_other_sizes(dev, B, Hkv, G, Q, dtype, tiles):
    """Column blocks and parts as they are chosen for long prefixes, over short ones."""
    rng = np.random.default_rng(tiles)
    prefix, pre = make_rows(rng, [(1500, 40, 0, 701, 32, 33, 1, 900)[h] for h in range(Hkv)], dtype, dev)
    rows, kv = make_rows(rng, [(5, 40, 64)[r % 3] + Q for r in range(B * Hkv)], dtype, dev)
    q = _q(rng, B, Hkv * G, Q, dtype, dev)
    meta = lambda s: (s.k, s.v, s.row_tile_off, s.row_len)
    got = ops.shared_attn(q, meta(prefix), meta(rows), Hkv, SCALE, prefix_tiles=tiles, row_tiles=4)
    _check(got, q, pre, kv, G, SCALE, dtype)
