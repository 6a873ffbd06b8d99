"""Rotated append (ops.append_rotated, KVStore.append_rotated) against its plain 64-bit form."""
import numpy as np
import pytest
import torch

from heterocache_amd import _lib, ops
from heterocache_amd.store import KVStore
from tests.serving_util import D, rotate, rounding, unpack, within

pytestmark = pytest.mark.gpu
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32


def _randn(rng, *shape):
    return torch.as_tensor(rng.standard_normal(shape), dtype=torch.float32)


def _inputs(rng, B, Hkv, G, T, dtype, tdt, dev, heads_first=False, shared_table=False):
    shape = lambda h: (B, h, T, D) if heads_first else (B, T, h, D)
    q, k, v = (_randn(rng, *shape(h)).to(dtype).to(dev) for h in (Hkv * G, Hkv, Hkv))
    if not heads_first:
        q, k, v = (x.transpose(1, 2) for x in (q, k, v))
    ang = rng.uniform(-3, 3, (1 if shared_table else B, T, D))  # halves differ: the general form
    cos, sin = (torch.as_tensor(f(ang), dtype=torch.float32).to(tdt).to(dev) for f in (np.cos, np.sin))
    return q, k, v, cos, sin


def _store(rng, start, room, dtype, dev):
    store = KVStore([int(n) + room for n in start], dtype, dev)
    for buf in (store.k, store.v):
        buf.copy_(_randn(rng, buf.numel()).to(dtype))
    store.set_lengths(start)
    return store


def _check(store, before, start, counts, q, k, v, cos, sin, got_q, Hkv, dtype):
    """The turned queries, every slot of the store and the lengths."""
    if cos.shape[0] != q.shape[0]:
        cos, sin = (t.expand(q.shape[0], -1, -1) for t in (cos, sin))
    wq, tq = rotate(q, cos, sin)
    assert within(got_q, wq, tq + rounding(wq, dtype))
    wk, tk = rotate(k, cos, sin)
    bk, bv = (x.double().clone() for x in unpack(*before))
    tol = torch.zeros_like(bk)
    off = store.host_tile_off * 32
    for r, n in enumerate(start):
        b, h = divmod(r, Hkv)
        at = int(off[r]) + int(n)
        c = int(counts[b])
        bk[at:at + c], bv[at:at + c] = wk[b, h, :c], v[b, h, :c].double()
        tol[at:at + c] = tk[b, h, :c] + rounding(wk[b, h, :c], dtype)
    gk, gv = unpack(store.k, store.v)
    assert within(gk, bk, tol)
    assert torch.equal(gv.double(), bv)


CASES = [
    # B, Hkv, G, T, counts, dtype, tables
    (1, 8, 4, 1, None, BF, BF), (3, 4, 7, 1, None, FP, FP), (2, 2, 8, 1, [1, 0], FL, FL),
    (2, 3, 5, 2, None, BF, FL), (1, 8, 4, 31, None, FP, FL), (2, 2, 4, 32, [32, 7], BF, BF),
    (3, 2, 1, 33, [0, 33, 20], FP, FP), (2, 1, 16, 64, None, BF, BF), (1, 2, 4, 65, [65], FL, FL),
    (4, 2, 4, 101, [101, 64, 1, 0], BF, FL), (1, 8, 4, 257, None, BF, BF), (2, 2, 2, 500, [499, 13], FL, FL),
]


@pytest.mark.parametrize("B,Hkv,G,T,counts,dtype,tdt", CASES)
@pytest.mark.parametrize("in_place", [True, False])
def test_matches_the_plain_form(dev, B, Hkv, G, T, counts, dtype, tdt, in_place):
    rng = np.random.default_rng(B * 1000 + T)
    q, k, v, cos, sin = _inputs(rng, B, Hkv, G, T, dtype, tdt, dev, heads_first=T % 2 == 0, shared_table=T == 257)
    start = rng.integers(0, 70, B * Hkv)
    start[0] = 0
    store = _store(rng, start, T + 3, dtype, dev)
    before = store.k.clone(), store.v.clone()
    n = np.full(B, T) if counts is None else np.asarray(counts)
    dc = None if counts is None else torch.as_tensor(n, dtype=torch.int32).to(dev)
    lens = store.row_len if in_place else torch.full_like(store.row_len, -7)
    got = ops.append_rotated(q, k, v, cos, sin, store.k, store.v, store.row_tile_off, store.row_len, store.row_cap,
                             counts=dc, len_out=lens, status=store.status)
    _check(store, before, start, n, q, k, v, cos, sin, got, Hkv, dtype)
    assert lens.tolist() == (start + np.repeat(n, Hkv)).tolist()
    if not in_place:
        assert store.row_len.tolist() == start.tolist()
    assert int(store.status) == 0


@pytest.mark.parametrize("T", [1, 40])
def test_full_row_is_left_alone(dev, T):
    rng = np.random.default_rng(T)
    B, Hkv, G = 2, 2, 4
    q, k, v, cos, sin = _inputs(rng, B, Hkv, G, T, BF, BF, dev)
    store = KVStore([64] * 4, BF, dev)
    for buf in (store.k, store.v):
        buf.copy_(_randn(rng, buf.numel()).to(BF))
    start = [10, 64, 64 - T + 1, 64 - T]  # rows 1 and 2 have no room
    store.set_lengths(start)
    before = store.k.clone(), store.v.clone()
    got = ops.append_rotated(q, k, v, cos, sin, store.k, store.v, store.row_tile_off, store.row_len, store.row_cap,
                             len_out=store.row_len, status=store.status)
    assert store.row_len.tolist() == [10 + T, 64, 64 - T + 1, 64]
    with pytest.raises(_lib.HCError):
        ops.read_status(store.status)
    gk, gv = unpack(store.k, store.v)
    ok, ov = unpack(*before)
    for r in (1, 2):
        lo = int(store.host_tile_off[r]) * 32
        assert torch.equal(gk[lo:lo + 64], ok[lo:lo + 64]) and torch.equal(gv[lo:lo + 64], ov[lo:lo + 64])
    assert torch.equal(gv[10:10 + T], v[0, 0])
    wq, tq = rotate(q, cos, sin)
    assert within(got, wq, tq + rounding(wq, BF))


def test_store_method_in_place_queries_and_lengths(dev):
    """KVStore.append_rotated token by token and in chunks: the mirror follows, q may be its own output."""
    rng = np.random.default_rng(7)
    B, Hkv, G = 2, 2, 4
    store = KVStore([100] * 4, FP, dev)
    total = np.zeros(2, dtype=int)
    ks, tols = [[], []], [[], []]
    for T, counts in ((37, [37, 20]), (1, None), (5, [0, 5]), (1, None), (33, None)):
        q, k, v, cos, sin = _inputs(rng, B, Hkv, G, T, FP, FP, dev)
        wq, tq = rotate(q, cos, sin)
        wk, tk = rotate(k, cos, sin)
        got = store.append_rotated(q, k, v, cos, sin, counts=counts, out=q)
        assert got.data_ptr() == q.data_ptr()
        assert within(q, wq, tq + rounding(wq, FP))
        n = np.full(2, T) if counts is None else np.asarray(counts)
        for b in range(2):
            ks[b].append(wk[b, :, :n[b]])
            tols[b].append(tk[b, :, :n[b]])
        total += n
        assert store.host_len.tolist() == np.repeat(total, 2).tolist() == store.row_len.tolist()
    for b in range(2):
        want = torch.cat(ks[b], dim=1)
        tols[b] = torch.cat(tols[b], dim=1)
        for h in range(2):
            got, _ = store.read_rows([b * 2 + h], int(total[b]))
            assert within(got[0], want[h], tols[b][h] + rounding(want[h], FP))
    with pytest.raises(RuntimeError, match="OOM"):
        store.append_rotated(*_inputs(rng, B, Hkv, G, 64, FP, FP, dev))
    assert store.host_len.tolist() == store.row_len.tolist()


def test_strided_views_and_another_stream(dev):
    """Views into wider projections (q, k, v of one tensor), tables with a token stride, a side stream."""
    rng = np.random.default_rng(9)
    B, Hkv, G, T = 2, 2, 4, 50
    wide = _randn(rng, B, T, (G + 2) * Hkv + 3, D).to(BF).to(dev)
    q, k, v = (wide[:, :, a:b].transpose(1, 2) for a, b in ((0, 8), (8, 10), (11, 13)))
    tabs = _randn(rng, B, T, 2, D).to(dev)
    cos, sin = tabs[:, :, 0], tabs[:, :, 1]
    start = rng.integers(0, 40, 4)
    store = _store(rng, start, T, BF, dev)
    before = store.k.clone(), store.v.clone()
    keep = wide.clone()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    got = store.append_rotated(q, k, v, cos, sin, counts=[50, 3], stream=side)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(wide, keep)
    _check(store, before, start, [50, 3], q, k, v, cos, sin, got, Hkv, BF)


def test_captured_steps_replay(dev):
    """A captured one-token step replayed with eager work between: lengths advance on the device."""
    rng = np.random.default_rng(11)
    B, Hkv, G = 2, 2, 4
    store = KVStore([64] * 4, BF, dev)
    store.set_lengths([5, 6, 7, 31])
    q, k, v, cos, sin = _inputs(rng, B, Hkv, G, 1, BF, BF, dev)
    out = torch.empty_like(q)
    args = (store.k, store.v, store.row_tile_off, store.row_len, store.row_cap)
    ops.append_rotated(q, k, v, cos, sin, *args, out=out)  # loads the kernels
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.append_rotated(q, k, v, cos, sin, *args, out=out, len_out=store.row_len, status=store.status)
    lens = np.array([5, 6, 7, 31])
    for step in range(4):
        nq, nk, nv, nc, ns = _inputs(rng, B, Hkv, G, 1, BF, BF, dev)
        for dst, src in ((q, nq), (k, nk), (v, nv), (cos, nc), (sin, ns)):
            dst.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        lens += 1
        assert store.row_len.tolist() == lens.tolist()
        wq, tq = rotate(nq, nc, ns)
        assert within(out, wq, tq + rounding(wq, BF))
        _, gv = unpack(store.k, store.v)
        for r in range(4):
            at = int(store.host_tile_off[r]) * 32 + int(lens[r]) - 1
            assert torch.equal(gv[at], nv[r // 2, r % 2, 0])


def test_rows_far_into_a_large_store(dev):
    """Tile offsets whose elements pass 2^31."""
    rng = np.random.default_rng(13)
    far = (1 << 31) // 4096 + 3
    buf = torch.zeros((2, (far + 2) * 4096), dtype=BF, device=dev)
    off = torch.tensor([0, far], dtype=torch.int64, device=dev)
    lens = torch.tensor([3, 30], dtype=torch.int32, device=dev)
    cap = torch.tensor([32, 64], dtype=torch.int32, device=dev)
    q, k, v, cos, sin = _inputs(rng, 1, 2, 2, 9, BF, BF, dev)
    ops.append_rotated(q, k, v, cos, sin, buf[0], buf[1], off, lens, cap, len_out=lens)
    assert lens.tolist() == [12, 39]
    tk, tv = unpack(buf[0, far * 4096:], buf[1, far * 4096:])
    wk, ek = rotate(k, cos, sin)
    assert torch.equal(tv[30:39], v[0, 1])
    assert within(tk[30:39], wk[0, 1], ek[0, 1] + rounding(wk[0, 1], BF))
    assert not tk[:30].any() and not tk[39:].any()


def test_empty_calls(dev):
    store = KVStore([32] * 2, BF, dev)
    store.set_lengths([4, 5])
    rng = np.random.default_rng(1)
    q, k, v, cos, sin = _inputs(rng, 1, 2, 4, 0, BF, BF, dev)
    assert store.append_rotated(q, k, v, cos, sin).shape == q.shape
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    ops.append_rotated(q, k, v, cos, sin, store.k, store.v, store.row_tile_off, store.row_len, store.row_cap,
                       len_out=lens)
    assert lens.tolist() == store.row_len.tolist() == [4, 5]


def test_refusals(dev):
    rng = np.random.default_rng(3)
    store = KVStore([64] * 4, BF, dev)
    q, k, v, cos, sin = _inputs(rng, 2, 2, 4, 3, BF, BF, dev)
    meta = (store.k, store.v, store.row_tile_off, store.row_len, store.row_cap)
    bad = [
        dict(q=q[..., :64]), dict(k=k[:, :, :2]), dict(k=k.to(FP)), dict(v=v[:1]), dict(q=q[:, :3]),
        dict(cos=cos[:, :2]), dict(cos=cos.to(FP), sin=sin.to(FP)), dict(cos=cos.float()),
        dict(q=q.cpu()), dict(counts=torch.zeros(3, dtype=torch.int32, device=dev)),
        dict(counts=torch.zeros(2, dtype=torch.int64, device=dev)), dict(out=torch.empty_like(q)[:, :4]),
        dict(len_out=torch.zeros(3, dtype=torch.int32, device=dev)),
    ]
    for change in bad:
        a = dict(q=q, k=k, v=v, cos=cos, sin=sin)
        kw = {x: change[x] for x in change if x not in a}
        a.update({x: change[x] for x in change if x in a})
        with pytest.raises((ValueError, TypeError)):
            ops.append_rotated(a["q"], a["k"], a["v"], a["cos"], a["sin"], *meta, **kw)
    both = torch.zeros(7, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="overlaps"):
        ops.append_rotated(q, k, v, cos, sin, *meta[:3], both[:4], store.row_cap, len_out=both[2:6])
    odd = torch.zeros(q.numel() + 1, dtype=BF, device=dev)[1:].view(q.shape)
    with pytest.raises(_lib.HCError, match="aligned"):
        ops.append_rotated(odd, k, v, cos, sin, *meta)
    with pytest.raises(ValueError):
        store.append_rotated(q, k, v, cos, sin, counts=[1, 4])
    with pytest.raises(ValueError):
        store.append_rotated(q[:1], k[:1], v[:1], cos[:1], sin[:1])
    assert store.row_len.tolist() == [0] * 4 and not store.k.any()
