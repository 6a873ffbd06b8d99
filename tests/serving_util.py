"""Plain 64-bit forms of the serving operators and the bounds of their error.

Tolerances are sums of what the arithmetic may lose: u(T) = finfo(T).eps / 2 per
rounding to the tensors' type, 2^-24 per float32 operation.
"""
import math

import numpy as np
import torch

D, TILE = 128, 32
F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(x, dtype):
    """Bound of one rounding of about |x| to dtype: half a step, which below the
    smallest normal number is half the spacing of the subnormal ones."""
    f = torch.finfo(dtype)
    return x.abs() * half_step(dtype) * 1.01 + f.tiny * f.eps / 2


def within(got, want, tol):
    """Largest excess of |got - want| over its bound is none."""
    bad = int(((got.double() - want).abs() > tol).sum())
    return bad == 0 and bool(torch.isfinite(got).all())


def unpack(buf_k, buf_v):
    """Tiled buffers in natural order: two [tokens, 128] tensors."""
    k = buf_k.view(-1, 2, 4, 4, 16, 8).permute(0, 1, 4, 2, 3, 5).reshape(-1, D)
    v = buf_v.view(-1, 8, 4, 16, 2, 4).permute(0, 4, 2, 5, 1, 3).reshape(-1, D)
    return k, v


def make_rows(rng, lens, dtype, dev, room=0, stale=float("nan")):
    """A store whose rows hold random keys and values; every other slot holds
    `stale`.  Returns (store, [(k, v) of each row])."""
    from heterocache_amd.store import KVStore
    store = KVStore([n + room for n in lens], dtype, dev)
    kv = [tuple(torch.as_tensor(rng.standard_normal((n, D)), dtype=torch.float32).to(dtype).to(dev) for _ in range(2))
          for n in lens]
    store.k.fill_(stale)
    store.v.fill_(stale)
    if max(lens, default=0) > 0:
        width = max(lens)
        src = torch.zeros((2, 1, len(lens), width, D), dtype=dtype, device=dev)
        for r, (k, v) in enumerate(kv):
            src[0, 0, r, :len(k)], src[1, 0, r, :len(v)] = k, v
        store.write_rows(src[0], src[1], [(0, r) for r in range(len(lens))], list(range(len(lens))), lens)
    return store, kv


def attend(q, k, v, scale, dtype):
    """softmax(scale q k^T) v in 64 bits and its bound: q [.., 128], k, v [n, 128].

    The score's float32 products and sum are off by at most 129 roundings of
    its absolute terms, its scaling and the exponent's argument by 4 of the
    score and the reference point; a probability by that difference, 2 ulp of
    exp2, and one rounding to the input type where it enters the product with
    V; the sums by one rounding a term and 8 a fold; the output by one to its type."""
    q, k, v = q.double(), k.double(), v.double()
    n = k.shape[0]
    if n == 0:
        z = torch.zeros_like(q)
        return z, z
    s = q @ k.t() * scale
    p = torch.softmax(s, dim=-1)
    out = p @ v
    mass = p @ v.abs()
    gap = F32 * (129 * (q.abs() @ k.abs().t()) * scale + 8 * s.abs() + 8).amax(-1, keepdim=True) * 2
    u = half_step(dtype)
    tol = mass * (u + 2 * gap + F32 * (2 * n + 64)) + rounding(out, dtype)
    return out, tol * 1.05


def close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = float((err - tol).max()) if err.numel() else -1.0
    assert worst <= 0, f"{what}: error above its bound by {worst:.3e} (largest error {float(err.max()):.3e})"


def exponent(top):
    e = -48
    while e < 48 and top > 127.0 * 2.0 ** e:
        e += 1
    return e


def bounds(k, block):
    """(hi, lo, e) of the complete blocks of one row's keys [n, 128]."""
    k = k.double().cpu().numpy()
    n = len(k) // block
    hi, lo, ex = np.zeros((n, D), np.int64), np.zeros((n, D), np.int64), np.zeros(n, np.int64)
    for j in range(n):
        part = k[j * block:(j + 1) * block]
        top, bot = part.max(0), part.min(0)
        ex[j] = exponent(max(np.abs(top).max(), np.abs(bot).max()))
        hi[j] = np.clip(np.ceil(top / 2.0 ** ex[j]), -127, 127)
        lo[j] = np.clip(np.floor(bot / 2.0 ** ex[j]), -127, 127)
    return hi, lo, ex


def select(q, hi, lo, ex, seen, block, keep, sink, local):
    """Kept blocks (ascending) of one query [G, 128] that sees `seen` tokens."""
    have = -(-seen // block)
    if have <= keep:
        return np.arange(have)
    score = np.full(have, -np.inf)
    for row in q.double().cpu().numpy():
        eq = exponent(np.abs(row).max())
        q8 = np.clip(np.rint(row / 2.0 ** eq), -127, 127)
        for j in range(sink, have - local):
            score[j] = max(score[j], np.maximum(q8 * hi[j], q8 * lo[j]).sum() * 2.0 ** (eq + ex[j]))
    score[:sink] = np.inf
    score[have - local:] = np.inf
    return np.sort(np.lexsort((np.arange(have), -score))[:keep])


def rotate(x, cos, sin):
    """x [B, H, T, 128] turned by tables [B, T, 128], in 64 bits, and its bound
    before the last rounding (two products and a sum in float32)."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = x[..., :64], x[..., 64:]
    out = torch.cat([a * c[..., :64] - b * s[..., :64], b * c[..., 64:] + a * s[..., 64:]], dim=-1)
    size = torch.cat([a.abs() * c[..., :64].abs() + b.abs() * s[..., :64].abs(),
                      b.abs() * c[..., 64:].abs() + a.abs() * s[..., 64:].abs()], dim=-1)
    return out, 3 * F32 * size
