"""Paged caches for the tests, and the plain 64-bit forms of what is done to them."""
import numpy as np
import torch

from heterocache_amd import ops
from tests.serving_util import D, F32, half_step, rounding


def _random(rng, shape, dtype, dev):
    return torch.as_tensor(rng.standard_normal(shape), dtype=torch.float32).to(dtype).to(dev)


class Cache:
    """pages: the ops.Pages; kv[row b * Hkv + h]: its (keys, values) [n, 128].

    lens: tokens of each table row (cycled), rows = batch * (Hkv if apart else
    1).  Pages lie in random order, slots that hold nothing are `stale`, table
    entries behind a row's room are -1.  order: a token's heads together
    ("token"), or a head's tokens ("head")."""

    def __init__(self, rng, batch, kv_heads, lens, page, dtype, dev, apart=False, room=0, stale=float("nan"), order="token",
                 ledger=False, width=None, spare=3):
        heads = 1 if apart else kv_heads
        rows = batch * kv_heads // heads
        self.lens = np.array([lens[r % len(lens)] for r in range(rows)], dtype=np.int64)
        need = -(-(self.lens + room) // page)
        width = max(int(need.max()), 1) if width is None else width
        total = int(need.sum()) + spare
        ids = rng.permutation(total)
        table = np.full((rows, width), -1, dtype=np.int32)
        at = 0
        for r in range(rows):
            table[r, :need[r]] = ids[at:at + need[r]]
            at += need[r]
        shape = (total, page, heads, D) if order == "token" else (total, heads, page, D)
        self.k, self.v = (torch.full(shape, stale, dtype=dtype, device=dev) for _ in range(2))
        if order == "head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.table, self.page, self.heads, self.kv_heads, self.batch = table, page, heads, kv_heads, batch
        self.kv = []
        for x in range(batch * kv_heads):
            r, h = (x, 0) if apart else (x // kv_heads, x % kv_heads)
            k, v = (_random(rng, (self.lens[r], D), dtype, dev) for _ in range(2))
            pg, sl = self.slots(r, np.arange(self.lens[r]))
            self.k[pg, sl, h], self.v[pg, sl, h] = k, v
            self.kv.append((k, v))
        i32 = lambda a: torch.as_tensor(a, dtype=torch.int32).to(dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        extra = {}
        if ledger:
            cap = width * page
            w = np.where(rng.random((batch * kv_heads, cap)) < 0.05, 0.0, rng.exponential(size=(batch * kv_heads, cap)))
            # Positions: earlier evictions let later tokens take earlier slots.
            pos = np.stack([rng.permutation(cap) if r % 2 else np.arange(cap) for r in range(rows)])
            for r in range(rows):
                pos[r, :self.lens[r]] = rng.permutation(self.lens[r]) if r % 2 else np.arange(self.lens[r])
            extra = {"weights": torch.as_tensor(w, dtype=torch.float32).to(dev), "pos": i32(pos),
                     "dropped": i32(rng.integers(0, 50, rows))}
        self.pages = ops.Pages(self.k, self.v, i32(table), i32(self.lens), kv_heads, status=self.status, **extra)

    def slots(self, row, tok):
        dev = self.k.device
        tok = np.asarray(tok, dtype=np.int64)
        page = self.table[row, tok // self.page].astype(np.int64)
        return torch.as_tensor(page).to(dev), torch.as_tensor(tok % self.page).to(dev)

    def row(self, b, h):
        """Table row and head of its pages."""
        return (b * self.kv_heads + h, 0) if self.heads == 1 else (b, h)

    def read(self, b, h, n):
        r, hd = self.row(b, h)
        pg, sl = self.slots(r, np.arange(n))
        return self.k[pg, sl, hd], self.v[pg, sl, hd]


def queries(rng, batch, heads, tokens, dtype, dev):
    """[B, H, T, 128] as the projections leave it: heads seen first."""
    return _random(rng, (batch, tokens, heads, D), dtype, dev).transpose(1, 2)


def attend_causal(q, k, v, base, scale, dtype):
    """Queries [T, G, 128] of one row, query i over k, v [n, 128] below base + i
    + 1, in 64 bits: outputs [T, G, 128], their bound, every token's summed
    probability [n] and its bound.

    As serving_util.attend counts: a score's error of 129 roundings of its
    absolute terms, 8 of the score and the reference point; a probability by
    twice that, 2 ulp of exp2, and where it enters the product with V one
    rounding to the input type; a float32 rounding a term of the sums."""
    q, k, v = q.double(), k.double(), v.double()
    T, G, _ = q.shape
    n = k.shape[0]
    out, tol = torch.zeros_like(q), torch.full_like(q, 1e-30)
    w, wtol = torch.zeros(n, dtype=torch.float64, device=k.device), torch.zeros(n, dtype=torch.float64, device=k.device)
    u = half_step(dtype)
    for i in range(T):
        m = min(max(base + i + 1, 0), n)
        if m == 0:
            continue
        s = q[i] @ k[:m].t() * scale
        p = torch.softmax(s, dim=-1)
        out[i] = p @ v[:m]
        gap = F32 * (129 * (q[i].abs() @ k[:m].abs().t()) * scale + 8 * s.abs() + 8).amax(-1, keepdim=True) * 2
        tol[i] = ((p @ v[:m].abs()) * (u + 2 * gap + F32 * (2 * m + 64)) + rounding(out[i], dtype)) * 1.05
        w[:m] += p.sum(0)
        wtol[:m] += (p * (2 * gap + F32 * (2 * m + 64))).sum(0)
    return out, tol, w, wtol * 1.05 + F32 * (T * G + 8) * w


def evict_order(weights, pos, n, keep, sink, recent, dropped):
    """(slots that stay, where each slot below keep takes its token from) of a
    row, from its heads' weights [heads, >= n] and positions."""
    if n <= keep:
        return np.arange(n)
    score = weights[:, :n].astype(np.float64).sum(axis=0).astype(np.float32)
    score = np.where(np.isnan(score), -np.inf, score)
    nan = np.isnan(weights[:, :n].astype(np.float64).sum(axis=0))
    held = (pos[:n] < sink) | (pos[:n] >= n + dropped - recent)
    score, nan = np.where(held, 0.0, score), nan & ~held  # (protected tokens rank alike)
    stay = np.lexsort((np.arange(n), -score, nan, ~held))[:keep]
    free = np.setdiff1d(np.arange(keep), stay)
    src = np.arange(keep)
    src[free] = np.sort(stay[stay >= keep])
    return src
