"""What is timed of the serving operators on the ragged tiled store, and what their results have to be.

Three operators: the rotated append (position rotation of new queries and keys
with their store into the rows' tiles), attention of a batch over one shared
prefix and the sequences' own rows, and attention over the key blocks that a
score selects for each query.  Where `own` is false each is computed in its
plain form, where it is true by the calls a program makes of this package.
"""
import math

import numpy as np
import torch

own = False

D = 128
TILE = 32
SCALE = 1.0 / math.sqrt(D)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def listed():
    return [
        # One decode token of one sequence, one layer: launches count.
        {"name": "append-token", "op": "append", "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4, "tokens": 1,
         "start": 4091, "ragged": False, "tables": "model", "lens": 1},
        # A decode step of a batch in the loader's default type; every row at its own, odd length.
        {"name": "append-step", "op": "append", "dtype": "fp16", "batch": 64, "kv_heads": 4, "group": 7, "tokens": 1,
         "start": 2047, "ragged": True, "tables": "model", "lens": 2},
        # Question prompts of several lengths behind a shared document, padded to the longest.
        {"name": "append-questions", "op": "append", "dtype": "bf16", "batch": 8, "kv_heads": 8, "group": 4,
         "tokens": 509, "start": 33, "ragged": True, "tables": "fp32", "lens": 3},
        # A whole document prompt of one sequence.
        {"name": "append-document", "op": "append", "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4,
         "tokens": 32768, "start": 0, "ragged": False, "tables": "model", "lens": 4},
        # A few sequences a few tokens behind a short system prompt.
        {"name": "shared-chat", "op": "shared", "dtype": "fp32", "batch": 3, "kv_heads": 8, "group": 4, "queries": 1,
         "prefix": 1021, "suffix": 19, "ragged": True, "lens": 5},
        # A batch of questions over one document compressed per head: a ragged prefix.
        {"name": "shared-document", "op": "shared", "dtype": "bf16", "batch": 32, "kv_heads": 8, "group": 4,
         "queries": 1, "prefix": 32768, "suffix": 512, "ragged": True, "lens": 6},
        # Drafted tokens checked four at a time, grouped-query heads of seven.
        {"name": "shared-drafts", "op": "shared", "dtype": "fp16", "batch": 16, "kv_heads": 4, "group": 7,
         "queries": 4, "prefix": 12289, "suffix": 701, "ragged": False, "lens": 7},
        # The largest: a wide batch over a 128K prefix, long continuations.
        {"name": "shared-wide", "op": "shared", "dtype": "bf16", "batch": 128, "kv_heads": 8, "group": 4,
         "queries": 1, "prefix": 131072, "suffix": 2048, "ragged": True, "lens": 8},
        # One short sequence of full-KV heads.
        {"name": "blocks-4k", "op": "blocks", "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4, "queries": 1,
         "context": 4093, "block": 32, "keep": 16, "sink": 1, "local": 2, "build": False, "lens": 9},
        # One decode token over a 128K context, 2048 tokens kept.
        {"name": "blocks-128k", "op": "blocks", "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4, "queries": 1,
         "context": 131072, "block": 32, "keep": 64, "sink": 1, "local": 2, "build": False, "lens": 10},
        # A ragged batch with two drafted tokens a step.
        {"name": "blocks-batch", "op": "blocks", "dtype": "fp16", "batch": 24, "kv_heads": 4, "group": 7, "queries": 2,
         "context": 32003, "block": 64, "keep": 32, "sink": 1, "local": 1, "build": False, "lens": 11},
        # The step after a prompt: the blocks' bounds are built first.
        {"name": "blocks-build", "op": "blocks", "dtype": "bf16", "batch": 2, "kv_heads": 8, "group": 4, "queries": 1,
         "context": 65521, "block": 64, "keep": 48, "sink": 2, "local": 2, "build": True, "lens": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case no dearer than the largest listed one."""
    most = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        w = work(case)
        if all(w[x] <= max(m[x] for m in most) for x in ("bytes", "flops")):
            return case


def _draw(rng):
    op = rng.choice(("append", "shared", "blocks"))
    kv_heads, group = rng.choice(((8, 4), (8, 4), (4, 7), (8, 5), (2, 8), (16, 1), (1, 16)))
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "kv_heads": kv_heads, "group": group,
            "lens": rng.randrange(1 << 20)}
    if op == "append":
        batch = _log(rng, 1, 64)
        tokens = rng.choice((1, rng.randint(2, 40), _log(rng, 41, max(16384 // batch, 64))))
        case.update(batch=batch, tokens=tokens, start=rng.choice((0, _log(rng, 1, 4096))), ragged=rng.random() < 0.6,
                    tables=rng.choice(("model", "fp32")))
    elif op == "shared":
        batch = _log(rng, 1, 96)
        queries = rng.choice((1, 1, 1, 2, 5, 8))
        case.update(batch=batch, queries=queries, prefix=rng.choice((0, _log(rng, 1, 200), _log(rng, 200, 60000))),
                    suffix=_log(rng, queries, 1500), ragged=rng.random() < 0.6)
    else:
        batch = _log(rng, 1, 16)
        block = rng.choice((32, 32, 64, 128, 96))
        context = _log(rng, 20, 100000 // batch)
        sink, local = rng.randint(0, 2), rng.randint(1, 3)
        case.update(batch=batch, queries=rng.choice((1, 1, 1, 2, 4)), context=context, block=block,
                    keep=sink + local + _log(rng, 1, 80), sink=sink, local=local, build=rng.random() < 0.25)
    return case


# -- lengths, from the case alone ---------------------------------------------
def _append_lens(case):
    """Rows' lengths [batch, kv_heads] before the call and tokens appended a sequence [batch]."""
    rng = np.random.RandomState(case["lens"])
    b, h, t = case["batch"], case["kv_heads"], case["tokens"]
    if not case["ragged"]:
        return np.full((b, h), case["start"], dtype=np.int64), np.full(b, t, dtype=np.int64)
    start = rng.randint(0, case["start"] + 1, (b, h)).astype(np.int64)
    counts = rng.randint(t // 4, t + 1, b).astype(np.int64) if t > 1 else np.ones(b, dtype=np.int64)
    counts[0] = t
    return start, counts


def _shared_lens(case):
    """Prefix tokens of each head [kv_heads] and own tokens of each row [batch, kv_heads]."""
    rng = np.random.RandomState(case["lens"])
    b, h, p, s = case["batch"], case["kv_heads"], case["prefix"], case["suffix"]
    if not case["ragged"]:
        return np.full(h, p, dtype=np.int64), np.full((b, h), s, dtype=np.int64)
    heads = np.minimum((p * rng.uniform(0.2, 1.3, h)).astype(np.int64), p)
    own_len = np.repeat(rng.randint(min(case["queries"], s), s + 1, b), h).reshape(b, h).astype(np.int64)
    own_len[0] = s
    return heads, own_len


def _block_lens(case):
    """Tokens of each row [batch, kv_heads]."""
    rng = np.random.RandomState(case["lens"])
    b, h, n = case["batch"], case["kv_heads"], case["context"]
    lens = np.repeat(rng.randint(n // 3, n + 1, b), h).reshape(b, h).astype(np.int64)
    lens[0] = n
    return lens


# -- inputs -------------------------------------------------------------------
def _generator(seed, salt):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + salt)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _loud(g, kv_heads):
    """A gain per channel: four loud key channels a head, as trained models have them."""
    ch = torch.rand((kv_heads, D), generator=g, device=DEV).topk(4, dim=1).indices
    return torch.ones((kv_heads, D), device=DEV).scatter_(1, ch, 4.0)


def _tiles(lens, room):
    """First tile of each row, rows' capacities and the tiles of all rows of a store."""
    tiles = (np.asarray(lens).reshape(-1) + room + TILE - 1) // TILE
    off = np.concatenate([[0], np.cumsum(tiles)[:-1]]).astype(np.int64)
    return off, tiles * TILE, int(tiles.sum())


def _prepare_append(case, seed):
    g = _generator(seed, 1)
    b, h, t = case["batch"], case["kv_heads"], case["tokens"]
    hq, dt = h * case["group"], DTYPES[case["dtype"]]
    start, counts = _append_lens(case)
    off, cap, ntiles = _tiles(start, t + 5)
    # The projections' [batch, tokens, heads, 128], seen heads first.
    q = _randn(g, b, t, hq, D).to(dt).transpose(1, 2)
    k = (_randn(g, b, t, h, D) * _loud(g, h)).to(dt).transpose(1, 2)
    v = _randn(g, b, t, h, D).to(dt).transpose(1, 2)
    # Rotation tables as a model forms them: angles of the positions (the
    # sequence's own, which a compressed row's length lies below), then the
    # tables' type.
    pos = torch.as_tensor(start.max(axis=1) + 1000 * (seed % 7), device=DEV, dtype=torch.float64)[:, None]
    pos = pos + torch.arange(t, device=DEV, dtype=torch.float64)
    inv = 500000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    ang = pos[:, :, None] * inv
    tdt = dt if case["tables"] == "model" else torch.float32
    cos, sin = (torch.cat([f(ang)] * 2, dim=-1).to(tdt) for f in (torch.cos, torch.sin))
    kbuf = _randn(g, ntiles * TILE * D).to(dt)
    vbuf = _randn(g, ntiles * TILE * D).to(dt)
    as_dev = lambda a, d: torch.as_tensor(a, dtype=d).to(DEV)
    st = {"case": case, "q": q, "k": k, "v": v, "cos": cos, "sin": sin, "kbuf": kbuf, "vbuf": vbuf,
          "off": as_dev(off, torch.int64), "cap": as_dev(cap, torch.int32),
          "len": as_dev(start.reshape(-1), torch.int32),
          "counts": as_dev(counts, torch.int32) if case["ragged"] else None}
    st["len_out"] = torch.zeros_like(st["len"])
    st["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    return st


def _fill(lens, k, v, dtype, room=0):
    """A store whose row r holds the first lens[r] tokens of k[r] and v[r] ([rows, tokens, 128])."""
    from heterocache_amd.store import KVStore
    lens = np.asarray(lens).reshape(-1)
    store = KVStore([int(n) + room for n in lens], dtype, torch.device(DEV, torch.cuda.current_device()))
    rows = list(range(len(lens)))
    if lens.max(initial=0) > 0:
        store.write_rows(k[None], v[None], [(0, r) for r in rows], rows, lens)
    return store


def _prepare_shared(case, seed):
    g = _generator(seed, 2)
    b, h, n = case["batch"], case["kv_heads"], case["queries"]
    hq, dt = h * case["group"], DTYPES[case["dtype"]]
    plen, slen = _shared_lens(case)
    p, s = max(int(plen.max()), 1), max(int(slen.max()), 1)
    gain = _loud(g, h)
    lean = 0.5 * _randn(g, h, D)
    pk = _randn(g, h, p, D) * gain[:, None]
    pk[:, :4] = 3.0 * lean[:, None]       # sinks that every query leans to
    pv = _randn(g, h, p, D).to(dt)
    pk = pk.to(dt)
    sk = (_randn(g, b, h, s, D) * gain[:, None]).to(dt)
    sv = _randn(g, b, h, s, D).to(dt)
    q = _randn(g, b, n, h, case["group"], D) + lean[:, None]
    q = q.view(b, n, hq, D).to(dt).transpose(1, 2)
    st = {"case": case, "q": q}
    if own:
        st["prefix"] = _fill(plen, pk, pv, dt)
        st["rows"] = _fill(slen, sk.view(b * h, s, D), sv.view(b * h, s, D), dt, room=64)
    else:
        st.update(pk=pk, pv=pv, sk=sk, sv=sv, plen=torch.as_tensor(plen).to(DEV), slen=torch.as_tensor(slen).to(DEV))
    return st


def _prepare_blocks(case, seed):
    g = _generator(seed, 3)
    b, h, n = case["batch"], case["kv_heads"], case["queries"]
    hq, dt, size = h * case["group"], DTYPES[case["dtype"]], case["block"]
    lens = _block_lens(case)
    width = -(-int(lens.max()) // size) * size
    # Keys drift from topic to topic: a direction for each stretch of 80
    # tokens under the tokens' own noise.
    topics = _randn(g, b * h, width // 80 + 2, D)
    k = _randn(g, b * h, width, D)
    k += topics.repeat_interleave(80, dim=1)[:, 37:37 + width]
    k = (k * _loud(g, h).repeat(b, 1)[:, None]).to(dt)
    v = _randn(g, b * h, width, D).to(dt)
    q = _randn(g, b, n, h, case["group"], D) + _randn(g, b, 1, h, 1, D)
    q = q.view(b, n, hq, D).to(dt).transpose(1, 2)
    st = {"case": case, "q": q}
    if own:
        st["rows"] = _fill(lens, k, v, dt, room=64)
        st["index"] = st["rows"].block_index(size)
        if not case["build"]:
            st["index"].update()
    else:
        st.update(k=k, v=v, lens=torch.as_tensor(lens.reshape(-1)).to(DEV))
        if not case["build"]:
            st["bounds"] = _bounds(k, size)
    return st


def prepare(case, seed):
    return {"append": _prepare_append, "shared": _prepare_shared, "blocks": _prepare_blocks}[case["op"]](case, seed)


# -- plain forms --------------------------------------------------------------
def _rotate(x, cos, sin):
    x, cos, sin = x.float(), cos.float()[:, None], sin.float()[:, None]
    turned = torch.cat([-x[..., D // 2:], x[..., :D // 2]], dim=-1)
    return x * cos + turned * sin


def _plain_append(st):
    k = _rotate(st["k"], st["cos"], st["sin"]).to(st["k"].dtype)
    q = _rotate(st["q"], st["cos"], st["sin"]).to(st["q"].dtype)
    b, h, t, _ = k.shape
    # Tile element of (token of the tile, channel): K keeps 8 channels of a
    # token together, V 8 tokens of a channel.
    d = torch.arange(D, device=DEV)
    slot = st["len"].view(b, h, 1).long() + torch.arange(t, device=DEV)
    m = slot % TILE
    base = (st["off"].view(b, h, 1) + slot // TILE) * (TILE * D)
    kd = (d >> 5) * 512 + ((d >> 3) & 3) * 128 + (d & 7)
    vd = (d >> 4) * 512 + (d & 15) * 8
    at_k = (base + (m >> 4) * 2048 + (m & 15) * 8)[..., None] + kd
    at_v = (base + ((m & 15) >> 2) * 128 + ((m >> 4) * 4 + (m & 3)))[..., None] + vd
    v = st["v"]
    counts = st["counts"]
    if counts is None:
        st["kbuf"][at_k.reshape(-1)] = k.reshape(-1)
        st["vbuf"][at_v.reshape(-1)] = v.reshape(-1)
        st["len_out"].copy_(st["len"] + t)
    else:
        live = (torch.arange(t, device=DEV) < counts[:, None])[:, None].expand(b, h, t)
        st["kbuf"][at_k[live].reshape(-1)] = k[live].reshape(-1)
        st["vbuf"][at_v[live].reshape(-1)] = v[live].reshape(-1)
        st["len_out"].copy_(st["len"] + counts.repeat_interleave(h))
    return q, st["kbuf"], st["vbuf"], st["len_out"]


def _plain_shared(st):
    q, sk, sv, plen, slen = st["q"], st["sk"], st["sv"], st["plen"], st["slen"]
    b, hq, n, _ = q.shape
    h, s = sk.shape[1], sk.shape[2]
    grp = hq // h
    p = st["pk"].shape[1]
    out = torch.empty((b, n, hq, D), dtype=q.dtype, device=DEV)
    i = torch.arange(n, device=DEV)
    for j in range(h):
        qj = q[:, j * grp:(j + 1) * grp].float()                                  # [b, grp, n, D]
        lp = torch.matmul(qj.reshape(-1, D), st["pk"][j].float().t()) * SCALE
        lp = lp.masked_fill(torch.arange(p, device=DEV) >= plen[j], -math.inf).view(b, grp, n, p)
        seen = (slen[:, j, None] - n + 1 + i).clamp(min=0)                         # [b, n]
        own_keys = sk[:, j].float().transpose(1, 2).contiguous()
        ls = torch.matmul(qj.reshape(b, grp * n, D), own_keys).view(b, grp, n, s) * SCALE
        ls = ls.masked_fill(torch.arange(s, device=DEV) >= seen[:, None, :, None], -math.inf)
        top = torch.maximum(lp.amax(-1), ls.amax(-1))
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)[..., None]
        lp, ls = torch.exp(lp - top), torch.exp(ls - top)
        mass = lp.sum(-1) + ls.sum(-1)
        num = torch.matmul(lp.view(-1, p), st["pv"][j].float()).view(b, grp, n, D)
        num = num + torch.matmul(ls.view(b, grp * n, s), sv[:, j].float().contiguous()).view(b, grp, n, D)
        res = torch.where(mass[..., None] > 0, num / mass[..., None], torch.zeros_like(num))
        out[:, :, j * grp:(j + 1) * grp] = res.transpose(1, 2).to(q.dtype)
    return out


def _power(e):
    """2.0 ** e for int32 e in [-126, 127], exact."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(top):
    """The least e in [-48, 48] with top <= 127 * 2**e, as a float32 [..] -> int32 (-48 where top is 0)."""
    e = torch.frexp(top).exponent.to(torch.int32) - 7
    e = torch.where(top > 0, e, torch.full_like(e, -48)).clamp(-48, 48)
    return (e + ((top * _power(-e)) > 127).to(torch.int32)).clamp(max=48)


def _bounds(k, size):
    """Of every block of `size` keys: channel maxima rounded up and minima rounded down to
    whole multiples (-127..127) of 2**e, and e."""
    r, width, _ = k.shape
    blocks = k.view(r, width // size, size, D)
    hi, lo = blocks.amax(2).float(), blocks.amin(2).float()
    e = _exponent(torch.maximum(hi.abs().amax(-1), lo.abs().amax(-1)))
    down = _power(-e)[..., None]
    return torch.ceil(hi * down).clamp(-127, 127), torch.floor(lo * down).clamp(-127, 127), e


def _plain_blocks(st):
    case, q, k, v, lens = st["case"], st["q"], st["k"], st["v"], st["lens"]
    size, keep, sink, local = case["block"], case["keep"], case["sink"], case["local"]
    hi, lo, e = _bounds(k, size) if case["build"] else st["bounds"]
    b, hq, n, _ = q.shape
    r = k.shape[0]
    h = r // b
    grp = hq // h
    nb = hi.shape[1]
    # Queries in 8 bits: the nearest whole multiple of their head's power of two.
    qf = q.float().view(b, h, grp, n, D).transpose(2, 3).reshape(r, n, grp, D)
    eq = _exponent(qf.abs().amax(-1))
    q8 = torch.round(qf * _power(-eq)[..., None]).clamp(-127, 127).view(r, n * grp, D)
    # Whole numbers below 2**24: exact in float32 whatever the order.
    s = torch.matmul(q8.clamp(min=0), hi.transpose(1, 2).contiguous()) + torch.matmul(
        q8.clamp(max=0), lo.transpose(1, 2).contiguous())
    s = s.view(r, n, grp, nb) * _power(eq)[..., None] * _power(e)[:, None, None]
    s = s.amax(2)                                                                  # [r, n, nb]
    seen = (lens[:, None] - n + 1 + torch.arange(n, device=DEV)).clamp(min=0)      # [r, n]
    have = (seen + size - 1) // size
    j = torch.arange(nb, device=DEV)
    s = torch.where((j < sink) | (j >= have[..., None] - local), torch.full_like(s, math.inf), s)
    s = torch.where(j < have[..., None], s, torch.full_like(s, -math.inf))
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :keep]
    counts = have.clamp(max=keep)
    width = order.shape[-1]
    order = torch.where(torch.arange(width, device=DEV) < counts[..., None], order, torch.full_like(order, nb))
    order = torch.sort(order, dim=-1).values
    idx = torch.full((r, n, keep), -1, dtype=torch.int32, device=DEV)
    idx[..., :width] = torch.where(order < nb, order, torch.full_like(order, -1)).to(torch.int32)
    # Attention over the kept blocks' visible tokens.
    pos = (order.clamp(max=nb - 1)[..., None] * size + torch.arange(size, device=DEV)).view(r, n, width * size)
    live = ((order < nb)[..., None].expand(-1, -1, -1, size).reshape(r, n, -1)) & (pos < seen[..., None])
    row = torch.arange(r, device=DEV)[:, None, None]
    ks = k[row, pos].float().view(r * n, -1, D).transpose(1, 2).contiguous()
    logits = torch.matmul(qf.view(r * n, grp, D), ks) * SCALE
    logits = logits.masked_fill(~live.view(r * n, 1, -1), -math.inf)
    top = logits.amax(-1, keepdim=True)
    probs = torch.exp(logits - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    mass = probs.sum(-1, keepdim=True)
    vs = torch.where(live.view(r * n, -1, 1), v[row, pos].float().view(r * n, -1, D), torch.zeros((), device=DEV))
    res = torch.matmul(probs, vs)
    res = torch.where(mass > 0, res / mass, torch.zeros_like(res)).view(b, h, n, grp, D)
    out = res.permute(0, 2, 1, 3, 4).reshape(b, n, hq, D).to(q.dtype)
    return out, idx, counts.to(torch.int32)


# -- this package's calls -------------------------------------------------------
def _own_append(st):
    from heterocache_amd import ops
    q = ops.append_rotated(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["kbuf"], st["vbuf"], st["off"], st["len"],
                           st["cap"], counts=st["counts"], len_out=st["len_out"], status=st["status"])
    return q, st["kbuf"], st["vbuf"], st["len_out"]


def _own_shared(st):
    return st["rows"].attend_shared(st["q"], st["prefix"], SCALE)


def _own_blocks(st):
    case = st["case"]
    if case["build"]:
        st["index"].update()
    return st["rows"].attend_blocks(st["q"], st["index"], case["keep"], SCALE, sink=case["sink"], local=case["local"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "shared": _own_shared, "blocks": _own_blocks}[op](state)
    return {"append": _plain_append, "shared": _plain_shared, "blocks": _plain_blocks}[op](state)


# -- bytes and operations ---------------------------------------------------------
def work(case):
    esz = 4 if case["dtype"] == "fp32" else 2
    b, h, g = case["batch"], case["kv_heads"], case["group"]
    if case["op"] == "append":
        _, counts = _append_lens(case)
        t, n = case["tokens"], int(counts.sum())
        tables = 2 * b * t * D * (esz if case["tables"] == "model" else 4)
        # Every query is rotated, a padded batch's stored tokens alone are read of K and V.
        return {"bytes": 2 * b * t * h * g * D * esz + 4 * n * h * D * esz + tables + 8 * b * h,
                "flops": 3 * D * h * (b * t * g + n)}
    if case["op"] == "shared":
        plen, slen = _shared_lens(case)
        n = case["queries"]
        pairs = n * (b * int(plen.sum()) + int(slen.sum())) * g
        return {"bytes": (2 * int(plen.sum()) + 2 * int(slen.sum()) + 2 * b * n * h * g) * D * esz,
                "flops": 4 * D * pairs}
    lens, n, size = _block_lens(case), case["queries"], case["block"]
    blocks = int((lens // size).sum())
    seen = np.maximum(lens.reshape(-1, 1) - n + 1 + np.arange(n), 0)
    # The tokens a query attends: whole blocks and its last, partly visible one.
    full = np.minimum(seen, case["keep"] * size - (-seen) % size)
    build = int((lens // size * size).sum()) * D * esz if case["build"] else 0
    # Queries of a row may keep the same blocks: a row's longest is read at least.
    return {"bytes": 2 * int(full.max(axis=1).sum()) * D * esz + 2 * b * n * h * g * D * esz + blocks * (2 * D + 1) + build
            + 4 * b * h * n * (case["keep"] + 1),
            "flops": 4 * D * g * int(full.sum()) + 4 * D * g * n * blocks}


# -- 64-bit results, from the definitions ----------------------------------------
def _exact_append(st):
    case = st["case"]
    start, counts = _append_lens(case)
    h, half = case["kv_heads"], D // 2
    c, s = st["cos"].double()[:, None], st["sin"].double()[:, None]

    def turn(x):
        a, z = x.double().split(half, dim=-1)
        return torch.cat([a * c[..., :half] - z * s[..., :half], z * c[..., half:] + a * s[..., half:]], dim=-1)
    q, k, v = turn(st["q"]), turn(st["k"]), st["v"].double()
    # The tiles in natural order: [tile, token, channel].
    kn = st["kbuf"].double().view(-1, 2, 4, 4, 16, 8).permute(0, 1, 4, 2, 3, 5).reshape(-1, D).clone()
    vn = st["vbuf"].double().view(-1, 8, 4, 16, 2, 4).permute(0, 4, 2, 5, 1, 3).reshape(-1, D).clone()
    off = st["off"].tolist()
    for b in range(case["batch"]):
        for j in range(h):
            lo = off[b * h + j] * TILE + int(start[b, j])
            kn[lo:lo + counts[b]] = k[b, j, :counts[b]]
            vn[lo:lo + counts[b]] = v[b, j, :counts[b]]
    kt = kn.view(-1, 2, 16, 4, 4, 8).permute(0, 1, 3, 4, 2, 5).reshape(-1)
    vt = vn.view(-1, 2, 4, 4, 8, 16).permute(0, 4, 2, 5, 1, 3).reshape(-1)
    lens = torch.as_tensor((start + counts[:, None]).reshape(-1), dtype=torch.int32).to(DEV)
    return q, kt, vt, lens


def _exact_shared(st):
    case = st["case"]
    plen, slen = _shared_lens(case)
    q = st["q"].double()
    b, hq, n, _ = q.shape
    grp = case["group"]
    out = torch.zeros((b, n, hq, D), dtype=torch.float64, device=DEV)
    for j in range(case["kv_heads"]):
        pk, pv = st["pk"][j, :plen[j]].double(), st["pv"][j, :plen[j]].double()
        for x in range(b):
            m = int(slen[x, j])
            keys = torch.cat([pk, st["sk"][x, j, :m].double()])
            vals = torch.cat([pv, st["sv"][x, j, :m].double()])
            for i in range(n):
                upto = int(plen[j]) + max(m - n + 1 + i, 0)
                if upto == 0:
                    continue
                w = torch.softmax((q[x, j * grp:(j + 1) * grp, i] @ keys[:upto].t()) / math.sqrt(D), dim=-1)
                out[x, i, j * grp:(j + 1) * grp] = w @ vals[:upto]
    return out


def _exact_exponent(top):
    e = -48
    while e < 48 and top > 127.0 * 2.0 ** e:
        e += 1
    return e


def _exact_blocks(st):
    case = st["case"]
    lens = _block_lens(case).reshape(-1)
    size, keep, sink, local = case["block"], case["keep"], case["sink"], case["local"]
    q = st["q"].double()
    b, hq, n, _ = q.shape
    h, grp = case["kv_heads"], case["group"]
    out = torch.zeros((b, n, hq, D), dtype=torch.float64, device=DEV)
    idx = np.full((b * h, n, keep), -1, dtype=np.int32)
    counts = np.zeros((b * h, n), dtype=np.int32)
    for r in range(b * h):
        x, j = r // h, r % h
        m = int(lens[r])
        keys, vals = st["k"][r, :m].double(), st["v"][r, :m].double()
        done = m // size
        cut = keys[:done * size].view(done, size, D)
        hi, lo = (cut.amax(1).cpu().numpy(), cut.amin(1).cpu().numpy()) if done else (np.zeros((0, D)),) * 2
        top = np.maximum(np.abs(hi).max(axis=1), np.abs(lo).max(axis=1)) if done else np.zeros(0)
        e = np.array([_exact_exponent(t) for t in top], dtype=np.float64)
        unit = np.exp2(e)[:, None]
        hi, lo = np.clip(np.ceil(hi / unit), -127, 127), np.clip(np.floor(lo / unit), -127, 127)
        for i in range(n):
            seen = max(m - n + 1 + i, 0)
            have = -(-seen // size)
            head = q[x, j * grp:(j + 1) * grp, i]
            if have <= keep:
                chosen = np.arange(have)
            else:
                qn = head.cpu().numpy()
                score = np.full(have, -np.inf)
                for row in qn:
                    eq = 2.0 ** _exact_exponent(np.abs(row).max())
                    q8 = np.clip(np.rint(row / eq), -127, 127)
                    # The middle blocks are complete.
                    mid = slice(sink, have - local)
                    val = np.maximum(q8 * hi[mid], q8 * lo[mid]).sum(axis=1) * eq * unit[mid, 0]
                    score[mid] = np.maximum(score[mid], val)
                score[:sink] = np.inf
                score[have - local:] = np.inf
                chosen = np.sort(np.lexsort((np.arange(have), -score))[:keep])
            counts[r, i] = len(chosen)
            idx[r, i, :len(chosen)] = chosen
            if len(chosen) == 0:
                continue
            pos = (chosen[:, None] * size + np.arange(size)).reshape(-1)
            pos = torch.as_tensor(pos[pos < seen]).to(DEV)
            w = torch.softmax((head @ keys[pos].t()) / math.sqrt(D), dim=-1)
            out[x, i, j * grp:(j + 1) * grp] = w @ vals[pos]
    return out, torch.as_tensor(idx).to(DEV), torch.as_tensor(counts).to(DEV)


def exact(case, seed):
    global own
    if case["op"] == "shared" and case["batch"] * case["kv_heads"] * case["queries"] > 4096:
        return None
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "shared": _exact_shared, "blocks": _exact_blocks}[case["op"]](st)
