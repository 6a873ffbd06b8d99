"""What is timed of the paged cache's operators, and what their results have to be.

Three operators on pools of pages [pages, page tokens, heads, 128] reached
through tables: new tokens stored and attended over the cache ("chunk"), the
same with every cached token's share of the attention added to its weight
("weigh"), and the eviction of the lightest tokens ("evict").  A table serves
one (sequence, KV head) row, or all KV heads of a sequence.  Where `own` is
false each is computed in its plain form, where it is true by the calls a
program makes of this package.
"""
import math

import numpy as np
import torch

own = False

D = 128
SCALE = 1.0 / math.sqrt(D)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def listed():
    return [
        # One decode token of one short sequence, one layer: launches count.
        {"name": "chunk-token", "op": "chunk", "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4, "tokens": 1,
         "context": 4091, "page": 16, "apart": False, "ragged": False, "lens": 1},
        # A decode step of a serving batch in the loader's default type, sequences of all lengths.
        {"name": "chunk-step", "op": "chunk", "dtype": "fp16", "batch": 48, "kv_heads": 4, "group": 7, "tokens": 1,
         "context": 16384, "page": 64, "apart": False, "ragged": True, "lens": 2},
        # A mixed batch, padded: some sequences bring a token, some a short prompt; a table a head, pages of 256.
        {"name": "chunk-mixed", "op": "chunk", "dtype": "bf16", "batch": 12, "kv_heads": 8, "group": 4, "tokens": 33,
         "context": 8191, "page": 256, "apart": True, "ragged": True, "lens": 3},
        # The largest: a long prompt's later chunk.
        {"name": "chunk-prompt", "op": "chunk", "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4, "tokens": 2048,
         "context": 63488, "page": 64, "apart": False, "ragged": False, "lens": 4},
        # Full precision, a page size that is no power of two.
        {"name": "chunk-fp32", "op": "chunk", "dtype": "fp32", "batch": 2, "kv_heads": 8, "group": 4, "tokens": 251,
         "context": 2801, "page": 48, "apart": False, "ragged": True, "lens": 5},
        # One decode token over a 128K context whose heads keep different numbers of tokens.
        {"name": "weigh-token", "op": "weigh", "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4, "tokens": 1,
         "context": 131071, "page": 256, "apart": True, "ragged": True, "lens": 6},
        # A decode step of a batch held to 2048 tokens a head.
        {"name": "weigh-step", "op": "weigh", "dtype": "fp16", "batch": 16, "kv_heads": 4, "group": 7, "tokens": 1,
         "context": 2111, "page": 64, "apart": True, "ragged": False, "lens": 7},
        # Prompts' chunks that weigh what the cache holds.
        {"name": "weigh-chunk", "op": "weigh", "dtype": "bf16", "batch": 4, "kv_heads": 8, "group": 4, "tokens": 509,
         "context": 8003, "page": 32, "apart": False, "ragged": True, "lens": 8},
        # One sequence's heads give up one token a step each.
        {"name": "evict-one", "op": "evict", "dtype": "bf16", "batch": 1, "kv_heads": 8, "context": 1025, "keep": 1024,
         "sink": 4, "recent": 32, "page": 16, "apart": True, "ragged": False, "lens": 9},
        # A batch's heads give up 64 tokens every 64 steps.
        {"name": "evict-step", "op": "evict", "dtype": "fp16", "batch": 16, "kv_heads": 8, "context": 2112,
         "keep": 2048, "sink": 4, "recent": 256, "page": 64, "apart": True, "ragged": False, "lens": 10},
        # All heads of a sequence together, ragged, down to half.
        {"name": "evict-together", "op": "evict", "dtype": "bf16", "batch": 8, "kv_heads": 8, "context": 8190,
         "keep": 4096, "sink": 4, "recent": 512, "page": 64, "apart": False, "ragged": True, "lens": 11},
        # A long prompt, each head down to its own budget.
        {"name": "evict-prompt", "op": "evict", "dtype": "bf16", "batch": 1, "kv_heads": 8, "context": 131072,
         "keep": 32768, "sink": 4, "recent": 1024, "page": 256, "apart": True, "ragged": True, "lens": 12},
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
    op = rng.choice(("chunk", "chunk", "weigh", "evict"))
    kv_heads, group = rng.choice(((8, 4), (8, 4), (4, 7), (8, 5), (2, 8), (16, 1), (1, 16)))
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "kv_heads": kv_heads,
            "page": rng.choice((16, 16, 32, 64, 256, 48, _log(rng, 1, 300))), "apart": rng.random() < 0.5,
            "ragged": rng.random() < 0.6, "lens": rng.randrange(1 << 20)}
    if op == "evict":
        batch = _log(rng, 1, 16)
        context = _log(rng, 40, 131072 // batch)
        keep = max(int(context * rng.choice((rng.uniform(0.05, 1.0), 1 - 64 / max(context, 100)))), 8)
        case.update(batch=batch, context=context, keep=keep, sink=rng.choice((0, 4)),
                    recent=rng.choice((0, _log(rng, 1, max(keep // 2, 1)))))
        case["sink"] = min(case["sink"], keep - case["recent"])
        return case
    batch = _log(rng, 1, 32)
    tokens = rng.choice((1, 1, rng.randint(2, 40), _log(rng, 41, max(1024 // batch, 64))))
    case.update(batch=batch, group=group, tokens=tokens,
                context=rng.choice((0, _log(rng, 1, 300), _log(rng, 300, 100000 // batch))))
    return case


# -- lengths, from the case alone ---------------------------------------------
def _rows(case):
    """Table rows of a sequence, and KV heads of a table row."""
    return (case["kv_heads"], 1) if case["apart"] else (1, case["kv_heads"])


def _lens(case):
    """Tokens of each table row [batch, rows] before the call, and new tokens a sequence [batch]."""
    rng = np.random.RandomState(case["lens"])
    b, r, n = case["batch"], _rows(case)[0], case["context"]
    t = case.get("tokens", 0)
    if not case["ragged"]:
        return np.full((b, r), n, dtype=np.int64), np.full(b, t, dtype=np.int64)
    lens = rng.randint(n // 4, n + 1, (b, r)).astype(np.int64)
    lens[0, 0] = n
    counts = np.where(rng.rand(b) < 0.5, rng.randint(0, t + 1, b), min(t, 1)).astype(np.int64)
    counts[0] = t
    return lens, counts


def _keeps(case):
    """Budget of each table row [batch, rows]."""
    rng = np.random.RandomState(case["lens"] + 1)
    shape = (case["batch"], _rows(case)[0])
    if not case["ragged"]:
        return np.full(shape, case["keep"], dtype=np.int64)
    low = max(case["keep"] // 2, case["sink"] + case["recent"])
    keep = rng.randint(low, case["keep"] + 1, shape).astype(np.int64)
    keep[0, 0] = case["keep"]
    return keep


# -- inputs -------------------------------------------------------------------
def _generator(seed, salt):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + salt)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _loud(g, kv_heads):
    """A gain per channel: four loud key channels a head, as trained models have them."""
    ch = torch.rand((kv_heads, D), generator=g, device=DEV).topk(4, dim=1).indices
    return torch.ones((kv_heads, D), device=DEV).scatter_(1, ch, 4.0)


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32).to(DEV)


def _pool(case, g, room):
    """Pools, tables and lengths of a cache in use: pages lie in any order and a few are free."""
    b, r = case["batch"], _rows(case)[0]
    h, size, dt = case["kv_heads"], case["page"], DTYPES[case["dtype"]]
    lens, _ = _lens(case)
    width = max(-(-(int(lens.max()) + room) // size), 1)          # a table row's entries
    used = -(-(lens.reshape(-1) + room) // size)
    total = int(used.sum()) + 7
    heads = _rows(case)[1]
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b * r, width), -1, dtype=torch.int32, device=DEV)
    live = torch.arange(width, device=DEV) < torch.as_tensor(used).to(DEV)[:, None]
    table[live] = order[:int(used.sum())]
    # A page's tokens of one head lie together; seen [pages, page tokens, heads, 128].
    gain = _loud(g, h)
    k = _randn(g, total, heads, size, D)
    if heads == h:
        k *= gain[None, :, None]
    k = k.to(dt).transpose(1, 2)
    v = _randn(g, total, heads, size, D).to(dt).transpose(1, 2)
    return {"case": case, "k": k, "v": v, "table": table, "len": _i32(lens.reshape(-1)), "gain": gain, "width": width * size}


def _prepare_attn(case, seed):
    g = _generator(seed, 1)
    b, h, t, n = case["batch"], case["kv_heads"], case["tokens"], case["group"]
    dt = DTYPES[case["dtype"]]
    lens, counts = _lens(case)
    st = _pool(case, g, t)
    lean = 0.5 * _randn(g, h, D)
    # The projections' [batch, tokens, heads, 128], seen heads first.
    q = _randn(g, b, t, h, n, D) + lean[:, None]
    st["q"] = q.view(b, t, h * n, D).to(dt).transpose(1, 2)
    k = _randn(g, b, t, h, D) * st["gain"]
    # New tokens of a prompt's start are sinks that every query leans to.
    if case["context"] == 0:
        k[:, 0] = 3.0 * lean
    st["k_new"] = k.to(dt).transpose(1, 2)
    st["v_new"] = _randn(g, b, t, h, D).to(dt).transpose(1, 2)
    st["counts"] = _i32(counts) if case["ragged"] else None
    st["len_out"] = torch.zeros_like(st["len"])
    if case["op"] == "weigh":
        st["weights"] = torch.exp(1.5 * _randn(g, b * h, st["width"]) - 3.0)
        st["pos"] = _positions(case, g, st["width"], lens)
        st["dropped"] = _i32(np.random.RandomState(case["lens"] + 2).randint(0, 1000, lens.size))
        st["weights_out"] = torch.zeros_like(st["weights"])
    if own:
        st["pages"] = _pages(st)
    return st


def _positions(case, g, width, lens, total=None):
    """Positions of the tokens a row holds: some were dropped before, and later ones took their slots."""
    rows = lens.size
    pos = torch.arange(width, device=DEV).repeat(rows, 1)
    n = torch.as_tensor(lens.reshape(-1, 1)).to(DEV)
    shuffled = torch.rand((rows, width), generator=g, device=DEV)
    few = torch.rand((rows, width), generator=g, device=DEV) < 0.2
    # Of a fifth of the slots the tokens change places within the row.
    key = torch.where(few & (pos < n), shuffled, torch.full_like(shuffled, 2.0)).argsort(dim=1, stable=True)
    rank = (few & (pos < n)).long().cumsum(1) - 1
    moved = pos.gather(1, key.gather(1, rank.clamp(min=0)))
    return torch.where(few & (pos < n), moved, pos).to(torch.int32)


def _prepare_evict(case, seed):
    g = _generator(seed, 2)
    b, h = case["batch"], case["kv_heads"]
    lens, _ = _lens(case)
    st = _pool(case, g, 0)
    w = torch.exp(2.0 * _randn(g, b * h, st["width"]) - 3.0)
    # Tokens that nothing attends yet weigh zero: ties.
    st["weights"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.02, torch.zeros_like(w), w)
    st["pos"] = _positions(case, g, st["width"], lens)
    st["dropped"] = torch.zeros_like(st["len"])
    st["keep"] = _i32(_keeps(case).reshape(-1))
    st["len_out"], st["dropped_out"] = torch.zeros_like(st["len"]), torch.zeros_like(st["len"])
    st["weights_out"], st["pos_out"] = torch.zeros_like(st["weights"]), torch.zeros_like(st["pos"])
    if own:
        st["pages"] = _pages(st)
    return st


def prepare(case, seed):
    return _prepare_evict(case, seed) if case["op"] == "evict" else _prepare_attn(case, seed)


# -- plain forms --------------------------------------------------------------
def _slots(st, rows, tok):
    """Pages and places in them of tokens `tok` of table rows `rows`; entries past a row's pages are not followed."""
    size = st["case"]["page"]
    return st["table"][rows, tok // size].long().clamp(min=0), tok % size


def _plain_attn(st):
    case, q, table = st["case"], st["q"], st["table"]
    b, hq, t, _ = q.shape
    h, (per, heads) = case["kv_heads"], _rows(case)
    grp, weigh = case["group"], case["op"] == "weigh"
    n = st["counts"].long() if st["counts"] is not None else torch.full((b,), t, device=DEV)
    lens = st["len"].view(b, per).long()
    # Store the new tokens.
    i = torch.arange(t, device=DEV)
    for r in range(per):
        live = (i < n[:, None])
        at = (lens[:, r, None] + i)[live]
        seq = torch.arange(b, device=DEV)[:, None].expand(b, t)[live]
        page, slot = _slots(st, seq * per + r, at)
        for name in ("k", "v"):
            new = st[name + "_new"].transpose(1, 2)[live]                        # [new tokens, h, D]
            st[name][page, slot] = new if heads > 1 or h == 1 else new[:, r:r + 1]
        if weigh:
            st["pos"][seq * per + r, at] = (at + st["dropped"][seq * per + r]).to(torch.int32)
    total = lens + n[:, None]
    st["len_out"].copy_(total.reshape(-1))
    longest = int(st["width"])
    out = torch.empty((b, t, hq, D), dtype=q.dtype, device=DEV)
    j = torch.arange(longest, device=DEV)
    real = (i < n[:, None])                                                      # [b, t]
    for x in range(h):
        r = x if per > 1 else 0
        rows = torch.arange(b, device=DEV) * per + r
        page, slot = _slots(st, rows[:, None].expand(b, longest), j.expand(b, longest))
        head = x if heads > 1 else 0
        held = (j < total[:, r, None])[..., None]
        ks = torch.where(held, st["k"][page, slot, head].float(), torch.zeros((), device=DEV))   # [b, tokens, D]
        vs = torch.where(held, st["v"][page, slot, head].float(), torch.zeros((), device=DEV))
        qx = q[:, x * grp:(x + 1) * grp].float().reshape(b, grp * t, D)
        s = torch.matmul(qx, ks.transpose(1, 2).contiguous()).view(b, grp, t, longest) * SCALE
        seen = torch.where(real, lens[:, r, None] + i + 1, torch.zeros_like(i))  # [b, t]
        s.masked_fill_(j >= seen[:, None, :, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        s = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        mass = s.sum(-1, keepdim=True)
        s = s / torch.where(mass > 0, mass, torch.ones_like(mass))
        o = torch.matmul(s.view(b, grp * t, longest), vs).view(b, grp, t, D)
        out[:, :, x * grp:(x + 1) * grp] = o.transpose(1, 2).to(q.dtype)
        if weigh:
            rows_w = torch.arange(b, device=DEV) * h + x
            old = torch.where(j < lens[:, r, None], st["weights"][rows_w], torch.zeros((), device=DEV))
            got = old + s.sum((1, 2))
            st["weights_out"][rows_w] = torch.where(held[..., 0], got, st["weights_out"][rows_w])
    if weigh:
        return out, st["k"], st["v"], st["len_out"], st["weights_out"], st["pos"]
    return out, st["k"], st["v"], st["len_out"]


def _plain_evict(st):
    case = st["case"]
    h, (per, heads) = case["kv_heads"], _rows(case)
    n, keep, drop = st["len"].long()[:, None], st["keep"].long()[:, None], st["dropped"].long()[:, None]
    rows, width = st["pos"].shape
    slot = torch.arange(width, device=DEV).expand(rows, width)
    pos = st["pos"].long()
    score = st["weights"].view(rows, heads, width).double().sum(1).float()
    held = (pos < case["sink"]) | (pos >= n + drop - case["recent"])
    score = torch.where(held, torch.full_like(score, math.inf), score)
    score = torch.where(slot < n, score, torch.full_like(score, -math.inf))
    order = torch.sort(score, dim=1, descending=True, stable=True).indices
    new = torch.minimum(n, keep)
    kept = torch.zeros((rows, width), dtype=torch.bool, device=DEV).scatter_(1, order, slot < new)
    free = (~kept & (slot < new)).nonzero()
    come = (kept & (slot >= new)).nonzero()
    to_page, to_slot = _slots(st, free[:, 0], free[:, 1])
    of_page, of_slot = _slots(st, come[:, 0], come[:, 1])
    st["k"][to_page, to_slot] = st["k"][of_page, of_slot]
    st["v"][to_page, to_slot] = st["v"][of_page, of_slot]
    live = slot < new
    src = slot.clone()
    src[free[:, 0], free[:, 1]] = come[:, 1]
    st["pos_out"].copy_(torch.where(live, st["pos"].gather(1, src), st["pos_out"]))
    src, live = src.repeat_interleave(heads, dim=0), live.repeat_interleave(heads, dim=0)
    st["weights_out"].copy_(torch.where(live, st["weights"].gather(1, src), st["weights_out"]))
    st["len_out"].copy_(new[:, 0])
    st["dropped_out"].copy_((drop + n - new)[:, 0])
    return st["k"], st["v"], st["len_out"], st["weights_out"], st["pos_out"], st["dropped_out"]


# -- this package's calls -------------------------------------------------------
def _pages(st):
    from heterocache_amd import ops
    ledger = {x: st[x] for x in ("weights", "pos", "dropped")} if "weights" in st else {}
    return ops.Pages(st["k"], st["v"], st["table"], st["len"], st["case"]["kv_heads"], **ledger)


def _own_attn(st):
    from heterocache_amd import ops
    if st["case"]["op"] == "weigh":
        out = ops.paged_attn(st["q"], st["pages"], SCALE, st["k_new"], st["v_new"], counts=st["counts"], weigh=True,
                             len_out=st["len_out"], weights_out=st["weights_out"])
        return out, st["k"], st["v"], st["len_out"], st["weights_out"], st["pos"]
    out = ops.paged_attn(st["q"], st["pages"], SCALE, st["k_new"], st["v_new"], counts=st["counts"],
                         len_out=st["len_out"])
    return out, st["k"], st["v"], st["len_out"]


def _own_evict(st):
    from heterocache_amd import ops
    case = st["case"]
    ops.paged_evict(st["pages"], st["keep"], sink=case["sink"], recent=case["recent"], len_out=st["len_out"],
                    weights_out=st["weights_out"], pos_out=st["pos_out"], dropped_out=st["dropped_out"])
    return st["k"], st["v"], st["len_out"], st["weights_out"], st["pos_out"], st["dropped_out"]


def run(state):
    evict = state["case"]["op"] == "evict"
    if own:
        return _own_evict(state) if evict else _own_attn(state)
    return _plain_evict(state) if evict else _plain_attn(state)


# -- bytes and operations ---------------------------------------------------------
def work(case):
    esz = 4 if case["dtype"] == "fp32" else 2
    lens, counts = _lens(case)
    h, (per, heads) = case["kv_heads"], _rows(case)
    if case["op"] == "evict":
        keep = np.minimum(lens, _keeps(case))
        # Tokens that have to move: those kept behind the budget, were the weights spread evenly.
        share = keep / np.maximum(lens, 1)
        moved = int(((lens - keep) * share).sum())
        return {"bytes": 4 * int(lens.sum()) * (heads + 1) + 4 * int(keep.sum()) * (heads + 1) + 4 * D * esz * moved * heads,
                "flops": int(lens.sum()) * heads}
    g, t, b = case["group"], case["tokens"], case["batch"]
    rows = heads * int(lens.sum())
    fresh = int(counts.sum()) * h
    pairs = g * int((lens * counts[:, None]).sum()) * heads + g * h * int((counts * (counts + 1) // 2).sum())
    out = {"bytes": 2 * D * esz * (rows + 2 * fresh) + D * esz * g * (fresh + b * t * h), "flops": 4 * D * pairs}
    if case["op"] == "weigh":
        out["bytes"] += 8 * rows + 4 * fresh + 4 * int(counts.sum()) * per
        out["flops"] += pairs
    return out


# -- 64-bit results, from the definitions ----------------------------------------
def _exact_attn(st):
    case = st["case"]
    lens, counts = _lens(case)
    h, grp, size, per = case["kv_heads"], case["group"], case["page"], _rows(case)[0]
    weigh = case["op"] == "weigh"
    q = st["q"].double()
    b, hq, t, _ = q.shape
    table = st["table"].cpu().numpy()
    k, v = st["k"].double(), st["v"].double()
    out = torch.zeros((b, t, hq, D), dtype=torch.float64, device=DEV)
    w_out = st["weights_out"].double() if weigh else None
    pos = st["pos"].cpu().numpy().copy() if weigh else None
    dropped = st["dropped"].cpu().numpy() if weigh else None
    for s in range(b):
        n = int(counts[s])
        for x in range(h):
            row, head = (s * h + x, 0) if per > 1 else (s, x)
            have = int(lens[s, x if per > 1 else 0])
            at = np.arange(have + n)
            page, slot = torch.as_tensor(table[row, at // size].astype(np.int64)).to(DEV), torch.as_tensor(at % size).to(DEV)
            k[page[have:], slot[have:], head] = st["k_new"][s, x, :n].double()
            v[page[have:], slot[have:], head] = st["v_new"][s, x, :n].double()
            if weigh:
                pos[row, have:have + n] = np.arange(have, have + n) + dropped[row]
                w_out[s * h + x, :have] = st["weights"][s * h + x, :have].double()
                w_out[s * h + x, have:have + n] = 0.0
            if n == 0:
                continue
            keys, vals = k[page, slot, head], v[page, slot, head]
            hide = torch.arange(have + n, device=DEV) > have + torch.arange(n, device=DEV)[:, None]
            for j in range(x * grp, (x + 1) * grp):
                p = torch.softmax((q[s, j, :n] @ keys.t() / math.sqrt(D)).masked_fill(hide, -math.inf), dim=-1)
                out[s, :n, j] = p @ vals
                if weigh:
                    w_out[s * h + x, :have + n] += p.sum(0)
    new = torch.as_tensor((lens + counts[:, None]).reshape(-1), dtype=torch.int32).to(DEV)
    if weigh:
        return out, k, v, new, w_out, torch.as_tensor(pos).to(DEV)
    return out, k, v, new


def _exact_evict(st):
    case = st["case"]
    lens, keeps = _lens(case)[0].reshape(-1), _keeps(case).reshape(-1)
    heads, size = _rows(case)[1], case["page"]
    w = st["weights"].cpu().numpy()
    pos, table, dropped = (st[x].cpu().numpy() for x in ("pos", "table", "dropped"))
    k, v = st["k"].double(), st["v"].double()
    w_out, pos_out = st["weights_out"].double().cpu().numpy(), st["pos_out"].cpu().numpy().copy()
    new_len, new_drop = lens.copy(), dropped.copy()
    for r, (n, keep) in enumerate(zip(lens.tolist(), keeps.tolist())):
        mine = slice(r * heads, (r + 1) * heads)
        at = np.arange(n)
        if n > keep:
            score = w[mine, :n].astype(np.float64).sum(axis=0).astype(np.float32)
            held = (pos[r, :n] < case["sink"]) | (pos[r, :n] >= n + int(dropped[r]) - case["recent"])
            order = np.lexsort((at, -score, ~held))
            stay = np.sort(order[:keep])
            free = np.setdiff1d(np.arange(keep), stay)
            come = stay[stay >= keep]
            at = np.arange(keep)
            at[free] = come
            to, of = (torch.as_tensor(x.astype(np.int64)).to(DEV) for x in (table[r, free // size], table[r, come // size]))
            to_s, of_s = torch.as_tensor(free % size).to(DEV), torch.as_tensor(come % size).to(DEV)
            k[to, to_s], v[to, to_s] = k[of, of_s], v[of, of_s]
            new_len[r], new_drop[r] = keep, dropped[r] + n - keep
        w_out[mine, :len(at)] = w[mine][:, at]
        pos_out[r, :len(at)] = pos[r, at]
    i32 = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32).to(DEV)
    return k, v, i32(new_len), torch.as_tensor(w_out).to(DEV), i32(pos_out), i32(new_drop)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return _exact_evict(st) if case["op"] == "evict" else _exact_attn(st)
