"""Paged KV cache of one layer: rows that grow and shrink by pages.

The reference keeps a layer's cache in pools of pages behind block tables, a
table a (sequence, KV head) row (`key_pools` / `value_pools` / `block_tables` /
`heads_len`, heterocache/cache_utils.py:693-766), each row's pages allocated
for its whole lifetime.  Here pages come from a common list when a row needs
them and return to it when a row gives tokens up or ends, so sequences of
unknown length share the memory of a pool.  KVStore, whose rows are contiguous,
reads faster and stays the store of rows whose size is known.
"""
import numpy as np
import torch

from . import _lib, ops

HEAD_DIM = ops.HEAD_DIM


class PagedStore:
    """Pools, tables and lengths of one layer, with the list of free pages.

    batch sequences of kv_heads KV heads; `pages` pages of page_tokens tokens
    (of all heads; with per_head=True of one head, and every head has a table of
    its own, so its rows may be held to different lengths); a row holds at most
    max_tokens.  track=True keeps what evict goes by: every token's accumulated
    attention weight, its position, and the tokens that a row has given up.

    `host_len` bounds the rows' lengths on the host (exact unless counts were
    given on the device or calls captured): pages are reserved by it, the
    kernels read the lengths on the device.  Pages are handed out in host order:
    calls that use one store go to one stream, or are ordered by the caller.
    """

    def __init__(self, batch, kv_heads, pages, dtype, device, max_tokens, page_tokens=64, per_head=False, track=False,
                 layer_idx=None):
        batch, kv_heads, pages, page_tokens = int(batch), int(kv_heads), int(pages), int(page_tokens)
        if min(batch, kv_heads, pages, page_tokens, int(max_tokens)) < 1:
            raise ValueError(f"batch={batch} kv_heads={kv_heads} pages={pages} page_tokens={page_tokens} "
                             f"max_tokens={max_tokens}")
        self.batch, self.kv_heads, self.page_tokens, self.layer_idx = batch, kv_heads, page_tokens, layer_idx
        self.dtype, self.device = dtype, torch.device(device)
        self.per_sequence = kv_heads if per_head else 1  # table rows of a sequence
        self.rows = batch * self.per_sequence
        heads = 1 if per_head else kv_heads
        width = -(-int(max_tokens) // page_tokens)
        self.capacity = width * page_tokens
        # A head's tokens of a page lie together; seen [pages, page_tokens, heads, 128].
        shape = (pages, heads, page_tokens, HEAD_DIM)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=self.device).transpose(1, 2) for _ in range(2))
        i32 = lambda *n, fill=0: torch.full(n, fill, dtype=torch.int32, device=self.device)
        self.table, self.row_len, self.status = i32(self.rows, width, fill=-1), i32(self.rows), i32(1)
        ledger = {}
        if track:
            ledger = {"weights": torch.zeros((batch * kv_heads, self.capacity), dtype=torch.float32, device=self.device),
                      "pos": i32(self.rows, self.capacity), "dropped": i32(self.rows)}
        self.pages = ops.Pages(self.k, self.v, self.table, self.row_len, kv_heads, status=self.status, **ledger)
        self.host_len = np.zeros(self.rows, dtype=np.int64)
        self._along = None                                   # the same along a graph that is being captured
        self.held = np.zeros(self.rows, dtype=np.int64)      # pages of each row
        self._ids = np.full((self.rows, width), -1, dtype=np.int32)
        self._free = list(range(pages - 1, -1, -1))          # the next page is the last

    @property
    def free_pages(self):
        return len(self._free)

    # -- lengths ---------------------------------------------------------------
    def _bound(self):
        """Bound of the lengths ahead of a call on the current stream."""
        if not torch.cuda.is_current_stream_capturing():
            self._along = None
        return self.host_len if self._along is None else self._along

    def _advance(self, lens):
        """The lengths behind a call.  One that is captured has not run: the host's bound falls with none, and holds
        at every point of the first replay."""
        if torch.cuda.is_current_stream_capturing():
            self._along, lens = lens, np.maximum(self.host_len, lens)
        self.host_len = lens

    # -- pages ---------------------------------------------------------------
    def _oom(self):
        name = "?" if self.layer_idx is None else self.layer_idx
        return RuntimeError(f"Layer {name} OOM.")

    def reserve(self, tokens):
        """Pages for `tokens` more tokens in every row (or one number a
        sequence).  Appending calls do it by themselves; a call that is
        captured in a graph needs its replays' pages reserved before.  Raises
        the reference's "Layer i OOM." when a row would pass max_tokens or the
        pool has no page left (heterocache/cache_utils.py:988-990)."""
        more = np.asarray(tokens, dtype=np.int64)
        if (more < 0).any():
            raise ValueError(f"tokens={tokens}")
        self._reserve(self._bound() + (np.repeat(more, self.per_sequence) if more.ndim else more))

    def _reserve(self, lens):
        need = -(-lens // self.page_tokens)
        if not (need > self.held).any():
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages are reserved before a call is captured (PagedStore.reserve)")
        if (lens > self.capacity).any() or int(np.maximum(need - self.held, 0).sum()) > len(self._free):
            raise self._oom()
        at, ids = [], []
        for r in np.nonzero(need > self.held)[0]:
            for j in range(self.held[r], need[r]):
                self._ids[r, j] = self._free.pop()
                at.append(r * self._ids.shape[1] + j)
                ids.append(self._ids[r, j])
            self.held[r] = need[r]
        self._write(at, ids)

    def _write(self, at, ids):
        """Table entries, on the current stream."""
        at = ops.host_counts("a page table", np.asarray(at, dtype=np.int64), self.device, torch.int64)
        ids = ops.host_counts("a page table", np.asarray(ids), self.device, torch.int32)
        self.table.view(-1).index_copy_(0, at, ids)

    def _give_back(self, lens, rows):
        """The pages of `rows` behind their first lens tokens (a number a row of them) become free."""
        at = []
        for r, n in zip(rows, -(-lens // self.page_tokens)):
            for j in range(n, self.held[r]):
                self._free.append(int(self._ids[r, j]))
                self._ids[r, j] = -1
                at.append(r * self._ids.shape[1] + j)
            self.held[r] = min(self.held[r], n)
        if at:
            # An entry that pointed on would let an append reach another row's page.
            self._write(at, [-1] * len(at))

    def _added(self, counts, tokens):
        """Tokens that a call may add to each row."""
        if counts is None or torch.is_tensor(counts):
            return np.full(self.rows, tokens, dtype=np.int64)
        counts = np.asarray(counts, dtype=np.int64).reshape(-1)
        if len(counts) != self.batch or (counts < 0).any() or (counts > tokens).any():
            raise ValueError(f"counts must be one integer in 0..{tokens} per sequence")
        return np.repeat(counts, self.per_sequence)

    # -- operators -------------------------------------------------------------
    def append(self, k, v, counts=None, stream=None):
        """New keys and values [B, Hkv, T, 128] at the ends of their rows
        (ops.paged_append), for instance of a prompt that ops.prefill_attn
        attends.  counts: tokens of each sequence (host integers, or an int32
        device tensor; None: all T)."""
        with torch.cuda.stream(stream):  # (None: the current one)
            lens = self._bound() + self._added(counts, k.shape[2])
            self._reserve(lens)
            ops.paged_append(k, v, self.pages, counts=counts)
            self._advance(lens)

    def extend(self, q, k, v, scale, counts=None, weigh=None, out=None, stream=None):
        """Appends new tokens and attends them over their rows: queries [B, Hq,
        T, 128], keys and values [B, Hkv, T, 128], turned by their positions;
        [B, T, Hq, 128] (ops.paged_attn).  weigh (default: whether the store
        tracks): every token's share of the attention is added to its weight."""
        weigh = self.pages.weights is not None if weigh is None else weigh
        with torch.cuda.stream(stream):
            lens = self._bound() + self._added(counts, k.shape[2])
            self._reserve(lens)
            out = ops.paged_attn(q, self.pages, scale, k, v, counts=counts, weigh=weigh, out=out)
            self._advance(lens)
        return out

    def attend(self, q, scale, counts=None, weigh=False, out=None, stream=None):
        """Attention of the last T tokens, which the store holds already."""
        return ops.paged_attn(q, self.pages, scale, counts=counts, weigh=weigh, out=out, stream=stream)

    def evict(self, keep, sink=0, recent=0, stream=None):
        """Holds every row to its `keep` heaviest tokens (an integer, or one a
        row), the positions below `sink` and the last `recent` first
        (ops.paged_evict); pages that no token is left in become free (not by a
        captured call: the next eager one after sync_host_lengths frees them)."""
        host = np.broadcast_to(np.asarray(keep, dtype=np.int64), (self.rows,))
        if (host < sink + recent).any():
            raise ValueError(f"keep={keep} holds less than sink={sink} and recent={recent}")
        with torch.cuda.stream(stream):
            lens = np.minimum(self._bound(), host)
            arg = int(keep) if np.ndim(keep) == 0 else ops.host_counts("keep", host.copy(), self.device)
            ops.paged_evict(self.pages, arg, sink=sink, recent=recent)
            if not torch.cuda.is_current_stream_capturing():
                self._give_back(lens, range(self.rows))
            self._advance(lens)

    def release(self, sequences, stream=None):
        """Ends sequences: their rows are empty, their pages free."""
        rows = [r for b in sequences for r in range(b * self.per_sequence, (b + 1) * self.per_sequence)]
        if any(r < 0 or r >= self.rows for r in rows):
            raise ValueError(f"sequences {list(sequences)} of {self.batch}")
        if not rows:
            return
        with torch.cuda.stream(stream):
            at = ops.host_counts("sequences", np.asarray(rows), self.device, torch.int64)
            self.row_len.index_fill_(0, at, 0)
            if self.pages.dropped is not None:
                self.pages.dropped.index_fill_(0, at, 0)
            self._give_back(np.zeros(len(rows), dtype=np.int64), rows)
        self.host_len[rows], self._along = 0, None

    def sync_host_lengths(self, lens):
        """The lengths that the device holds, where the host has only a bound
        (after replays of captured calls, or counts given on the device)."""
        lens = np.asarray(lens, dtype=np.int64)
        if lens.shape != (self.rows,) or (lens > self.held * self.page_tokens).any() or (lens < 0).any():
            raise RuntimeError("row lengths outside their pages")
        self.host_len, self._along = lens.copy(), None

    def check_status(self, stream=None):
        """Wait for the stream and raise "Layer i OOM." if a row had no room
        for its tokens, HCError if a row reached behind its reserved pages."""
        try:
            ops.read_status(self.status, clear=True, stream=stream)
        except _lib.HCError as e:
            if e.code == _lib.HC_ERR_CAPACITY:
                raise self._oom() from e
            raise
