"""A paged key-value cache of bounded size: append, attention of the newest tokens over the pages, eviction by attention weight.

Keys and values live in pages [n_pages, Hkv, page, D] (page a power of two from 16 to 1024) that sequences own through a table
[B, max_pages] of page numbers; `lengths` [B] counts their tokens.  Table and lengths are read on the device, so a decoding step can be
captured in a CUDA graph and replayed while the sequences grow.  `PagedKVCache` keeps the pages; the functions below take any tensors
of that layout, pages that several sequences share included (for reading).
"""
import torch

from . import _lib as L


def paged_append(k, v, k_pages, v_pages, table, lengths, counts=None, weights=None):
    """Store rows 0 .. counts[b] - 1 (all T without counts) of k, v [B,Hkv,T,D] behind the tokens of every sequence and move `lengths`
    on, in place.  The pages must be in the table already.  Rows that have none are not stored (their keys count, and stay hidden), rows
    without room in the table do not count; `_lib.device_status()` says 601 or 602.  weights [B, Hkv, max_pages * page] (fp32) are set to 0 for the new keys.
    The numbers of k and v alone are stored: no gradients go through the cache, and tangents are refused."""
    L.host().paged_append(k, v, k_pages, v_pages, table, lengths, counts, weights)


def paged_attention(q, k_pages, v_pages, table, lengths, window=None, sinks=0, sm_scale=None, weights=None, decay=1.0):
    """Attention of the last T tokens of every sequence, q [B,H,T,D], over its cached keys: [B,H,T,D].

    Query t stands at position p = lengths[b] - T + t (its own key is in the cache already) and sees key j if j <= p and, with a window,
    (p - j < window or j < sinks).  H is a multiple of Hkv.  Rows that see nothing (an empty sequence) give zeros.
    weights: fp32 [B, Hkv, max_pages * page], updated in place for every j < lengths[b]:
      weights = decay * weights + sum of the key's attention weights over the T queries of the heads that share it;
    decay=0 overwrites them.  `paged_evict` goes by them.  bf16, fp16 or fp32, D a multiple of 8 up to 128; no gradients.
    T up to 1024, and up to 4096 query rows a key head (H / Hkv * T).  Values that some of the T tokens see are expected to be finite: one
    that is not can reach the other tokens of its sequence and key head.  A row whose scores are all -inf gives zeros, as one that sees nothing.
    Weights take a workspace of 4 bytes per query row and key of the table's capacity (B * H * T * max_pages * page), whatever the lengths."""
    return L.host().paged_attention(q, k_pages, v_pages, table, lengths, window, sinks, sm_scale, weights, decay)


def paged_evict(k_pages, v_pages, table, lengths, weights, fresh, budget, recent=0, sinks=0):
    """Bring every sequence of more than `budget` tokens down to it: the first `sinks`, the last `recent` and, of the rest, the
    budget - sinks - recent keys with the largest weights stay (the lower position first where weights are equal; NaN counts as the
    largest), chosen per key head, in order.  They are copied to the pages fresh [B, n] (n * page >= budget), which must belong to
    nobody; the pages in `table` are not written, and sequences within the budget keep theirs.
    Survivors that have no page become rows of zeros (`_lib.device_status()` says 601).
    Returns (table, lengths, weights, kept), new tensors; kept [B, Hkv, budget] are the survivors' former positions, -1 behind them."""
    return L.host().paged_evict(k_pages, v_pages, table, lengths, weights, fresh, budget, recent, sinks)


class PagedKVCache:
    """Keys and values of a batch of sequences in pages, with the page bookkeeping on the host.

    num_pages bounds the memory, max_tokens one sequence's length.  track_weights keeps a running sum of attention weights per key and key
    head, which `attend` adds to and `evict` goes by.  Calls belong on one stream at a time, like those of any cache that is
    written in place."""

    def __init__(self, batch, kv_heads, dim, dtype, device, max_tokens, page=64, num_pages=None, track_weights=False):
        self.page, self.max_pages = page, -(-max_tokens // page)
        if num_pages is None:
            num_pages = batch * self.max_pages
        self.k_pages = torch.empty((num_pages, kv_heads, page, dim), dtype=dtype, device=device)
        self.v_pages = torch.empty_like(self.k_pages)
        self.table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros((batch,), dtype=torch.int32, device=device)
        self.weights = (torch.zeros((batch, kv_heads, self.max_pages * page), dtype=torch.float32, device=device)
                        if track_weights else None)
        self._tokens = [0] * batch                # the lengths as the host knows them
        self._owned = [[] for _ in range(batch)]
        self._free = list(range(num_pages - 1, -1, -1))

    def refresh(self):
        """Take the lengths from the device, after replays of a captured step."""
        self._tokens = self.lengths.tolist()
        return self._tokens

    def _all_stored(self):
        # Replays that went on behind the reserved pages stored nothing there (status 601); pages given now would show whatever they hold.
        for b, t in enumerate(self._tokens):
            if t > len(self._owned[b]) * self.page:
                raise ValueError(f"sequence {b} has {t} tokens in pages for {len(self._owned[b]) * self.page}: the others were not stored; drop it")

    def reserve(self, tokens):
        """Give every sequence pages for `tokens` more tokens (a number, or one per sequence), e.g. before a step is captured."""
        more = [tokens] * len(self._tokens) if isinstance(tokens, int) else list(tokens)
        if len(more) != len(self._tokens):
            raise ValueError(f"expected one number of tokens for each of {len(self._tokens)} sequences")
        self._all_stored()
        need = [-(-(n + m) // self.page) for n, m in zip(self._tokens, more)]
        if max(need) > self.max_pages:
            raise ValueError(f"a sequence would exceed the cache's {self.max_pages * self.page} tokens")
        where = [(b, i) for b, n in enumerate(need) for i in range(len(self._owned[b]), n)]
        if not where:
            return
        if len(where) > len(self._free):
            raise ValueError(f"{len(where)} pages needed, {len(self._free)} free")
        if self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("reserve() pages before a step is captured")
        ids = [self._free.pop() for _ in where]
        for (b, _), page_id in zip(where, ids):
            self._owned[b].append(page_id)
        at = torch.tensor(where, device=self.table.device)
        self.table[at[:, 0], at[:, 1]] = torch.tensor(ids, dtype=torch.int32, device=self.table.device)

    def append(self, k, v, counts=None):
        """Store k, v [B,Hkv,T,D] behind the cached tokens; counts: how many of the T rows each sequence has (a list), for ragged prompts."""
        if counts is not None and self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("append with counts cannot be captured: paged_append takes them from the device")
        n = [k.shape[2]] * len(self._tokens) if counts is None else [min(max(int(c), 0), k.shape[2]) for c in counts]
        if len(n) != len(self._tokens):
            raise ValueError(f"expected one count for each of {len(self._tokens)} sequences")
        self.reserve(n)
        on_device = None if counts is None else torch.tensor(n, dtype=torch.int32, device=self.table.device)
        paged_append(k, v, self.k_pages, self.v_pages, self.table, self.lengths, on_device, self.weights)
        self._tokens = [a + b for a, b in zip(self._tokens, n)]

    def attend(self, q, window=None, sinks=0, sm_scale=None, decay=1.0):
        """paged_attention of the newest tokens; with track_weights their attention weights are added to the running sums."""
        return paged_attention(q, self.k_pages, self.v_pages, self.table, self.lengths, window, sinks, sm_scale, self.weights, decay)

    def evict(self, budget, recent=0, sinks=0):
        """paged_evict with pages of this cache; returns `kept`.  Reads the lengths back, so the host waits; not for captured steps.

        All sequences go at once where ceil(budget / page) pages for each that is over the budget are free, otherwise as many at a time as
        there is room for; with room for none, one goes through a copy of its pages."""
        if self.weights is None:
            raise ValueError("evict goes by attention weights: make the cache with track_weights=True")
        if self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("evict cannot be captured")
        if budget < 1:
            raise ValueError("the budget must be at least 1 token")
        n = -(-budget // self.page)
        over = [b for b, t in enumerate(self.refresh()) if t > budget]
        self._all_stored()
        if n * len(over) <= len(self._free):
            return self._evict(None, over, n, budget, recent, sinks)
        kept = torch.empty((len(self._tokens), self.k_pages.shape[1], budget), dtype=torch.int32, device=self.table.device)
        rest = [b for b, t in enumerate(self._tokens) if t <= budget]
        if rest:
            kept[rest] = self._evict(rest, [], n, budget, recent, sinks)
        while over:                               # a sequence gives back at least as many pages as it takes
            room = len(self._free) // n
            some, over = over[:max(room, 1)], over[max(room, 1):]
            kept[some] = (self._evict if room else self._evict_through_copy)(some, some, n, budget, recent, sinks)
        return kept

    def _evict(self, rows, over, n, budget, recent, sinks):
        """Evict from the sequences `rows` (None: all), of which `over` are beyond the budget: n free pages for each of these."""
        count = len(self._tokens) if rows is None else len(rows)
        taken = dict(zip(over, (self._free[i * n:(i + 1) * n] for i in range(len(over)))))
        fresh = torch.tensor([taken.get(b, [-1] * n) for b in (range(count) if rows is None else rows)], dtype=torch.int32,
                             device=self.table.device).view(count, n)
        mine = (self.table, self.lengths, self.weights)
        if rows is not None:
            at = torch.tensor(rows, device=self.table.device)
            mine = tuple(t.index_select(0, at) for t in mine)
        *new, kept = paged_evict(self.k_pages, self.v_pages, *mine, fresh, budget, recent, sinks)
        for to, x in zip((self.table, self.lengths, self.weights), new):      # in place: captured steps read these tensors
            to.copy_(x) if rows is None else to.index_copy_(0, at, x)
        del self._free[:n * len(over)]
        for b in over:
            self._free.extend(self._owned[b])
            self._owned[b] = taken[b]
            self._tokens[b] = budget
        return kept

    def _evict_through_copy(self, rows, over, n, budget, recent, sinks):
        """The same for one sequence and no free pages: out of a copy of its pages, back into the first n of them."""
        (b,) = rows
        own = torch.tensor(self._owned[b], device=self.table.device)
        m = own.numel()
        pools = [torch.cat((p.index_select(0, own), p.new_empty((n, *p.shape[1:])))) for p in (self.k_pages, self.v_pages)]
        table = torch.full_like(self.table[:1], -1)
        table[0, :m] = torch.arange(m, device=own.device)
        fresh = torch.arange(m, m + n, dtype=torch.int32, device=own.device).view(1, n)
        _, lengths, weights, kept = paged_evict(*pools, table, self.lengths[b:b + 1], self.weights[b:b + 1], fresh, budget, recent, sinks)
        for p, copy in zip((self.k_pages, self.v_pages), pools):
            p.index_copy_(0, own[:n], copy[m:])
        self.table[b, n:] = -1
        self.lengths[b:b + 1] = lengths
        self.weights[b:b + 1] = weights
        self._free.extend(self._owned[b][n:])
        self._owned[b], self._tokens[b] = self._owned[b][:n], budget
        return kept

    def drop(self, sequence):
        """Forget a sequence and take its pages back."""
        self._free.extend(self._owned[sequence])
        self._owned[sequence], self._tokens[sequence] = [], 0
        self.table[sequence] = -1
        self.lengths[sequence] = 0
