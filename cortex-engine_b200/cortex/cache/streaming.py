"""Paged cache of per-window rows in HBM (cortex/cache/streaming.py:79-236).

Same API and policy as the reference ``StreamingKVCache``: a pool of
``num_pages`` pages of ``page_size`` rows of ``hidden_dim`` elements, a page
table keyed by ``(session_id, bin_start)``, least-recently-used eviction across
sessions, ``read`` / ``write`` / ``evict_session`` / ``hit_rate`` /
``pages_used``. The pool is one CUDA tensor; the table and the LRU order are
host metadata.

Two additions wire it to the forward (``CortexModel.forward_streaming``):

* an entry may span several pages (``write_rows``): the kv_proj rows of a
  whole window, ``ceil(rows / page_size)`` pages, evicted together;
* ``segments`` gives the (src_row, dst_row, rows) copy list between the pool
  and a packed row buffer that ``ck_copy_rows`` executes on the device, so
  cached rows move HBM to HBM with no host round trip.

What is cached must be a function of the key alone. kv_proj rows of a window
are (they depend only on the window's own events), so the key is the window
identity (session, first bin). Rows of the same spike in an overlapping window
are NOT the same: time bins are window-relative (a max_time_bins vocabulary),
so a shifted window shifts every time embedding.

An entry that grew or shrank (``append_rows``, ``evict_rows``) is no such
function: its rows are nowhere else. It makes room for nothing and stays until
``evict_session`` frees it or its key is written again.
"""

from __future__ import annotations

import time
from collections import OrderedDict
from collections.abc import Sequence
from dataclasses import dataclass, field

import torch

from cortex import _lib as L


@dataclass
class PageMeta:
    """One cache entry (cortex/cache/streaming.py:67-75); ``pages`` lists its
    pages in row order (one page for entries made by ``write``)."""

    page_id: int
    session_id: str
    bin_start: int
    n_events: int
    last_used_at: float
    pages: list[int] = field(default_factory=list)
    edited: bool = False  # rows appended or evicted since the entry was written


def _check_not_capturing(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: the cache's host state cannot be captured into a CUDA graph")


class StreamingKVCache:
    """Paged row cache in device memory.

    Args (cortex/cache/streaming.py:92-99): num_pages, page_size (rows per
    page), hidden_dim (elements per row), dtype, device (a CUDA device).
    """

    def __init__(self, num_pages: int = 128, page_size: int = 64, hidden_dim: int = 512,
                 dtype: torch.dtype = torch.float32, device: str | torch.device = "cuda") -> None:
        if num_pages <= 0 or page_size <= 0 or hidden_dim <= 0:
            raise ValueError("num_pages, page_size and hidden_dim must be positive")
        self.num_pages = num_pages
        self.page_size = page_size
        self.hidden_dim = hidden_dim
        self.device = torch.device(device)
        self._pool = torch.zeros(num_pages, page_size, hidden_dim, dtype=dtype,
                                 device=self.device)
        L.require_cuda(self._pool, what="StreamingKVCache")
        self.device = self._pool.device  # with its index (cuda -> cuda:N)
        self._table: dict[tuple[str, int], int] = {}      # key -> entry id (its first page)
        self._meta: dict[int, PageMeta] = {}              # entry id -> metadata
        self._free: list[int] = list(range(num_pages))
        # entry ids: those that may make room, most recent last, and the edited ones
        self._lru: OrderedDict[int, None] = OrderedDict()
        self._held: set[int] = set()
        self._hits = 0
        self._misses = 0

    # ── reference API ────────────────────────────────────────────────────────

    def read(self, session_id: str, bin_start: int) -> torch.Tensor | None:
        """The cached rows of (session_id, bin_start), or None (a miss).
        A one-page entry returns a view of its page, as the reference does."""
        meta = self.lookup(session_id, bin_start)
        if meta is None:
            return None
        if len(meta.pages) == 1:
            return self._pool[meta.pages[0], :meta.n_events, :]
        return self._pool[meta.pages].reshape(-1, self.hidden_dim)[:meta.n_events]

    def write(self, session_id: str, bin_start: int, embeddings: torch.Tensor) -> None:
        """Cache the first ``page_size`` rows of ``embeddings`` in one page,
        reusing the key's page if present (cortex/cache/streaming.py:150-184).
        Raises ``RuntimeError`` when edited entries hold every page."""
        n = min(int(embeddings.shape[0]), self.page_size)
        if self._pages_but(self._held - {self._table.get((session_id, bin_start))}) < 1:
            raise RuntimeError("write: edited entries hold every page")
        meta = self._entry_for(session_id, bin_start, n_pages=1)
        self._pool[meta.pages[0], :n, :] = embeddings[:n].detach().to(
            dtype=self._pool.dtype, device=self.device)
        meta.n_events = n
        meta.last_used_at = time.monotonic()

    def evict_session(self, session_id: str) -> int:
        """Free every entry of ``session_id``; returns how many (:186-195)."""
        keys = [k for k in self._table if k[0] == session_id]
        for key in keys:
            self._free_entry(self._table[key])
        return len(keys)

    @property
    def hit_rate(self) -> float:
        total = self._hits + self._misses
        return self._hits / total if total > 0 else 0.0

    @property
    def pages_used(self) -> int:
        return self.num_pages - len(self._free)

    # ── multi-page entries and device copies ─────────────────────────────────

    def lookup(self, session_id: str, bin_start: int) -> PageMeta | None:
        """Entry of the key (counted as a hit, and made most recent) or None
        (counted as a miss)."""
        eid = self._table.get((session_id, bin_start))
        if eid is None:
            self._misses += 1
            return None
        self._touch(eid)
        meta = self._meta[eid]
        meta.last_used_at = time.monotonic()
        self._hits += 1
        return meta

    def write_rows(self, session_id: str, bin_start: int, n_rows: int) -> PageMeta | None:
        """Reserve pages for ``n_rows`` rows of the key (replacing an older
        entry); None when they cannot fit beside the edited entries. The caller
        copies the rows in (``segments(meta, ..., into_pool=True)`` + ``ck_copy_rows``)."""
        n_pages = max(1, -(-n_rows // self.page_size))
        if n_pages > self._pages_but(self._held - {self._table.get((session_id, bin_start))}):
            return None
        meta = self._entry_for(session_id, bin_start, n_pages)
        meta.n_events = n_rows
        return meta

    def segments(self, meta: PageMeta, row0: int, into_pool: bool) -> list[tuple[int, int, int]]:
        """(src_row, dst_row, rows) between the entry's pages (pool rows) and
        rows row0.. of a packed buffer; pool -> buffer unless ``into_pool``."""
        out = []
        for k, page in enumerate(meta.pages):
            n = min(self.page_size, meta.n_events - k * self.page_size)
            if n <= 0:
                break
            p, b = page * self.page_size, row0 + k * self.page_size
            out.append((b, p, n) if into_pool else (p, b, n))
        return out

    # ── entries that grow and shrink ─────────────────────────────────────────
    #
    # The pages and lengths of entries are host metadata, copied to the device by
    # each call: a captured call would change them once and copy the same ones in
    # every replay, so these methods refuse to be captured.

    @property
    def pool(self) -> torch.Tensor:
        """(num_pages, page_size, hidden_dim), the pages themselves."""
        return self._pool

    def page_table(self, metas: Sequence[PageMeta]) -> tuple[torch.Tensor, torch.Tensor]:
        """(page_table (B, pages) int32, lengths (B,) int32) of entries on the
        device, as ``paged_attention`` takes them. The copy is queued on the
        current stream. Entries may be listed more than once."""
        _check_not_capturing("page_table")
        self._check_live(metas, distinct=False)
        width = max((len(m.pages) for m in metas), default=0)
        host = torch.zeros(len(metas), width + 1, dtype=torch.int32)
        for b, m in enumerate(metas):
            host[b, 0] = m.n_events
            host[b, 1:1 + len(m.pages)] = torch.tensor(m.pages, dtype=torch.int32)
            self._touch(m.page_id)
        dev = host.pin_memory().to(self.device, non_blocking=True)
        return dev[:, 1:], dev[:, 0].contiguous()

    def append_rows(self, metas: Sequence[PageMeta], rows: torch.Tensor) -> None:
        """Add ``rows[b]`` ((B, n, hidden_dim), the pool's dtype) behind the rows
        of every entry (all different), in pages taken from the pool; least
        recently used entries that are neither listed nor edited make room. Raises
        ``RuntimeError``, changing nothing, when the pool cannot hold them."""
        _check_not_capturing("append_rows")
        self._check_live(metas, distinct=True)
        dev = L.require_cuda(rows, what="append_rows")
        if rows.dim() != 3 or rows.shape[0] != len(metas) or rows.shape[2] != self.hidden_dim:
            raise ValueError(f"append_rows: rows must be ({len(metas)}, n, {self.hidden_dim}), "
                             f"got {tuple(rows.shape)}")
        if rows.dtype != self._pool.dtype or dev != self.device:
            raise ValueError(f"append_rows: rows must be {self._pool.dtype} on {self.device}")
        n = rows.shape[1]
        if not metas or n == 0:
            return
        row_bytes = self.hidden_dim * rows.element_size()
        if row_bytes % 16 != 0:
            raise NotImplementedError("append_rows: rows must be a multiple of 16 bytes")
        need = [max(0, -(-(m.n_events + n) // self.page_size) - len(m.pages)) for m in metas]
        spare = self._pages_but(self._held | {m.page_id for m in metas})
        if sum(need) > spare:
            raise RuntimeError(f"append_rows: {sum(need)} pages needed, {spare} can be had")
        # what may fail comes before the entries change
        src = rows.contiguous()
        lo, hi = L.memory_range(src)
        pool_lo, pool_hi = L.memory_range(self._pool)
        if lo % 16 != 0 or (lo < pool_hi and pool_lo < hi):
            src = src.clone()  # (a pool page that is read below may be written as well)
        n_segs = sum(-(-(m.n_events + n) // self.page_size) - m.n_events // self.page_size
                     for m in metas)
        host = torch.empty(n_segs, 3, dtype=torch.int32, pin_memory=True)
        seg = torch.empty(n_segs, 3, dtype=torch.int32, device=self.device)
        for m in metas:  # none of them makes room below
            self._hold(m)
        segs = []
        for b, (m, k) in enumerate(zip(metas, need)):
            m.pages.extend(self._allocate(k))
            at, end = m.n_events, m.n_events + n
            while at < end:
                page, off = divmod(at, self.page_size)
                take = min(self.page_size - off, end - at)
                segs.append((b * n + at - m.n_events, m.pages[page] * self.page_size + off, take))
                at += take
            m.n_events = end
            m.last_used_at = time.monotonic()
        host.copy_(torch.tensor(segs, dtype=torch.int32))
        with torch.cuda.device(self.device):
            seg.copy_(host, non_blocking=True)
            rc = L.load().ck_copy_rows(src.data_ptr(), len(metas) * n, self.rows.data_ptr(),
                                       self.num_pages * self.page_size, row_bytes, seg.data_ptr(),
                                       n_segs, L.stream_of(self.device))
        L.check(rc, "ck_copy_rows")

    def evict_rows(self, metas: Sequence[PageMeta], weights: torch.Tensor,
                   positions: torch.Tensor, *, budget: int, recent: int = 0) -> None:
        """``evict_by_weight`` on the rows of entries (all different): each keeps
        ``budget`` rows at most, ``weights`` and ``positions`` ((B, slots) float32
        and int32, slots >= the longest entry's pages * page_size) change in place,
        and the pages behind the budget go back to the pool."""
        from cortex.kernels.kv_evict import evict_by_weight

        _check_not_capturing("evict_rows")
        self._check_live(metas, distinct=True)
        if not metas:
            return
        table, lengths = self.page_table(metas)
        evict_by_weight(self._pool, table, lengths, weights, positions, budget=budget,
                        recent=recent, out=(lengths, weights, positions))
        for m in metas:
            if m.n_events > budget:
                keep = max(1, -(-budget // self.page_size))
                self._free.extend(m.pages[keep:])
                del m.pages[keep:]
                m.n_events = budget
                self._hold(m)
            m.last_used_at = time.monotonic()

    def _check_live(self, metas: Sequence[PageMeta], distinct: bool) -> None:
        for m in metas:
            if not self.is_live(m):
                raise ValueError(f"entry ({m.session_id!r}, {m.bin_start}) is no longer in the cache")
        if distinct and len({m.page_id for m in metas}) != len(metas):
            raise ValueError("an entry is listed more than once")

    def is_live(self, meta: PageMeta) -> bool:
        """Whether ``meta`` is still the entry that owns its pages."""
        return self._meta.get(meta.page_id) is meta

    @property
    def rows(self) -> torch.Tensor:
        """The pool as (num_pages * page_size, hidden_dim) rows."""
        return self._pool.view(self.num_pages * self.page_size, self.hidden_dim)

    # ── internals ────────────────────────────────────────────────────────────

    def _touch(self, eid: int) -> None:
        if eid in self._lru:
            self._lru.move_to_end(eid)

    def _hold(self, meta: PageMeta) -> None:
        """The entry's rows are no longer its window's: they cannot be computed again."""
        meta.edited = True
        self._lru.pop(meta.page_id, None)
        self._held.add(meta.page_id)

    def _pages_but(self, entries: set[int]) -> int:
        """Pages that do not belong to these entries: free, or to be had by eviction
        if all edited entries are among them."""
        return self.num_pages - sum(len(self._meta[e].pages) for e in entries)

    def _entry_for(self, session_id: str, bin_start: int, n_pages: int) -> PageMeta:
        key = (session_id, bin_start)
        eid = self._table.get(key)
        # (an edited entry's rows are its holder's: what replaces them is a new entry,
        # and the old PageMeta is no longer live)
        if eid is not None and (len(self._meta[eid].pages) != n_pages or self._meta[eid].edited):
            self._free_entry(eid)
            eid = None
        if eid is None:
            pages = self._allocate(n_pages)
            eid = pages[0]
            self._table[key] = eid
            self._meta[eid] = PageMeta(eid, session_id, bin_start, 0, time.monotonic(), pages)
            self._lru[eid] = None
        self._lru.move_to_end(eid)
        return self._meta[eid]

    def _allocate(self, n_pages: int) -> list[int]:
        """``n_pages`` free pages, evicting least-recently-used entries first."""
        while len(self._free) < n_pages:
            lru, _ = self._lru.popitem(last=False)
            self._free_entry(lru)
        return [self._free.pop() for _ in range(n_pages)]

    def _free_entry(self, eid: int) -> None:
        meta = self._meta.pop(eid, None)
        if meta is not None:
            self._table.pop((meta.session_id, meta.bin_start), None)
            self._free.extend(meta.pages)
        self._lru.pop(eid, None)
        self._held.discard(eid)


__all__ = ["PageMeta", "StreamingKVCache"]
