"""A KV cache in pages for many sessions that fork, rewind and end: histories are shared page by page instead of copied.

:class:`PagedKVCache` owns the pages of every layer, the device page table (:class:`~reelcache_b200.ops.paged.PageTable`)
and the sessions' bookkeeping. Lengths are known to the host (they do not depend on data), so calls that the pool cannot
serve raise :class:`~reelcache_b200.errors.CapacityError` before anything is launched, and no call reads the device.

A step over a batch of sessions::

    batch = cache.extend([(a, 4680), (b, 4680)])      # room for the new tokens
    q = cache.append(layer, batch, q, k, v, positions, rope)
    o = cache.attend(layer, batch, q)

A session is rewound by forking it at the earlier length and closing it. A batch is good as long as its sessions are open
and their pages where they were; it can be written as long as no fork has taken its new tokens. :meth:`PagedKVCache.again`
gives a new one.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Sequence

import torch

from .errors import CapacityError, ConfigurationError, StateError, UnsupportedError
from .ops import paged
from .ops.rope import AxisRope


class _Block:
    """One page that sessions hold, as the host counts it: its holders, and the forks that copied its first rows (when, and
    how many; of several, those that no later one exceeds)."""

    __slots__ = ("holders", "copies")

    def __init__(self):
        self.holders = 1
        self.copies = []

    def copied(self, when: int, rows: int):
        while self.copies and self.copies[-1][1] <= rows:
            self.copies.pop()
        self.copies.append((when, rows))


@dataclass
class PagedSession:
    """A session's slot in the page table and its history's length in tokens."""

    slot: int
    length: int = 0
    open: bool = True
    blocks: list = field(default_factory=list, repr=False)
    cache: "PagedKVCache | None" = field(default=None, repr=False, compare=False)


@dataclass(frozen=True)
class PagedBatch:
    """Sessions with new tokens, as the device operators take them: rows of the block table, lengths with the new tokens,
    where each session's new tokens begin. Made by a cache, whose calls refuse it once it is out of date."""

    sessions: tuple
    counts: tuple
    lengths: tuple
    table: torch.Tensor
    kv_lens: torch.Tensor
    cu_q: torch.Tensor
    cache: "PagedKVCache" = field(repr=False, compare=False)
    made: int = field(repr=False, compare=False)  # the cache's change before it
    checked: list = field(repr=False, compare=False)  # [the change after which it was last found good to write]

    @property
    def tokens(self) -> int:
        return sum(self.counts)


class PagedKVCache:
    """``pages`` pages (below 2^20) of ``page_size`` tokens (a multiple of 8, at most 65536) for ``layers`` layers of
    ``kv_heads`` heads of ``head_dim`` channels; at most ``max_sessions`` open sessions (below 2^20) of at most ``max_tokens``
    tokens.

    ``storage`` is ``[layers, 2, pages, page_size, kv_heads, head_dim]`` (K, V). A page is ``page_size`` consecutive token
    rows of one layer and target, the layout that the restore kernels write, so a restored chunk can go straight into
    a session's pages (:meth:`rows`)."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, *, pages: int, page_size: int, max_sessions: int,
                 max_tokens: int, device="cuda", dtype=torch.bfloat16):
        device = torch.device(device)
        if device.type != "cuda":
            raise UnsupportedError("PagedKVCache needs a CUDA device")
        for name, value in (("layers", layers), ("kv_heads", kv_heads), ("pages", pages), ("max_sessions", max_sessions),
                            ("max_tokens", max_tokens)):
            if type(value) is not int or value < 1:
                raise ConfigurationError(f"PagedKVCache: {name} must be a positive integer, got {value!r}")
        if head_dim not in (64, 128) or dtype not in (torch.bfloat16, torch.float16):
            raise ConfigurationError(f"PagedKVCache: head_dim is 64 or 128 and the type bf16 or fp16, got {head_dim} {dtype}")
        if type(page_size) is not int or not 8 <= page_size <= 65536 or page_size % 8:
            raise ConfigurationError(f"PagedKVCache: page_size must be a multiple of 8 tokens, at most 65536, got {page_size!r}")
        if max(pages, max_sessions) >= 1 << 20:  # what the page table's prefix sums hold
            raise ConfigurationError(f"PagedKVCache: pages and max_sessions must be below 2^20, got {pages} and {max_sessions}")
        self.page_size, self.pages, self.max_tokens = page_size, pages, max_tokens
        self.storage = torch.zeros(layers, 2, pages, page_size, kv_heads, head_dim, dtype=dtype, device=device)
        self.table = paged.PageTable.empty(pages, max_sessions, -(-max_tokens // page_size), page_size, device)
        self.device = self.storage.device
        self._planes = self.storage.flatten(0, 1)
        self._free_slots = list(range(max_sessions))[::-1]
        self._held = 0
        self._changes = self._compacted = 0  # forks, ends and compactions so far; which of them was the last compaction

    # -- sessions --------------------------------------------------------------------------------------------------------

    @property
    def free_pages(self) -> int:
        return self.pages - self._held

    @property
    def nbytes(self) -> int:
        return self.storage.numel() * self.storage.element_size()

    def _ints(self, values) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32).pin_memory().to(self.device, non_blocking=True)

    def _check(self, sessions: Sequence[PagedSession]):
        for s in sessions:
            if s.cache is not self:
                raise StateError(f"the session in slot {s.slot} is another cache's")
            if not s.open:
                raise StateError(f"session in slot {s.slot} is closed")

    def _next_slots(self, count: int) -> list[int]:
        """The slots that the next sessions get, last in the list of free ones first (they stay in it)."""
        if count > len(self._free_slots):
            raise CapacityError(f"{count} session slots wanted, {len(self._free_slots)} free")
        return self._free_slots[::-1][:count]

    def _admit(self, pages: int):
        if pages > self.free_pages:
            raise CapacityError(f"{pages} pages wanted, {self.free_pages} of {self.pages} free")

    def open(self) -> PagedSession:
        """A session without history."""
        (slot,) = self._next_slots(1)
        self._free_slots.pop()
        return PagedSession(slot, cache=self)

    def fork(self, session: PagedSession, lengths: Sequence[int] | None = None, *, count: int | None = None) -> list[PagedSession]:
        """Sessions that begin with the first ``lengths[i]`` tokens of ``session`` (``count`` times all of it): whole pages
        are shared, the rows of a partly filled last page are copied."""
        self._check([session])
        if lengths is None:
            lengths = [session.length] * (1 if count is None else count)
        elif count is not None:
            raise ConfigurationError("fork takes lengths or a count")
        lengths = [int(n) for n in lengths]
        if not all(0 <= n <= session.length for n in lengths):
            raise ConfigurationError(f"fork lengths {lengths} must lie within the session's {session.length} tokens")
        if not lengths:
            return []
        self._admit(sum(n % self.page_size > 0 for n in lengths))
        slots = self._next_slots(len(lengths))
        # (the host's books follow the device: what raises until here has changed neither)
        self.table.fork(self._ints([session.slot] * len(slots)), self._ints(slots), self._ints(lengths), self._planes)
        del self._free_slots[len(self._free_slots) - len(slots):]
        self._changes += 1
        children = []
        for slot, n in zip(slots, lengths):
            child = PagedSession(slot, n, True, session.blocks[:n // self.page_size], self)
            for block in child.blocks:
                block.holders += 1
            if n % self.page_size:
                session.blocks[n // self.page_size].copied(self._changes, n % self.page_size)
                child.blocks.append(_Block())
                self._held += 1
            children.append(child)
        return children

    def close(self, *sessions: PagedSession):
        """Sessions end; pages that no other session holds are free."""
        self._check(sessions)
        if len({s.slot for s in sessions}) < len(sessions):
            raise StateError("a session is named twice")
        if not sessions:
            return
        self.table.release(self._ints(s.slot for s in sessions))
        self._changes += 1
        for s in sessions:
            for block in s.blocks:
                block.holders -= 1
                self._held -= block.holders == 0
            s.blocks, s.open, s.length = [], False, 0
            self._free_slots.append(s.slot)

    def extend(self, pairs: Sequence[tuple[PagedSession, int]]) -> PagedBatch:
        """Room for new tokens: ``[(session, new tokens), ...]``. The new tokens are the last ones of each session from
        here on; :meth:`append` writes them layer by layer."""
        pairs = [(s, int(n)) for s, n in pairs]
        sessions = [s for s, _ in pairs]
        self._check(sessions)
        if len({s.slot for s in sessions}) < len(sessions) or not pairs:
            raise StateError("extend takes each session once, and at least one")
        for s, n in pairs:
            if n < 0 or s.length + n > self.max_tokens:
                raise CapacityError(f"a session of {s.length} tokens cannot take {n} more (at most {self.max_tokens})")
        blocks = [-(-(s.length + n) // self.page_size) - len(s.blocks) for s, n in pairs]
        self._admit(sum(blocks))
        batch, slots = self._batch(sessions, [n for _, n in pairs], [s.length + n for s, n in pairs])
        self.table.allocate(slots, batch.kv_lens)
        for (s, n), b in zip(pairs, blocks):
            s.length += n
            s.blocks.extend(_Block() for _ in range(b))
        self._held += sum(blocks)
        return self._name_pages(batch, slots)

    def again(self, pairs: Sequence[tuple[PagedSession, int]]) -> PagedBatch:
        """The last tokens of sessions once more, as :meth:`extend` gave them (a further denoising step over a chunk)."""
        pairs = [(s, int(n)) for s, n in pairs]
        sessions = [s for s, _ in pairs]
        self._check(sessions)
        if not pairs or len({s.slot for s in sessions}) < len(sessions) or any(not 0 <= n <= s.length for s, n in pairs):
            raise StateError("again takes each session once, with tokens that it has")
        shared = [s.slot for s, n in pairs if any(b.holders > 1 for b in s.blocks[(s.length - n) // self.page_size:]) and n]
        if shared:
            raise StateError(f"the last tokens of the sessions in slots {shared} are shared with others: fork before them")
        return self._name_pages(*self._batch(sessions, [n for _, n in pairs], [s.length for s in sessions]))

    def _batch(self, sessions, counts, lengths) -> tuple[PagedBatch, torch.Tensor]:
        """A batch whose rows of the block table are yet to be filled in, and its slots."""
        width = max(-(-max(lengths) // self.page_size), 1)
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        table = torch.empty(len(sessions), width, dtype=torch.int32, device=self.device)
        return PagedBatch(tuple(sessions), tuple(counts), tuple(lengths), table, self._ints(lengths), self._ints(starts), self,
                          self._changes, [self._changes]), self._ints(s.slot for s in sessions)

    def _name_pages(self, batch: PagedBatch, slots: torch.Tensor) -> PagedBatch:
        torch.index_select(self.table.block_table[:, :batch.table.shape[1]], 0, slots, out=batch.table)
        return batch

    def _check_batch(self, batch: PagedBatch, q, *, write: bool):
        """Refuse fewer rows than the batch has new tokens (lengths would no longer say where they are), a batch whose pages may hold something else by now, or (``write``) whose new tokens a fork has taken:
        writing them would change the child's history, or leave what it copied behind."""
        if batch.cache is not self:
            raise StateError("the batch is another cache's")
        if q is not None and q.shape[0] < batch.tokens:
            raise ConfigurationError(f"the batch has {batch.tokens} new tokens, q has {q.shape[0]} rows")
        if batch.checked[0] == self._changes:
            return
        self._check(batch.sessions)
        if batch.made < self._compacted:
            raise StateError("the batch is from before a compaction, which moved pages: make it again")
        if not write:
            return
        for s, n, length in zip(batch.sessions, batch.counts, batch.lengths):
            first = length - n
            for i in range(first // self.page_size, -(-length // self.page_size) if n else 0):
                block, row = s.blocks[i], max(first - i * self.page_size, 0)
                if block.holders > 1 or any(when > batch.made and rows > row for when, rows in block.copies):
                    raise StateError(f"the session in slot {s.slot} was forked after the batch, with its new tokens: fork before "
                                     "them, or make the batch again")
        batch.checked[0] = self._changes

    def compact(self) -> int:
        """Move the pages in use to the front of the pool (the rest of the storage is then free in one piece). Returns how
        many there are. Batches made before are refused from here on."""
        self.table.compact(self._planes)
        self._changes += 1
        self._compacted = self._changes
        return self._held

    # -- layers ----------------------------------------------------------------------------------------------------------

    def append(self, layer: int, batch: PagedBatch, q, k, v, positions, rope: AxisRope, *, out=None):
        """Write the new tokens of one layer (``k`` rotated at ``positions``, ``v`` as it is); returns ``q`` rotated."""
        self._check_batch(batch, q, write=True)
        return paged.append(q, k, v, positions, rope, self.storage[layer, 0], self.storage[layer, 1], batch.table,
                            batch.kv_lens, batch.cu_q, out=out)

    def attend(self, layer: int, batch: PagedBatch, q, *, causal: bool = False, window: int | None = None, sinks: int = 0,
               scale: float | None = None, return_lse: bool = False, out=None):
        """Attention of the new tokens over their sessions (:func:`reelcache_b200.ops.paged.attention`)."""
        self._check_batch(batch, q, write=False)
        return paged.attention(q, self.storage[layer, 0], self.storage[layer, 1], batch.table, batch.kv_lens, batch.cu_q,
                               max_q_len=max(max(batch.counts), 1), causal=causal, window=window, sinks=sinks, scale=scale,
                               return_lse=return_lse, out=out)

    def token_rows(self, layer: int, which: str) -> torch.Tensor:
        """All token rows ``[pages * page_size, kv_heads * head_dim]`` of one layer's K or V (``which``), page by page."""
        return self.storage[layer, 0 if which == "K" else 1].flatten(0, 1).flatten(1)

    def new_rows(self, batch: PagedBatch) -> torch.Tensor:
        """Where the batch's new tokens lie in :meth:`token_rows` (int64, one after the other), for a kernel that writes them
        itself instead of :meth:`append`."""
        self._check_batch(batch, None, write=True)
        token = torch.arange(batch.tokens, dtype=torch.int32, device=self.device)
        seq = torch.bucketize(token, batch.cu_q[1:], right=True)
        at = (batch.kv_lens - batch.cu_q[1:])[seq] + token
        return batch.table[seq, at // self.page_size].long() * self.page_size + at % self.page_size

    def rows(self, layer: int, which: str, page: int) -> torch.Tensor:
        """Token rows ``[page_size, kv_heads * head_dim]`` of one page (``which``: ``"K"`` or ``"V"``)."""
        return self.storage[layer, 0 if which == "K" else 1, page].flatten(1)
