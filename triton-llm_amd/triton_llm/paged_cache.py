"""Many sequences in one paged KV cache: page tables on the host, pages on the GPU.

:class:`~triton_llm.kv_cache.GpuKVCache` holds one sequence in contiguous
memory, as the reference's models do (smollm2_triton/model.py:190-225).
:class:`PagedKVCache` serves a batch of sequences from pools of pages: a sequence
takes pages as it grows, forks share their prefix, and a page is copied when one of
those that share it writes to it.

A step of the batch::

    cache.begin([1, 1, 0, 7])           # new tokens of each slot: pages are found, shared ones copied
    for layer in range(n_layer):
        out = cache.attention(layer, q, k, v, cos, sin)   # RoPE, cache write, attention
    cache.advance()

and between steps :meth:`~PagedKVCache.open`, :meth:`~PagedKVCache.fork`,
:meth:`~PagedKVCache.close`, :meth:`~PagedKVCache.reorder` (a beam search's parents) and
:meth:`~PagedKVCache.compact`.  Tables and lengths reach the GPU by value with their
launches: nothing here synchronises.  :class:`PageTables` is the host's part alone.
"""

from __future__ import annotations

import ctypes

import numpy as np

from triton_llm import gpu
from triton_llm.kernels.paged import (allocate_kv_pages, check_page_size, check_window, copy_kv_pages,
                                      paged_attention_decode, paged_attention_prefill, paged_decode_workspace,
                                      paged_kv_append, write_i32)

__all__ = ["PageTables", "PagedKVCache"]


def _differing(a: list[int], b: list[int]) -> list[int]:
    """Where two lists of pages differ, places that one has alone among them.  What they share is compared 32 pages at a time:
    beams have most of theirs in common."""
    out, n = [], min(len(a), len(b))
    for lo in range(0, n, 32):
        hi = min(lo + 32, n)
        x, y = a[lo:hi], b[lo:hi]
        if x != y:
            out.extend(lo + i for i, (p, q) in enumerate(zip(x, y)) if p != q)
    out.extend(range(n, max(len(a), len(b))))
    return out


class PageTables:
    """Which pages every slot's sequence has, and which are free.  Host only.

    ``tables[slot]`` lists a slot's pages in order (-1: given back behind the window),
    ``lens[slot]`` its cached tokens.  Changes that the GPU has to follow are collected in
    ``table_edits`` ``{(slot, column): page}`` and ``copies`` ``[(source, destination)]``
    until :meth:`take_edits`.
    """

    def __init__(self, n_pages: int, page_size: int, max_batch: int, max_seq: int, window: int = 0, sinks: int = 0):
        if n_pages <= 0 or max_batch <= 0 or max_seq <= 0:
            raise ValueError(f"n_pages, max_batch and max_seq must be positive, got {n_pages}, {max_batch}, {max_seq}")
        if page_size <= 0:
            raise ValueError(f"page_size must be positive, got {page_size}")
        if window < 0 or sinks < 0:
            raise ValueError(f"window and sinks must be >= 0, got {window} and {sinks}")
        self.n_pages, self.page_size = n_pages, page_size
        self.max_batch, self.max_seq = max_batch, max_seq
        self.window, self.sinks = window, sinks
        self.max_pages = -(-max_seq // page_size)
        self.tables: list[list[int] | None] = [None] * max_batch  # None: the slot is closed
        self.lens = [0] * max_batch
        self.new = [0] * max_batch
        self.refs = [0] * n_pages
        self._gone = [0] * max_batch  # columns before it are given back, the sinks' aside
        self._free = list(range(n_pages - 1, -1, -1))
        self.table_edits: dict[tuple[int, int], int] = {}
        self.copies: list[tuple[int, int]] = []

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _check_slot(self, slot: int) -> None:
        if not 0 <= slot < self.max_batch or self.tables[slot] is None:
            raise ValueError(f"slot {slot} is not open")

    def _check_idle(self) -> None:
        if any(self.new):
            raise ValueError("a step has begun: advance() ends it")

    def _take(self) -> int:
        page = self._free.pop()
        self.refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        if page >= 0:
            self.refs[page] -= 1
            if self.refs[page] == 0:
                self._free.append(page)

    def _set(self, slot: int, pages: list[int] | None) -> None:
        """The slot's pages become `pages`, whose references are the caller's."""
        old, new = self.tables[slot] or [], pages or []
        for c in _differing(old, new):
            self.table_edits[slot, c] = new[c] if c < len(new) else -1
        self.tables[slot] = pages

    def open(self) -> int:
        """An empty sequence in the lowest closed slot."""
        self._check_idle()
        for slot, t in enumerate(self.tables):
            if t is None:
                self.tables[slot] = []
                self.lens[slot] = self._gone[slot] = 0
                return slot
        raise ValueError(f"all {self.max_batch} slots are open")

    def close(self, slot: int) -> None:
        """Give a slot and its pages back."""
        self._check_idle()
        self._check_slot(slot)
        for page in self.tables[slot]:
            self._drop(page)
        self._set(slot, None)
        self.lens[slot] = 0

    def fork(self, slot: int) -> int:
        """A second sequence with the same tokens, in the lowest closed slot.  The pages are shared."""
        self._check_idle()
        self._check_slot(slot)
        other = self.open()
        self.reorder([other], [slot])
        return other

    def reorder(self, slots, parents) -> None:
        """Slot ``slots[i]`` takes over the sequence that ``parents[i]`` has now (all at once: a beam
        search's step).  The slots' own sequences are given up."""
        self._check_idle()
        slots, parents = [int(s) for s in slots], [int(p) for p in parents]
        if len(slots) != len(parents):
            raise ValueError(f"{len(slots)} slots, {len(parents)} parents")
        if len(set(slots)) != len(slots):
            raise ValueError("a slot is given twice")
        for s in slots + parents:
            self._check_slot(s)
        parents, slots = [p for s, p in zip(slots, parents) if s != p], [s for s, p in zip(slots, parents) if s != p]
        # pages that a slot and its parent have in the same place keep their references
        taken = []
        for s, p in zip(slots, parents):
            old, pages = self.tables[s], list(self.tables[p])
            places = _differing(old, pages)
            for c in places:
                if c < len(pages) and pages[c] >= 0:
                    self.refs[pages[c]] += 1
            taken.append((pages, places, self.lens[p], self._gone[p]))
        for s, (pages, places, n, gone) in zip(slots, taken):
            old = self.tables[s]
            for c in places:
                if c < len(old):
                    self._drop(old[c])
                self.table_edits[s, c] = pages[c] if c < len(pages) else -1
            self.tables[s] = pages
            self.lens[s], self._gone[s] = n, gone

    def begin(self, new) -> None:
        """Find room for ``new[slot]`` more tokens of every slot (0 for those that rest): new pages, and a copy of a
        shared last page that is not full.  Raises ValueError, with nothing changed, where a sequence would exceed
        max_seq or the pool has too few pages."""
        self._check_idle()
        new = [int(n) for n in new]
        if len(new) != self.max_batch:
            raise ValueError(f"new must have an entry for each of the {self.max_batch} slots, got {len(new)}")
        if not any(new):
            raise ValueError("a step needs at least one new token")
        ps = self.page_size
        need = 0
        left = {}  # references of pages once the slots before have taken their copies
        copied = set()
        for slot, n in enumerate(new):
            if n < 0:
                raise ValueError(f"new tokens must be >= 0, got {n}")
            if n == 0:
                continue
            self._check_slot(slot)
            at = self.lens[slot]
            if at + n > self.max_seq:
                raise ValueError(f"Total sequence length {at + n} exceeds max_seq ({self.max_seq})")
            need += -(-(at + n) // ps) - len(self.tables[slot])
            if at % ps:
                last = self.tables[slot][at // ps]
                refs = left.get(last, self.refs[last])
                if refs > 1:
                    left[last] = refs - 1
                    need += 1
                    copied.add(slot)
        if need > len(self._free):
            raise ValueError(f"{need} pages needed, {len(self._free)} free")
        for slot, n in enumerate(new):
            if n == 0:
                continue
            pages = self.tables[slot]
            at = self.lens[slot]
            if slot in copied:
                page = self._take()
                self.copies.append((pages[at // ps], page))
                self._drop(pages[at // ps])
                pages[at // ps] = self.table_edits[slot, at // ps] = page
            while len(pages) * ps < at + n:
                page = self._take()
                self.table_edits[slot, len(pages)] = page
                pages.append(page)
        self.new = new

    def advance(self) -> None:
        """End the step: its tokens are cached.  Pages that no later query sees (all of their positions behind
        the window and not among the sinks) are given back."""
        if not any(self.new):
            raise ValueError("no step has begun")
        for slot, n in enumerate(self.new):
            if n == 0:
                continue
            self.lens[slot] += n
            if self.window:
                first = (self.lens[slot] - self.window + 1) // self.page_size  # pages before it are out of sight
                pages = self.tables[slot]
                for c in range(max(self._gone[slot], -(-self.sinks // self.page_size)), min(first, len(pages))):
                    self._drop(pages[c])
                    pages[c] = self.table_edits[slot, c] = -1
                    self._gone[slot] = c + 1
        self.new = [0] * self.max_batch

    def compact(self) -> int:
        """Move the used pages to the pool's lowest numbers; returns how many moved."""
        self._check_idle()
        used = sorted(p for p in range(self.n_pages) if self.refs[p])
        low = [p for p in range(len(used)) if not self.refs[p]]
        moved = dict(zip([p for p in used if p >= len(used)], low))
        for a, b in moved.items():
            self.copies.append((a, b))
            self.refs[b], self.refs[a] = self.refs[a], 0
        for slot, pages in enumerate(self.tables):
            if pages is not None:
                self._set(slot, [moved.get(p, p) for p in pages])
        self._free = list(range(self.n_pages - 1, len(used) - 1, -1))
        return len(moved)

    def take_edits(self):
        """(copies, table edits) since the last call."""
        out = self.copies, self.table_edits
        self.copies, self.table_edits = [], {}
        return out


class PagedKVCache:
    """Per-layer page pools on the GPU, the slots' page tables, and the attention sub-block of a batch's step.

    ``layers[i]`` is ``{"k": DeviceTensor, "v": DeviceTensor}``, each
    ``(n_pages, n_kv_head, page_size, d_k)``.  With ``window`` > 0 a token sees the last ``window``
    positions up to its own and the first ``sinks``.
    """

    def __init__(self, n_layer: int, n_head: int, n_kv_head: int, d_k: int, *, n_pages: int, max_batch: int,
                 max_seq: int, page_size: int = 16, window: int = 0, sinks: int = 0, dtype=np.float32):
        if n_layer <= 0 or n_kv_head <= 0 or n_head <= 0 or n_head % n_kv_head:
            raise ValueError(f"bad head counts: n_layer={n_layer} n_head={n_head} n_kv_head={n_kv_head}")
        if d_k not in (64, 128):
            raise ValueError(f"paged attention supports d_k in (64, 128), got {d_k}")
        # what a step's append and attention would refuse
        check_page_size(page_size)
        check_window(window, sinks)
        if max_batch > 65535:
            raise ValueError(f"max_batch must be at most 65535, got {max_batch}")
        self.tables = PageTables(n_pages, page_size, max_batch, max_seq, window, sinks)
        if self.tables.max_pages * page_size > 1 << 30:
            raise ValueError(f"max_seq must be at most 2^30, got {max_seq}")
        blocks = self.tables.max_pages * page_size // 16
        if window:
            blocks = min(blocks, window // 16 + 2 + -(-sinks // 16))
        pairs = n_kv_head * -(-n_head // n_kv_head // 8)
        if max_batch * pairs * blocks >= 1 << 31:
            raise ValueError(f"{max_batch} sequences of {max_seq} tokens and {n_kv_head} KV heads are more than one-token "
                             f"attention counts (2^31 - 1 blocks of 16 positions a KV head and 8 of its query heads)")
        self.n_layer, self.n_head, self.n_kv_head, self.d_k = n_layer, n_head, n_kv_head, d_k
        self.window, self.sinks = window, sinks
        self.dtype = dtype
        self.layers = []
        for _ in range(n_layer):
            k, v = allocate_kv_pages(n_pages, n_kv_head, page_size, d_k, dtype=dtype)
            self.layers.append({"k": k, "v": v})
        self._pools = [layer[n] for layer in self.layers for n in "kv"]
        shape = (max_batch, self.tables.max_pages)
        self._table = gpu.to_device(np.full(shape, -1, np.int32))
        # row 0: tokens before the step, row 1: the step's, row 2: tokens with the step's (0 for a slot that rests)
        self._counts = gpu.zeros((3, max_batch), np.int32)
        self._host_new = (ctypes.c_int32 * max_batch)()
        self._most_new = self._longest = 0  # the step's tokens of a slot at most, the longest sequence with them
        self._told = [0] * (3 * max_batch)  # what the device has in it
        self._lens, self._new, self._ends = (self._row(i) for i in range(3))
        self._decode_ws = paged_decode_workspace(max_batch, n_head, n_kv_head, max_seq, d_k)

    def _row(self, i: int):
        n = self.tables.max_batch
        return gpu.DeviceTensor(ctypes.c_void_p(self._counts.data_ptr() + 4 * n * i), (n,), np.int32, 4 * n,
                                defer_free=False)

    @property
    def lens(self) -> list[int]:
        """Cached tokens of every slot."""
        return list(self.tables.lens)

    @property
    def free_pages(self) -> int:
        return self.tables.free_pages

    def _publish(self) -> None:
        """Bring the GPU up to date: page copies, table entries, counts."""
        t = self.tables
        copies, edits = t.take_edits()
        # in the order they were made, as many together as do not depend on one another
        start, sources, targets = 0, set(), set()
        for i, (a, b) in enumerate(copies):
            if a in targets or b in targets or b in sources:
                self._copy(copies[start:i])
                start, sources, targets = i, set(), set()
            sources.add(a)
            targets.add(b)
        self._copy(copies[start:])
        if edits:
            write_i32(self._table, [s * t.max_pages + c for s, c in edits], list(edits.values()))
        now = t.lens + t.new + [a + b if b else 0 for a, b in zip(t.lens, t.new)]
        changed = [i for i, n in enumerate(now) if n != self._told[i]]
        write_i32(self._counts, changed, [now[i] for i in changed])
        self._told = now

    def _copy(self, pairs) -> None:
        if pairs:
            copy_kv_pages(self._pools, [a for a, _ in pairs], [b for _, b in pairs])

    def open(self) -> int:
        """An empty sequence; returns its slot."""
        return self.tables.open()

    def close(self, slot: int) -> None:
        """Give a sequence and its pages back."""
        self.tables.close(slot)

    def fork(self, slot: int) -> int:
        """A second sequence with the same tokens; returns its slot.  Pages are shared until written to."""
        return self.tables.fork(slot)

    def reorder(self, slots, parents) -> None:
        """Slot ``slots[i]`` takes over the sequence of slot ``parents[i]``, all at once."""
        self.tables.reorder(slots, parents)

    def compact(self) -> int:
        """Move the used pages to the pools' lowest numbers; returns how many moved."""
        n = self.tables.compact()
        self._publish()
        return n

    def begin(self, new) -> None:
        """Start a step with ``new[slot]`` tokens of every slot (0: the slot rests)."""
        t = self.tables
        t.begin(new)
        self._most_new = max(t.new)
        self._host_new[:] = t.new  # in place: a recorded call finds the step's counts there
        self._longest = max(a + b for a, b in zip(t.lens, t.new) if b)
        self._publish()

    def advance(self) -> None:
        """End the step: its tokens are cached."""
        self.tables.advance()
        self._most_new = 0

    def attention(self, layer: int, q_dev, k_dev, v_dev, cos_dev=None, sin_dev=None, sm_scale: float | None = None,
                  interleaved: bool = False, out=None):
        """One layer's attention for the step: q ``(max_batch, n_new, n_head, d_k)``, k / v ``(max_batch, n_new,
        n_kv_head, d_k)`` in the cache's dtype, n_new at least the step's largest count; a slot's tokens are the first
        of its rows.  q is rotated in place.  cos/sin as in ``paged_kv_append``, of at least as many rows as the
        longest sequence has tokens.  Returns the attention output, like q; the rows that are no tokens
        hold nothing of meaning.  A slot that rests costs nothing: its pages are not read.
        """
        t = self.tables
        if not 0 <= layer < self.n_layer:
            raise ValueError(f"layer {layer} out of range [0, {self.n_layer})")
        if not self._most_new:
            raise ValueError("begin() starts a step")
        for name, x, heads in (("q", q_dev, self.n_head), ("k", k_dev, self.n_kv_head), ("v", v_dev, self.n_kv_head)):
            if len(x.shape) != 4 or x.shape[0] != t.max_batch or x.shape[2:] != (heads, self.d_k):
                raise ValueError(f"{name} must be ({t.max_batch}, n_new, {heads}, {self.d_k}), got {x.shape}")
        n_new = q_dev.shape[1]
        if n_new < self._most_new:
            raise ValueError(f"q has {n_new} rows a slot, the step {self._most_new} tokens")
        if cos_dev is not None and self._longest > cos_dev.shape[0]:
            raise ValueError(f"{self._longest} positions exceed the cos/sin table size ({cos_dev.shape[0]})")
        pool = self.layers[layer]
        paged_kv_append(q_dev, k_dev, v_dev, pool["k"], pool["v"], self._table, self._lens, cos_dev, sin_dev,
                        new_lens=self._new, interleaved=interleaved)
        if n_new == 1:
            return paged_attention_decode(q_dev, pool["k"], pool["v"], self._table, self._ends, self.n_head,
                                          self.n_kv_head, sm_scale=sm_scale, window=self.window, sinks=self.sinks,
                                          out=out, workspace=self._decode_ws)
        return paged_attention_prefill(q_dev, pool["k"], pool["v"], self._table, self._lens, self.n_head,
                                       self.n_kv_head, new_lens=self._new, sm_scale=sm_scale, window=self.window,
                                       sinks=self.sinks, out=out, host_new_lens=self._host_new)
