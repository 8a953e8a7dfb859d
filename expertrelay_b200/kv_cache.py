"""PagedKVCache: the keys and values of a whole model for many sequences, on
the operators of expertrelay_b200.kv.

The reference's KVCache (runtime/qwen_moe.py:90-106) is one sequence's
arrays, as long as the longest text allows. Here the sequences share a pool of
pages: PageTable gives each of them pages as it grows and takes them back,
one table serves every layer, and keys and values may be kept in 16 bits. Two
ways to make long texts cheaper, either or neither:

  select=(budget, sinks, recent)  one-token calls read, for each key head, only
                                  the pages that select_pages picks
  mass=True                       attention accumulates each position's weight,
                                  and evict() cuts sequences to a budget by it

All of a cache's work belongs on one stream: pages change hands in its order.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from . import kv


class PageTable:
    """Which pages the sequences have: host side, no device. `table`
    [seqs, width] int32 page ids (-1: none), `length` the places a sequence
    uses in the cache, `position` the tokens it has seen (more, once places
    were evicted)."""

    def __init__(self, seqs: int, width: int, pages: int, page_size: int):
        if min(seqs, width, pages, page_size) < 1:
            raise ValueError(f"{seqs} sequences, tables of {width}, {pages} pages of {page_size}: at least one each")
        self.page_size = page_size
        self.table = np.full((seqs, width), -1, dtype=np.int32)
        self.length = np.zeros(seqs, dtype=np.int64)
        self.position = np.zeros(seqs, dtype=np.int64)
        self.free = list(range(pages - 1, -1, -1))  # the next one to give out is the last

    def _pages(self, n: int) -> int:
        return -(-int(n) // self.page_size)

    def known(self, seqs) -> None:
        """ValueError for a sequence that is none of the table's (a negative one would count from the end)."""
        seqs = np.asarray(seqs)
        if seqs.size and (seqs.min() < 0 or seqs.max() >= len(self.length)):
            raise ValueError(f"sequences outside [0, {len(self.length)})")

    def extend(self, seqs) -> tuple[np.ndarray, np.ndarray]:
        """A place for one more token of each sequence in `seqs` (in order; a
        sequence may occur more than once): (positions, slots). Raises
        ValueError, changing nothing, if a table or the pool is full."""
        seqs = np.asarray(seqs, dtype=np.int64)
        if seqs.ndim != 1:
            raise ValueError(f"sequences: one for each row, got {seqs.shape}")
        self.known(seqs)
        ids, counts = np.unique(seqs, return_counts=True)
        new = []
        for s, c in zip(ids, counts):
            have, want = self._pages(self.length[s]), self._pages(self.length[s] + c)
            if want > self.table.shape[1]:
                raise ValueError(f"sequence length {self.length[s] + c} exceeds the KV cache "
                                 f"({self.table.shape[1] * self.page_size})")
            new += [(s, o) for o in range(have, want)]
        if len(new) > len(self.free):
            raise ValueError(f"the KV cache is out of pages ({len(new)} needed, {len(self.free)} free)")
        for s, o in new:
            self.table[s, o] = self.free.pop()
        nth = np.zeros(len(seqs), dtype=np.int64)  # how often the row's sequence came before it
        for s in ids:
            at = np.flatnonzero(seqs == s)
            nth[at] = np.arange(len(at))
        positions, slots = self.position[seqs] + nth, self.length[seqs] + nth
        self.length[ids] += counts
        self.position[ids] += counts
        return positions, slots

    def shrink(self, seqs) -> None:
        """Takes the last extend(seqs) back: places, positions and pages as before it."""
        ids, counts = np.unique(np.asarray(seqs, dtype=np.int64), return_counts=True)
        for s, c in zip(ids[::-1], counts[::-1]):
            self.length[s] -= c
            self.position[s] -= c
            for o in range(self._pages(self.length[s] + c) - 1, self._pages(self.length[s]) - 1, -1):
                self.free.append(int(self.table[s, o]))
                self.table[s, o] = -1

    def take(self, n: int) -> list[int]:
        """n free pages, out of the pool."""
        if n > len(self.free):
            raise ValueError(f"the KV cache is out of pages ({n} needed, {len(self.free)} free)")
        return [self.free.pop() for _ in range(n)]

    def replace(self, seq: int, pages: list[int], length: int) -> None:
        """The sequence's places are now `length`, in `pages`; its old pages that are none of them are free."""
        kept = set(pages)
        self.free += [int(p) for p in self.table[seq] if p >= 0 and int(p) not in kept]
        self.table[seq] = -1
        self.table[seq, :len(pages)] = pages
        self.length[seq] = length

    def release(self, seq: int) -> None:
        self.known(seq)
        self.replace(seq, [], 0)
        self.position[seq] = 0


@dataclass
class Step:
    """One call's rows on the device: the sequence, position, place and visible length of every row."""

    seqs: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    lens: torch.Tensor
    spans: dict[int, np.ndarray]  # rows of every sequence
    every: bool                   # one row for each sequence, in order
    lengths: torch.Tensor         # of all sequences, after the call
    start: torch.Tensor           # and before it
    number: int                   # which of the cache's steps
    longest: int                  # places of the longest sequence in the step
    mass: dict[int, torch.Tensor] # the sequences' weights before the call, of the layers that have attended


class PagedKVCache:
    """`seqs` sequences of up to max_seq places each in `pages` pages of
    page_size places (default: as many as all of them can need). config: a
    ModelConfig (layers, key heads, head_dim); dtype: float32 or bfloat16.
    Caches that are to be cut (mass=True, evict) have at most about 370000 places
    a sequence."""

    def __init__(self, config, seqs: int, max_seq: int, *, page_size: int = 64, pages: int | None = None,
                 dtype: torch.dtype = torch.float32, device="cuda", mass: bool = False,
                 select: tuple[int, int, int] | None = None):
        if mass and select is not None:
            raise ValueError("mass and select: attention over selected pages does not accumulate weights")
        if select is not None and (min(select) < 0 or select[0] < 1 or select[1] + select[2] > select[0]):
            raise ValueError(f"select: (budget, sinks, recent), got {select}")
        width = -(-max_seq // page_size) if page_size > 0 else 0  # PageTable refuses 0
        self.pages = PageTable(seqs, width, seqs * width if pages is None else pages, page_size)
        self.seqs, self.max_seq, self.page_size, self.device = seqs, width * page_size, page_size, torch.device(device)
        shape = (config.num_layers, len(self.pages.free), config.num_kv_heads, page_size, config.head_dim)
        # never read before they are written: places behind a sequence's length are masked out, and a call
        # that fails before every layer has written its places gives them back (undo)
        self.k = torch.empty(shape, dtype=dtype, device=self.device)
        self.v = torch.empty(shape, dtype=dtype, device=self.device)
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.layers = [kv.PagedKV(self.k[i], self.v[i], self.table, self.status) for i in range(config.num_layers)]
        self.mass = None
        if mass:
            self.mass = torch.zeros((config.num_layers, seqs, config.num_kv_heads, self.max_seq), device=self.device)
        self.select = select
        self.bounds = [kv.PageBounds.new(c) for c in self.layers] if select is not None else None
        self._number = 0  # steps, evictions and releases so far

    @property
    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()

    def length(self, seq: int = 0) -> int:
        """The places sequence `seq` uses."""
        self.pages.known(seq)
        return int(self.pages.length[seq])

    def _ints(self, a) -> torch.Tensor:
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(self.device)

    def step(self, seqs) -> Step:
        """Places for one more token of every sequence in `seqs`, row by row; the tables follow. Every layer
        has to attend with the step; where one cannot, undo(step) takes it back."""
        seqs = np.asarray(seqs, dtype=np.int64)
        before = self.pages.length.copy()
        positions, slots = self.pages.extend(seqs)
        self._number += 1
        try:
            self.table.copy_(torch.from_numpy(self.pages.table))
            rows = self._ints(np.stack([seqs, positions, slots, slots + 1]))
            both = self._ints(np.stack([self.pages.length, before]))
            spans = {int(s): np.flatnonzero(seqs == s) for s in np.unique(seqs)}
            return Step(rows[0], rows[1], rows[2], rows[3], spans,
                        len(seqs) == self.seqs and bool(np.all(seqs == np.arange(self.seqs))), both[0], both[1],
                        self._number, int(slots.max()) + 1 if len(slots) else 0, {})
        except BaseException:
            self._give_back(seqs)
            raise

    def undo(self, step: Step) -> None:
        """Takes a step back of which not every layer has attended (an error between layers): lengths,
        positions, pages and accumulated weights are what they were. Only the cache's last step, before
        any eviction or release after it."""
        if step.number != self._number:
            raise ValueError("undo: not the cache's last step")
        self._give_back([s for s, rows in step.spans.items() for _ in rows])
        for layer, before in step.mass.items():
            for i, s in enumerate(step.spans):
                self.mass[layer, s, :, :step.longest] = before[i]

    def _give_back(self, seqs) -> None:
        self._number += 1
        self.pages.shrink(seqs)
        self.table.copy_(torch.from_numpy(self.pages.table))

    def attend(self, layer: int, step: Step, qkv: torch.Tensor, heads: int, theta: float) -> torch.Tensor:
        """One layer's attention for a step: qkv [n, (heads + 2 kv_heads) head_dim]
        into the pages, then every row over its sequence up to itself; [n, heads, head_dim]."""
        cache = self.layers[layer]
        q = kv.append(cache, qkv, step.positions, heads, theta, seqs=step.seqs, slots=step.slots)
        if self.select is not None:
            kv.page_bounds(cache, self.bounds[layer], step.lengths, step.start)
            if all(len(r) == 1 for r in step.spans.values()):  # new tokens, not a prompt
                budget, sinks, recent = self.select
                pages, counts = kv.select_pages(cache, self.bounds[layer], q, step.lens, budget, sinks=sinks,
                                                recent=recent, seqs=step.seqs)
                return kv.attend(cache, q, step.lens, seqs=step.seqs, pages=pages, counts=counts)
        if self.mass is None:
            return kv.attend(cache, q, step.lens, seqs=step.seqs)
        mass = self.mass[layer]
        # kept for undo: 4 bytes a place and key head, beside the keys and values of a place
        seen = mass[:, :, :step.longest]
        if layer not in step.mass:
            step.mass[layer] = seen.clone() if step.every else torch.stack([seen[s] for s in step.spans])
        if step.every:
            return kv.attend(cache, q, step.lens, mass=mass)
        # rows of their own, some at a time (256 MB), then summed by sequence in row order: the same sum every time
        out, n = torch.empty_like(q), q.shape[0]
        each = min(n, max(1, (64 << 20) // mass[0].numel()))
        for r0 in range(0, n, each):
            r1 = min(n, r0 + each)
            rows = torch.zeros((r1 - r0, *mass.shape[1:]), device=self.device)
            kv.attend(cache, q[r0:r1], step.lens[r0:r1], seqs=step.seqs[r0:r1], mass=rows, out=out[r0:r1])
            for s, at in step.spans.items():
                at = at[(at >= r0) & (at < r1)] - r0
                if len(at):
                    mass[s] += rows[torch.from_numpy(at).to(self.device)].sum(0)
        return out

    def evict(self, budget: int, *, sinks: int = 4, recent: int = 128) -> None:
        """Cuts every sequence of more than `budget` places to `budget`: each
        layer and key head keeps the first `sinks`, the last `recent` and the
        places of the greatest accumulated weight (kv.evict). Later tokens keep
        their positions. As many sequences at a time as there are free pages
        for are copied to those, and their old pages are free afterwards; where
        there are none for a single one, it goes by way of new memory back into
        its own first pages. Caches of more than about 370000 places are
        refused (kv.evict), which changes nothing; an error that only a later
        sequence meets leaves the ones before it cut and the rest as they were."""
        if self.mass is None:
            raise ValueError("evict needs a cache made with mass=True")
        if not 1 <= budget <= self.max_seq or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError(f"budget {budget} of {self.max_seq} places, with {sinks} first and {recent} last")
        long = [s for s in range(self.seqs) if self.pages.length[s] > budget]
        each = -(-budget // self.page_size)
        while long:
            n = min(len(long), len(self.pages.free) // each)
            if n:
                pages = self.pages.take(n * each)
                try:
                    self._cut(long[:n], pages, self.k, self.v, pages, budget, sinks, recent)
                except BaseException:  # nothing has changed but pages that nothing names
                    self.pages.free += pages[::-1]
                    raise
            else:
                n, pages = 1, [int(p) for p in self.pages.table[long[0], :each]]
                shape = (self.k.shape[0], each, *self.k.shape[2:])
                k, v = (torch.empty(shape, dtype=self.k.dtype, device=self.device) for _ in range(2))
                self._cut(long[:1], range(each), k, v, pages, budget, sinks, recent)
            long = long[n:]

    def _cut(self, seqs: list[int], to: list[int], k: torch.Tensor, v: torch.Tensor, pages: list[int], budget: int,
             sinks: int, recent: int) -> None:
        """Evicts from `seqs` into the pages `to` of the pools k, v (all layers'), which become the cache's `pages`."""
        each = len(pages) // len(seqs)
        to_table = self._ints(np.asarray(to).reshape(len(seqs), each))
        at = torch.tensor(seqs, device=self.device)
        table, lens = self.table[at], self._ints(self.pages.length[seqs])
        own = None if k is self.k else torch.tensor(pages, device=self.device)
        masses = []
        for layer in range(len(self.layers)):
            old = kv.PagedKV(self.k[layer], self.v[layer], table, self.status)
            new = kv.PagedKV(k[layer], v[layer], to_table, self.status)
            mass = torch.zeros((len(seqs), *self.mass.shape[2:]), device=self.device)
            kv.evict(old, lens, self.mass[layer][at], new, mass, budget, sinks=sinks, recent=recent)
            masses.append(mass)
        # every layer has been chosen from: nothing is refused from here on
        self._number += 1
        for layer, mass in enumerate(masses):
            self.mass[layer].index_copy_(0, at, mass)
            if own is not None:
                self.k[layer].index_copy_(0, own, k[layer])
                self.v[layer].index_copy_(0, own, v[layer])
        for i, s in enumerate(seqs):
            self.pages.replace(s, pages[i * each:(i + 1) * each], budget)
        self.table.copy_(torch.from_numpy(self.pages.table))

    def release(self, seq: int) -> None:
        """Forgets a sequence; its pages are free."""
        self.pages.release(seq)
        self._number += 1
        self.table.copy_(torch.from_numpy(self.pages.table))
        if self.mass is not None:
            self.mass[:, seq].zero_()

    def check(self) -> None:
        """PagedKV.check() of all layers."""
        self.layers[0].check()
