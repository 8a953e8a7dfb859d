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

Several continuations of a text share what they have in common: reorder() lets
sequences go on from others (beams, forks) over the same pages, of which only
the partly filled last one is copied, and a step with parents= carries trees of
drafted tokens, of which accept() keeps one path.

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
    were evicted), `uses` how many sequences have a page. Sequences share full
    pages only: the page that a sequence writes next is its own."""

    def __init__(self, seqs: int, width: int, pages: int, page_size: int):
        if min(seqs, width, pages, page_size) < 1:
            raise ValueError(f"{seqs} sequences, tables of {width}, {pages} pages of {page_size}: at least one each")
        self.page_size = page_size
        self.table = np.full((seqs, width), -1, dtype=np.int32)
        self.length = np.zeros(seqs, dtype=np.int64)
        self.position = np.zeros(seqs, dtype=np.int64)
        self.free = list(range(pages - 1, -1, -1))  # the next one to give out is the last
        self.uses = np.zeros(pages, dtype=np.int32)

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
            self.table[s, o] = self.take(1)[0]
        nth = np.zeros(len(seqs), dtype=np.int64)  # how often the row's sequence came before it
        for s in ids:
            at = np.flatnonzero(seqs == s)
            nth[at] = np.arange(len(at))
        positions, slots = self.position[seqs] + nth, self.length[seqs] + nth
        self.length[ids] += counts
        self.position[ids] += counts
        return positions, slots

    def shrink(self, seqs) -> None:
        """Takes the last extend(seqs), or its last places, back: places, positions and pages as before them."""
        ids, counts = np.unique(np.asarray(seqs, dtype=np.int64), return_counts=True)
        for s, c in zip(ids[::-1], counts[::-1]):
            self.length[s] -= c
            self.position[s] -= c
            for o in range(self._pages(self.length[s] + c) - 1, self._pages(self.length[s]) - 1, -1):
                self.give_back([self.table[s, o]])
                self.table[s, o] = -1

    def take(self, n: int) -> list[int]:
        """n free pages, out of the pool."""
        if n > len(self.free):
            raise ValueError(f"the KV cache is out of pages ({n} needed, {len(self.free)} free)")
        pages = [self.free.pop() for _ in range(n)]
        self.uses[pages] = 1
        return pages

    def give_back(self, pages) -> None:
        """One use less of each page; those without any are free."""
        for p in pages:
            self.uses[p] -= 1
            if not self.uses[p]:
                self.free.append(int(p))

    def replace(self, seq: int, pages: list[int], length: int) -> None:
        """The sequence's places are now `length`, in `pages` (taken ones, or its own); its old pages that are none
        of them are given back."""
        kept = set(pages)
        self.give_back([p for p in self.table[seq] if p >= 0 and int(p) not in kept])
        self.table[seq] = -1
        self.table[seq, :len(pages)] = pages
        self.length[seq] = length

    def release(self, seq: int) -> None:
        self.known(seq)
        self.replace(seq, [], 0)
        self.position[seq] = 0

    def reorder(self, seqs, parents) -> tuple[list[int], list[int], list[int]]:
        """Sequence seqs[i] becomes what parents[i] was before the call: the same full pages, and of a partly filled
        last one a copy each, unless it is the only one left to have it. Returns the copies to make: from these
        pages, to these (free before or freed now), so many places. Raises ValueError, changing nothing, if the
        pool is full."""
        seqs, parents = (np.asarray(a, dtype=np.int64) for a in (seqs, parents))
        if seqs.ndim != 1 or seqs.shape != parents.shape or len(set(seqs.tolist())) != len(seqs):
            raise ValueError("reorder: distinct sequences, and a parent for each")
        self.known(seqs)
        self.known(parents)
        old, uses, free = self.table.copy(), self.uses.copy(), list(self.free)
        had, taken = set(seqs.tolist()), set()
        copies = []
        try:
            for s, p in zip(seqs.tolist(), parents.tolist()):
                full, part = divmod(int(self.length[p]), self.page_size)
                row = old[p].copy()
                if part and (p not in had or p in taken):  # the page stays the parent's, or another child has it
                    copies.append((s, full, int(row[full]), part))
                    row[full] = -1
                taken.add(p)
                self.uses[row[row >= 0]] += 1
                self.table[s] = row
            for s in seqs:
                self.give_back(old[s][old[s] >= 0])
            to = self.take(len(copies))
        except BaseException:
            self.table, self.uses, self.free = old, uses, free
            raise
        for (s, full, _, _), page in zip(copies, to):
            self.table[s, full] = page
        self.length[seqs], self.position[seqs] = self.length[parents], self.position[parents]
        return [c[2] for c in copies], to, [c[3] for c in copies]


@dataclass
class Tree:
    """The drafted tokens of a step: tree t's nodes are rows starts[t] .. starts[t + 1] - 1, after the first lens[t]
    places of sequence seqs[t]; parents as kv.attend_tree has them. On the host, and on the device."""

    seqs: np.ndarray
    starts: np.ndarray
    parents: np.ndarray
    lens: np.ndarray
    device: tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]


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
    tree: Tree | None = None      # a step of drafted tokens


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
        self.pools = kv.PagedLayers(self.k, self.v, self.table, self.status)
        self.layers = self.pools.layers
        self.mass = None
        if mass:
            self.mass = torch.zeros((config.num_layers, seqs, config.num_kv_heads, self.max_seq), device=self.device)
        self.select = select
        self.bounds = [kv.PageBounds.new(c) for c in self.layers] if select is not None else None
        self._number = 0  # steps, evictions, releases and the like so far
        self._drafted = None  # the step of drafted tokens that is neither accepted nor taken back

    @property
    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()

    def length(self, seq: int = 0) -> int:
        """The places sequence `seq` uses."""
        self.pages.known(seq)
        return int(self.pages.length[seq])

    def room(self, seq: int = 0) -> int:
        """The places that sequence `seq` can still get."""
        n = self.length(seq)
        return min(self.max_seq - n, -n % self.page_size + len(self.pages.free) * self.page_size)

    @property
    def drafted(self) -> Step | None:
        """The step of drafted tokens that accept() or undo() has to end."""
        return self._drafted

    def _ints(self, a) -> torch.Tensor:
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(self.device)

    def _settled(self) -> None:
        if self._drafted is not None:
            raise ValueError("drafted tokens are neither accepted nor taken back")

    def step(self, seqs, parents=None) -> Step:
        """Places for one more token of every sequence in `seqs`, row by row; the tables follow. Every layer
        has to attend with the step; where one cannot, undo(step) takes it back. With `parents` the rows are drafted
        tokens, each sequence's in a run: a row's parent is a row of its run before it, counted in the run, or
        -1 for the sequence's last token. The next call has to be accept() or undo()."""
        self._settled()
        seqs = np.asarray(seqs, dtype=np.int64)
        drafted = None if parents is None else self._trees(seqs, parents)
        before = self.pages.length.copy()
        positions, slots = self.pages.extend(seqs)
        self._number += 1
        try:
            self.table.copy_(torch.from_numpy(self.pages.table))
            tree = None
            if drafted is not None:
                starts, own, depth = drafted
                named = seqs[starts[:-1]]
                lens = before[named]
                positions = self.pages.position[seqs] - np.repeat(np.diff(starts), np.diff(starts)) + depth
                sent = self._ints(np.concatenate([named, starts, own, lens]))
                tree = Tree(named, starts, own, lens, sent.split([len(named), len(starts), len(own), len(lens)]))
            rows = self._ints(np.stack([seqs, positions, slots, slots + 1]))
            both = self._ints(np.stack([self.pages.length, before]))
            spans = {int(s): np.flatnonzero(seqs == s) for s in np.unique(seqs)}
            step = Step(rows[0], rows[1], rows[2], rows[3], spans,
                        len(seqs) == self.seqs and bool(np.all(seqs == np.arange(self.seqs))), both[0], both[1],
                        self._number, int(slots.max()) + 1 if len(slots) else 0, {}, tree)
        except BaseException:
            self._give_back(seqs)
            raise
        if tree is not None:
            self._drafted = step
        return step

    def _trees(self, seqs: np.ndarray, parents) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """(starts of the trees and their end, parents, every row's depth) of drafted tokens."""
        if self.mass is not None:
            raise ValueError("drafted tokens: not in a cache made with mass=True, whose weights they would enter")
        parents = np.asarray(parents, dtype=np.int64)
        if parents.shape != seqs.shape or seqs.ndim != 1 or not len(seqs):
            raise ValueError(f"parents: one for each of {seqs.shape} drafted tokens, got {parents.shape}")
        first = np.flatnonzero(np.concatenate([[True], seqs[1:] != seqs[:-1]]))
        starts = np.append(first, len(seqs))
        if len(set(seqs[first].tolist())) != len(first):
            raise ValueError("drafted tokens: each sequence's have to be in one run")
        within = np.arange(len(seqs)) - np.repeat(first, np.diff(starts))
        if np.any(parents < -1) or np.any(parents >= within):
            raise ValueError("parents: -1, or a token of the run before the child")
        if np.diff(starts).max() > 256 or len(first) > 4096:
            raise ValueError(f"{len(first)} trees of up to {np.diff(starts).max()} drafted tokens: at most 4096 of 256")
        depth = np.zeros(len(seqs), dtype=np.int64)
        for i, (p, w) in enumerate(zip(parents.tolist(), within.tolist())):
            if p >= 0:
                depth[i] = depth[i - w + p] + 1
        return starts, parents, depth

    def accept(self, step: Step, paths) -> None:
        """Keeps of each of a step's trees the drafted tokens `paths[t]`, from one with parent -1 on each the parent
        of the next (none: the sequence is as before the step); their keys and values move together behind what the
        sequence had, and the places of the others are given back. Only the cache's last step."""
        if step.tree is None or step is not self._drafted:
            raise ValueError("accept: not the cache's last step of drafted tokens")
        tree = step.tree
        if len(paths) != len(tree.seqs):
            raise ValueError(f"accept: {len(paths)} paths for {len(tree.seqs)} trees")
        paths = [[int(i) for i in path] for path in paths]
        for t, path in enumerate(paths):
            own = tree.parents[tree.starts[t]:tree.starts[t + 1]]
            if any(not 0 <= i < len(own) or own[i] != p for p, i in zip([-1, *path], path)):
                raise ValueError(f"accept: {path} is no path of tree {t}")
        moved = [t for t, path in enumerate(paths) if path != list(range(len(path)))]
        if moved:
            keep = np.full((len(moved), max(len(paths[t]) for t in moved)), -1)
            for row, t in zip(keep, moved):
                row[:len(paths[t])] = paths[t]
            rows = self._ints(np.stack([tree.seqs[moved], tree.lens[moved], [len(paths[t]) for t in moved]]))
            kv.compact(self.pools, rows[1], self._ints(keep), rows[2], seqs=rows[0])
        self._drafted = None
        sizes = np.diff(tree.starts)
        self._give_back(np.repeat(tree.seqs, [n - len(path) for n, path in zip(sizes, paths)]))
        if self.bounds is not None:
            now = self._ints(self.pages.length)
            for cache, bounds in zip(self.layers, self.bounds):
                kv.page_bounds(cache, bounds, now, step.start)

    def reorder(self, seqs, parents) -> None:
        """Sequence seqs[i] goes on from what parents[i] holds now, however many do: a text's beams after a choice,
        or copies of a text (its own sequence need not be among seqs). They share its full pages; of a partly
        filled last page all but one get copies, in every layer at once. What no sequence has any more is free."""
        self._settled()
        src, dst, used = self.pages.reorder(seqs, parents)
        self._number += 1
        self.table.copy_(torch.from_numpy(self.pages.table))
        if src:
            rows = self._ints(np.stack([src, dst, used]))
            kv.copy_pages(self.pools, rows[0], rows[1], used=rows[2])
        if self.mass is not None:
            to, frm = (torch.as_tensor(np.asarray(a, dtype=np.int64)).to(self.device) for a in (seqs, parents))
            self.mass[:, to] = self.mass[:, frm]

    def undo(self, step: Step) -> None:
        """Takes a step back of which not every layer has attended (an error between layers): lengths,
        positions, pages and accumulated weights are what they were. Only the cache's last step, before
        any eviction or release after it."""
        if step.number != self._number:
            raise ValueError("undo: not the cache's last step")
        self._drafted = None
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
        into the pages, then every row over its sequence up to itself; [n, heads, head_dim].
        Drafted tokens attend to all of their sequence's pages, selected or not, and
        to their ancestors."""
        cache = self.layers[layer]
        q = kv.append(cache, qkv, step.positions, heads, theta, seqs=step.seqs, slots=step.slots)
        if step.tree is not None:
            seqs, starts, parents, lens = step.tree.device
            return kv.attend_tree(cache, q, lens, starts, parents, seqs=seqs)
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
        the first pages that it shares with no other sequence, and free ones
        (ValueError where both are too few). Caches of more than about 370000 places are
        refused (kv.evict), which changes nothing; an error that only a later
        sequence meets leaves the ones before it cut and the rest as they were."""
        if self.mass is None:
            raise ValueError("evict needs a cache made with mass=True")
        if not 1 <= budget <= self.max_seq or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError(f"budget {budget} of {self.max_seq} places, with {sinks} first and {recent} last")
        self._settled()
        long = [s for s in range(self.seqs) if self.pages.length[s] > budget]
        each = -(-budget // self.page_size)
        while long:
            n = min(len(long), len(self.pages.free) // each)
            if n:
                pages = self.pages.take(n * each)
                try:
                    self._cut(long[:n], pages, self.k, self.v, pages, budget, sinks, recent)
                except BaseException:  # nothing has changed but pages that nothing names
                    self.pages.give_back(pages[::-1])
                    raise
            else:
                n, pages = 1, [int(p) for p in self.pages.table[long[0]] if p >= 0 and self.pages.uses[p] == 1][:each]
                taken = self.pages.take(each - len(pages))
                shape = (self.k.shape[0], each, *self.k.shape[2:])
                try:
                    k, v = (torch.empty(shape, dtype=self.k.dtype, device=self.device) for _ in range(2))
                    self._cut(long[:1], range(each), k, v, pages + taken, budget, sinks, recent)
                except BaseException:
                    self.pages.give_back(taken[::-1])
                    raise
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
        """Forgets a sequence; its pages that no other one has are free."""
        self._settled()
        self.pages.release(seq)
        self._number += 1
        self.table.copy_(torch.from_numpy(self.pages.table))
        if self.mass is not None:
            self.mass[:, seq].zero_()

    def check(self) -> None:
        """PagedKV.check() of all layers."""
        self.layers[0].check()
