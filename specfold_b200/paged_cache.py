"""Paged prefix cache: many sequences of different lengths in one pool of pages.

``PreallocatedKVCache`` holds one running prefix, like the reference's DynamicCache.  A server
runs many requests at once; this cache deals pages of ``page_size`` positions out of one pool to
them, so that a request takes memory for the positions it has, and pages go back when it ends.
The pages of all layers are dealt together: a sequence has one page table.

A step runs new tokens of some sequences through every layer::

    step = cache.step(seqs, q_lens, heads=32)          # reserves pages, plans the work once
    for layer in range(cache.num_layers):
        cache.append(layer, k, v, step)                # [T, Hkv, hd], T = sum(q_lens)
        out, lse = cache.attend(layer, q, step)        # [T, H, hd]
        cache.accumulate(layer, q, lse, step)          # only to evict by weight later

with single tokens, blocks and prompt chunks side by side in one step.  ``window`` / ``sinks``
limit what a token sees to the positions less than ``window`` back and the first ``sinks``
(``release`` then returns the pages no later token will see); ``evict`` cuts sequences to a
budget by accumulated attention weight.

Positions count cached keys: after an eviction a sequence is as long as what stayed, in order
(keys keep the rotary angles they were stored with).  Calls go to the current stream; a cache is
used on one stream at a time.
"""

from __future__ import annotations

import contextlib
import itertools
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from . import kernels as K


class PagedStep:
    """One step's plan and page table (``PagedKVCache.step``)."""

    def __init__(self, seqs: List[int], plan: K.PagedPlan, table: torch.Tensor):
        self.seqs, self.plan, self.table = seqs, plan, table

    def check(self) -> None:
        """Raises what the step's kernels reported.  Synchronises with the device."""
        self.plan.check()


class PagedKVCache:
    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_pages: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 track_mass: bool = False):
        if min(num_layers, num_kv_heads, head_dim, num_pages, page_size) <= 0:
            raise ValueError("layers, kv heads, head dim, pages and page size must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the paged KV cache lives on a CUDA device")
        self.num_layers, self.num_kv_heads, self.head_dim = num_layers, num_kv_heads, head_dim
        self.page_size, self.num_pages, self.dtype, self.device = page_size, num_pages, dtype, device
        self._store = torch.zeros(num_layers, 2, num_pages, num_kv_heads, page_size, head_dim,
                                  dtype=dtype, device=device)
        self._mass = (torch.zeros(num_layers, num_pages, num_kv_heads, page_size, device=device)
                      if track_mass else None)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: Dict[int, List[int]] = {}
        self._len: Dict[int, int] = {}
        self._next = 0

    # ---------------------------------------------------------------- sequences
    def add(self) -> int:
        """A new, empty sequence's id."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def remove(self, seq: int) -> None:
        """Ends a sequence and returns its pages."""
        self._free.extend(p for p in self._pages.pop(seq) if p >= 0)
        del self._len[seq]

    def length(self, seq: int) -> int:
        return self._len[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages(self, seq: int) -> List[int]:
        """The sequence's page ids in order, -1 for released ones."""
        return list(self._pages[seq])

    def _need(self, n: int) -> int:
        return -(-n // self.page_size)

    def _take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise MemoryError(f"{n} pages needed, {len(self._free)} of {self.num_pages} free")
        return [self._free.pop() for _ in range(n)]

    @contextlib.contextmanager
    def _taken(self, counts: Sequence[int]):
        """Lists of free pages, one of each length; they go back to the pool if the body fails."""
        fresh = self._take(sum(counts))
        try:
            it = iter(fresh)
            yield [list(itertools.islice(it, n)) for n in counts]
        except BaseException:
            self._free.extend(reversed(fresh))
            raise

    def _table(self, rows: List[List[int]]) -> torch.Tensor:
        width = max([len(r) for r in rows] + [1])
        return torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32
                            ).reshape(len(rows), width).to(self.device)

    # ---------------------------------------------------------------- a step
    def step(self, seqs: Sequence[int], q_lens: Sequence[int], *, heads: int, block: int = 1,
             window: int = 0, sinks: int = 0) -> PagedStep:
        """Makes room for ``q_lens[i]`` new tokens of ``seqs[i]``, counts them as cached and plans
        the step (``kernels.PagedPlan`` has the mask's meaning).  Nothing changes when the pool
        is too small (MemoryError) or the step fails in another way."""
        seqs = list(seqs)
        if len(set(seqs)) != len(seqs) or len(seqs) != len(q_lens):
            raise ValueError("a step takes every sequence once, with one chunk length each")
        if any(q < 0 for q in q_lens):
            raise ValueError("chunk lengths must not be negative")
        lens = [self._len[s] + q for s, q in zip(seqs, q_lens)]
        more = [self._need(n) - len(self._pages[s]) for s, n in zip(seqs, lens)]
        plan = K.PagedPlan(q_lens, lens, heads=heads, kv_heads=self.num_kv_heads,
                           head_dim=self.head_dim, page_size=self.page_size, dtype=self.dtype,
                           block=block, window=window, sinks=sinks, mass=self._mass is not None,
                           device=self.device)
        with self._taken(more) as fresh:
            rows = [self._pages[s] + new for s, new in zip(seqs, fresh)]
            step = PagedStep(seqs, plan, self._table(rows))
        for s, n, row in zip(seqs, lens, rows):
            self._pages[s], self._len[s] = row, n
        return step

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> None:
        """The step's new keys and values [T, Hkv, hd] of one layer into their pages."""
        K.paged_kv_append(self._store[layer, 0], self._store[layer, 1], k, v, step.table, step.plan,
                          mass_pages=None if self._mass is None else self._mass[layer])

    def attend(self, layer: int, q: torch.Tensor, step: PagedStep, scale: Optional[float] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        """(attention output [T, H, hd], lse [T, H]) of the step's queries over their caches."""
        return K.paged_attention(q, self._store[layer, 0], self._store[layer, 1], step.table, step.plan,
                                 scale=scale)

    def accumulate(self, layer: int, q: torch.Tensor, lse: torch.Tensor, step: PagedStep,
                   scale: Optional[float] = None) -> None:
        """Adds the weights that the step's softmax gave the cached keys (``track_mass``)."""
        if self._mass is None:
            raise ValueError("the cache was made without track_mass")
        K.paged_attention_mass(q, self._store[layer, 0], step.table, lse, self._mass[layer], step.plan,
                               scale=scale)

    # ---------------------------------------------------------------- bounding a sequence
    def release(self, seq: int, window: int, sinks: int = 0) -> int:
        """Returns the pages that no later token of a sequence run with this window and these
        sinks can see; how many."""
        if window <= 0 or sinks < 0:
            raise ValueError("a window must be positive, sinks not negative")
        first = self._len[seq] - window + 1              # the next token's first visible position
        pages, n = self._pages[seq], 0
        for w in range(self._need(sinks), max(0, first) // self.page_size):
            if pages[w] >= 0:
                self._free.append(pages[w])
                pages[w] = -1
                n += 1
        return n

    def evict(self, seqs: Sequence[int], keep: Union[int, Sequence[int]], sinks: int = 0, recent: int = 0
              ) -> List[torch.Tensor]:
        """Cuts every sequence to ``keep`` (or ``keep[i]``) positions, in every layer and kv head by
        accumulated weight: the first ``sinks``, the last ``recent`` and the heaviest others stay, in
        order.  Returns per layer the old positions of what stayed, int32 [len(seqs), Hkv, most
        kept] (-1 after the last).  A sequence within ``keep`` stays where it is; the survivors of
        the others move to free pages and the old ones are returned.  Nothing has changed when there
        are too few (MemoryError; sequence by sequence fewer will do) or the call fails in another
        way."""
        if self._mass is None:
            raise ValueError("the cache was made without track_mass")
        seqs = list(seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("an eviction takes every sequence once")
        lens = [self._len[s] for s in seqs]
        keep = list(keep) if hasattr(keep, "__len__") else [keep] * len(seqs)
        if len(keep) != len(seqs):
            raise ValueError(f"{len(keep)} budgets for {len(seqs)} sequences")
        over = [i for i, n in enumerate(lens) if n > keep[i]]
        cut = [seqs[i] for i in over]
        if any(-1 in self._pages[s] for s in cut):
            raise ValueError("a sequence with released pages cannot be cut by weight")
        plan = K.EvictPlan([lens[i] for i in over], [keep[i] for i in over], kv_heads=self.num_kv_heads,
                           page_size=self.page_size, sinks=sinks, recent=recent, device=self.device)
        with self._taken([self._need(n) for n in plan.stay]) as into:
            table, dst = self._table([self._pages[s] for s in cut]), self._table(into)
            kept = [K.paged_evict(self._store[x, 0], self._store[x, 1], self._mass[x], table, dst, plan)
                    for x in range(self.num_layers)]
            if len(cut) < len(seqs):
                kept = self._with_whole(kept, [min(n, k) for n, k in zip(lens, keep)], over)
        for s, n, new in zip(cut, plan.stay, into):
            self._free.extend(self._pages[s])
            self._pages[s], self._len[s] = new, n
        return kept

    def _with_whole(self, kept: List[torch.Tensor], stay: List[int], over: List[int]) -> List[torch.Tensor]:
        """``kept`` of the sequences ``over`` alone, with the rows of those that stayed whole."""
        j = torch.arange(max(stay), dtype=torch.int32)
        whole = torch.where(j < torch.tensor(stay)[:, None], j, -1)[:, None].repeat(1, self.num_kv_heads, 1).to(self.device)
        rows = torch.tensor(over, dtype=torch.long).to(self.device)
        out = [whole.clone() for _ in kept]
        for o, k in zip(out, kept):
            o[rows, :, :k.shape[2]] = k
        return out
