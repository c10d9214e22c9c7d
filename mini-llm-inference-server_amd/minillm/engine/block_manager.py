"""Pool block accounting for the paged KV cache (reference src/minillm/engine/block_manager.py:21-96 states
the rules; this is an independent design).

Rules the engine relies on:
- a block is held (by as many block tables as list it), idle-blank (no KV worth keeping) or idle-named
  (no holder, but the prefix cache names it, so its KV may be revived);
- allocation takes idle-blank blocks first, oldest release first (the pool starts as 0 .. n-1), and only
  then evicts idle-named blocks, least recently released first, dropping their names;
- a released table is walked from its last block to its first, so a chain's tail is evicted before its
  head (a lookup stops at the first unnamed block, so an evicted head would strand the rest).

Design: per-block holder counts in an int32 array, and one reclaim heap of (tier, ticket, block) for the
idle blocks, tier 0 blank and tier 1 named, tickets increasing with every release.  Popping the heap
yields exactly the order above.  Re-acquiring an idle block voids its entry by setting the block's ticket
to -1 (a stale entry is dropped when it surfaces), so nothing is searched or moved on a prefix hit.
"""

from __future__ import annotations

import heapq
from collections import Counter

import numpy as np

from ..attention.metadata import DeviceBlockTables

BLANK, NAMED = 0, 1


class BlockManager:
    def __init__(self, num_blocks: int, block_size: int, prefix=None) -> None:
        self.num_blocks = int(num_blocks)
        self.block_size = int(block_size)
        self.prefix = prefix
        self._holders = np.zeros(self.num_blocks, dtype=np.int32)
        self._ticket = np.arange(self.num_blocks, dtype=np.int64)  # ticket of a block's live heap entry, -1 if none
        self._heap: list[tuple[int, int, int]] = [(BLANK, b, b) for b in range(self.num_blocks)]  # already a heap
        self._next_ticket = self.num_blocks
        self._idle = self.num_blocks  # blocks without a holder
        self._idle_named = 0

    # ------------------------------------------------------------------ queries

    @property
    def num_free(self) -> int:
        """Blocks an allocation may take: idle-blank ones plus idle-named ones it would evict."""
        return self._idle

    @property
    def num_cached(self) -> int:
        """Idle blocks the prefix cache still names."""
        return self._idle_named

    def blocks_for(self, num_tokens: int) -> int:
        return -(-int(num_tokens) // self.block_size)

    def is_cached_unheld(self, block: int) -> bool:
        return self._holders[block] == 0 and self._named(block)

    # ------------------------------------------------------------------ transitions

    def allocate(self, n: int) -> list[int]:
        """`n` blocks, each with one holder: idle-blank blocks first, then evictions of idle-named ones."""
        if n > self._idle:
            raise RuntimeError(f"cannot allocate {n} KV blocks: only {self._idle} are free or evictable")
        out = []
        while len(out) < n:
            tier, ticket, b = heapq.heappop(self._heap)
            if self._ticket[b] != ticket:
                continue  # voided when the block was re-acquired, or superseded
            self._ticket[b] = -1
            if tier == NAMED:
                self._idle_named -= 1
                if self._named(b):
                    self.prefix.forget(b)
            self._holders[b] = 1
            self._idle -= 1
            out.append(b)
        return out

    def acquire(self, blocks: list[int]) -> None:
        """One more holder for each block (prefix-cache hits); an idle block leaves the reclaim heap."""
        for b in blocks:
            if self._holders[b] == 0:
                self._idle -= 1
                if self._named(b):
                    self._idle_named -= 1
                self._ticket[b] = -1
            self._holders[b] += 1
        if len(self._heap) > 2 * self.num_blocks + 64:  # stale entries of revived blocks: compact
            self._heap = [(tier, t, b) for t, (tier, b) in self._live()]
            heapq.heapify(self._heap)

    def free(self, blocks: list[int]) -> None:
        """Drops one holder of every block of a table, tail first; empties the list."""
        while blocks:
            b = blocks.pop()
            self._holders[b] -= 1
            if self._holders[b] == 0:
                self._park(b, NAMED if self._named(b) else BLANK)

    def fork(self, table: list[int], num_tokens: int, reserve_tokens: int = 0) -> tuple[list[int], list[tuple[int, int]]]:
        """A second table over the first `num_tokens` tokens of `table`: it shares the full blocks and gets a block of its own
        for a last one that is not full, with room for `reserve_tokens` in all.  Returns it and the (from, to) blocks to copy
        (PagedKVCache.copy_blocks) before either table grows."""
        full = int(num_tokens) // self.block_size
        used = self.blocks_for(num_tokens)
        if full < 0:
            raise ValueError(f"a table of {num_tokens} tokens")
        if used > len(table):
            raise ValueError(f"a table of {len(table)} blocks does not hold {num_tokens} tokens")
        fresh = self.allocate(max(used, self.blocks_for(reserve_tokens)) - full)  # first: it raises where none are left
        self.acquire(table[:full])
        return table[:full] + fresh, [(table[full], fresh[0])] if used > full else []

    def trim(self, table: list[int], num_tokens: int) -> None:
        """Releases the blocks of `table` behind its first `num_tokens` tokens, in place; resident block tables that mirror the list
        (DeviceBlockTables) follow it.  The owner's own counts are its own to cut: a request's num_cached, and of its names
        (num_named, block_hashes) those of blocks that are no longer full.  A page that the cut goes through will take other tokens:
        it loses its name, and ValueError if another table lists it too (`fork` then gives a table with a copy of it).  It keeps
        the scales of a pool that has them (include/minillm_hip.h)."""
        keep = self.blocks_for(num_tokens)
        if num_tokens < 0:
            raise ValueError(f"a table of {num_tokens} tokens")
        if keep <= len(table) and int(num_tokens) % self.block_size:
            cut = table[keep - 1]
            if self._holders[cut] > 1:
                raise ValueError(f"block {cut} is shared: cut a fork of the table instead")
            if self._named(cut):
                self.prefix.forget(cut)
        if keep < len(table):
            tail = table[keep:]
            del table[keep:]
            self.free(tail)
            DeviceBlockTables.shortened()

    def compact(self) -> list[tuple[int, int]]:
        """Moves every block that holds K/V (held, or named by the prefix cache) into the lowest ids: `gaps` and `move` in one.
        Returns the (from, to) blocks to copy (PagedKVCache.copy_blocks); tables that list a moved block are the caller's to
        rewrite."""
        moves = self.gaps()
        self.move(moves)
        return moves

    def gaps(self) -> list[tuple[int, int]]:
        """The (from, to) blocks that bring every block with K/V into the lowest ids: no block is in both roles, and those to copy
        to hold nothing.  Changes nothing itself."""
        tier = {b: tier for _, (tier, b) in self._live()}
        keeps = [b for b in range(self.num_blocks) if self._holders[b] or tier[b] == NAMED]
        gaps = [b for b in range(len(keeps)) if not self._holders[b] and tier[b] == BLANK]
        return list(zip((b for b in keeps if b >= len(keeps)), gaps))

    def move(self, moves: list[tuple[int, int]]) -> None:
        """The blocks `gaps` gave have been copied: names, holders and the order of eviction follow."""
        live = {b: (tier, t) for t, (tier, b) in self._live()}
        for src, dst in moves:
            self._holders[dst], self._holders[src] = self._holders[src], 0
            if self.prefix is not None:
                self.prefix.move(src, dst)
            blank, (tier, ticket) = live[dst][1], live.get(src, (BLANK, -1))
            # an idle named block keeps its place in the order (a held one has none), the gap passes its own on
            self._ticket[dst], self._ticket[src] = ticket, blank
            live[src] = (BLANK, blank)
            if ticket >= 0:
                live[dst] = (tier, ticket)
            else:
                del live[dst]
        self._heap = [(tier, t, b) for b, (tier, t) in live.items()]
        heapq.heapify(self._heap)

    def clear_cache(self) -> None:
        """Every idle-named block becomes blank (its name dropped), in eviction order."""
        named = sorted((t, b) for t, (tier, b) in self._live() if tier == NAMED)
        for _, b in named:
            self.prefix.forget(b)
            self._idle_named -= 1
            self._idle -= 1  # _park counts it again
            self._park(b, BLANK)

    def check(self, tables: list[list[int]]) -> None:
        """Raises AssertionError unless every block's holder count equals the number of tables listing it
        and every block is in exactly one state (held, idle-blank, idle-named)."""
        held = Counter(b for t in tables for b in t)
        want = np.zeros(self.num_blocks, dtype=np.int64)
        if held:
            idx = np.fromiter(held.keys(), dtype=np.int64, count=len(held))
            want[idx] = np.fromiter(held.values(), dtype=np.int64, count=len(held))
        wrong = np.flatnonzero(want != self._holders)
        if wrong.size:
            raise AssertionError(f"block refcounts disagree with the block tables at blocks {wrong[:10].tolist()}")
        live = self._live()
        idle = [b for _, (_, b) in live]
        no_holder = np.flatnonzero(self._holders == 0).tolist()
        named = sum(1 for _, (tier, _) in live if tier == NAMED)
        if sorted(idle) != no_holder or len(idle) != self._idle or named != self._idle_named:
            raise AssertionError(f"idle-block bookkeeping is inconsistent: {len(idle)} parked, {len(no_holder)} "
                                 f"without a holder, counter {self._idle}; {named} named vs {self._idle_named}")

    # ------------------------------------------------------------------ internals

    def _named(self, block: int) -> bool:
        return self.prefix is not None and self.prefix.is_cached(block)

    def _park(self, b: int, tier: int) -> None:
        t = self._next_ticket
        self._next_ticket += 1
        self._ticket[b] = t
        heapq.heappush(self._heap, (tier, t, b))
        self._idle += 1
        if tier == NAMED:
            self._idle_named += 1

    def _live(self) -> list[tuple[int, tuple[int, int]]]:
        """(ticket, (tier, block)) of every live heap entry."""
        return [(t, (tier, b)) for tier, t, b in self._heap if self._ticket[b] == t]
