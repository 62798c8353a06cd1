"""Cache and state bookkeeping of the serving engine (host side, no GPU): KV pages and recurrent-state slots.

The reference keeps a block allocator + per-sequence block tables for paged attention (src/engine/batch_engine.rs, block_size 16,
src/config/inference.rs:94-98).  Layer-list models with recurrent layers need a second resource: one state slot per live request
(convolution tails, state-space matrices, element-wise recurrent states), handed out on admission and returned on release; the
request's last token is kept beside it for embeddings that hash neighbouring tokens.  Pages and slots are reused; a new
request never sees what the previous owner left because a sequence at position 0 reads its carried state as zero and its pages
are written before they are read.

Requests may share pages (`fork`): a page has as many owners as requests hold it, and a request that is about to write into a page
with other owners gets a copy of its own first (`reserve` names the copies to make).  `truncate` takes a request's last tokens back,
`compact` moves the pages in use to the front of the pool.  `evict` cuts a request's cached rows back: from then on it has fewer rows
than tokens, and its next token's row is not its position.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple


class CacheFull(RuntimeError):
    pass


class PagePool:
    """free list of KV pages (last freed, first reused: recycled pages turn up early and out of order), with the number of owners of each"""

    def __init__(self, num_blocks: int, block_size: int):
        assert num_blocks >= 0 and block_size >= 1
        self.num_blocks, self.block_size = num_blocks, block_size
        self._free: List[int] = list(range(num_blocks - 1, -1, -1))
        self._owners: List[int] = [0] * num_blocks

    @property
    def free_blocks(self) -> int:
        return len(self._free)

    def owners(self, b: int) -> int:
        return self._owners[b]

    def alloc(self, n: int) -> List[int]:
        if n > len(self._free):
            raise CacheFull(f"{n} KV pages wanted, {len(self._free)} free")
        out = [self._free.pop() for _ in range(n)]
        for b in out:
            self._owners[b] = 1
        return out

    def share(self, blocks: Sequence[int]) -> None:
        """one more owner of each"""
        for b in blocks:
            assert self._owners[b] > 0
            self._owners[b] += 1

    def free(self, blocks: Sequence[int]) -> None:
        """one owner less; a page without owners is free"""
        for b in blocks:
            assert 0 <= b < self.num_blocks and self._owners[b] > 0
            self._owners[b] -= 1
            if self._owners[b] == 0:
                self._free.append(b)

    def compact(self) -> Dict[int, int]:
        """gives the pages in use the lowest numbers: {old: new} of those that move (the new ones were free)"""
        used = [b for b in range(self.num_blocks) if self._owners[b]]
        n = len(used)
        room = [b for b in range(n) if not self._owners[b]]
        moves = dict(zip([b for b in used if b >= n], room))
        for old, new in moves.items():
            self._owners[new], self._owners[old] = self._owners[old], 0
        self._free = list(range(self.num_blocks - 1, n - 1, -1))
        return moves


class SlotPool:
    def __init__(self, n: int):
        self.n = n
        self._free: List[int] = list(range(n - 1, -1, -1))

    @property
    def free_slots(self) -> int:
        return len(self._free)

    def alloc(self) -> int:
        if not self._free:
            raise CacheFull(f"all {self.n} state slots are in use")
        return self._free.pop()

    def free(self, s: int) -> None:
        assert 0 <= s < self.n and s not in self._free
        self._free.append(s)


@dataclass
class SeqState:
    """what one live request holds"""
    rid: str
    slot: int
    blocks: List[int] = field(default_factory=list)
    n_tokens: int = 0          # tokens already in the cache / folded into the state
    last_token: int = -1       # the last token fed (state of embeddings that hash the previous token with the current one)
    gone: int = 0              # tokens whose rows have left the cache
    whole_from: int = 0        # the rows of its tokens from here on are all there, in order

    @property
    def rows(self) -> int:
        return self.n_tokens - self.gone


class CacheManager:
    """pages for `max_tokens` tokens in all and `max_seqs` state slots.  pooled: sizes of the pooled blocks that layers keep (their means lie in the page of a
    block's first position, so a page is written again until the blocks that begin in it are complete)"""

    def __init__(self, max_tokens: int, max_seqs: int, block_size: int = 16, pooled: Sequence[int] = ()):
        self.block_size, self.pooled = block_size, tuple(pooled)
        # every live request may hold one partly filled page
        self.pages = PagePool(-(-max_tokens // block_size) + max_seqs, block_size)
        self.slots = SlotPool(max_seqs)
        self.live: Dict[str, SeqState] = {}

    def admit(self, rid: str) -> SeqState:
        if rid in self.live:
            raise ValueError(f"request {rid} is already live")
        s = SeqState(rid, self.slots.alloc())
        self.live[rid] = s
        return s

    def can_admit(self) -> bool:
        return self.slots.free_slots > 0

    def _first_written(self, seq: SeqState) -> int:
        """index of the first page that the request's next tokens write into"""
        return min([seq.rows] + [seq.rows // p * p for p in self.pooled]) // self.block_size

    def _shared(self, seq: SeqState) -> List[int]:
        return [i for i in range(self._first_written(seq), len(seq.blocks)) if self.pages.owners(seq.blocks[i]) > 1]

    def pages_to_copy(self, seq: SeqState) -> int:
        """shared pages that the request's next token makes it copy"""
        return len(self._shared(seq))

    def pages_needed(self, seq: SeqState, n_new: int) -> int:
        """free pages that n_new more tokens take: new ones, and copies of shared ones that would be written"""
        grow = max(0, -(-(seq.rows + n_new) // self.block_size) - len(seq.blocks))
        return grow + (len(self._shared(seq)) if n_new > 0 else 0)

    def reserve(self, seq: SeqState, n_new: int) -> List[Tuple[int, int]]:
        """make room for n_new more tokens of this request; returns the page copies (from, to) to make before they are written"""
        shared = self._shared(seq) if n_new > 0 else []
        new = self.pages.alloc(self.pages_needed(seq, n_new))
        copies = []
        for i in shared:
            b = new.pop()
            copies.append((seq.blocks[i], b))
            self.pages.free([seq.blocks[i]])
            seq.blocks[i] = b
        seq.blocks += new
        return copies

    def fork(self, rid: str, new_rid: str) -> SeqState:
        """a second request that continues from where `rid` is: its pages are shared, its state slot is its own (the caller copies the slot's contents)"""
        src = self.live[rid]
        s = self.admit(new_rid)
        self.pages.share(src.blocks)
        s.blocks, s.n_tokens, s.last_token = list(src.blocks), src.n_tokens, src.last_token
        s.gone, s.whole_from = src.gone, src.whole_from
        return s

    def truncate(self, rid: str, n_tokens: int, last_token: int) -> None:
        """the request's tokens from n_tokens on leave the cache; last_token: its token n_tokens - 1 (-1: none)"""
        s = self.live[rid]
        if not 0 <= n_tokens <= s.n_tokens:
            raise ValueError(f"request {rid} holds {s.n_tokens} tokens, not {n_tokens}")
        if s.gone and n_tokens < s.whole_from:
            raise ValueError(f"request {rid} has lost rows before its token {s.whole_from}: it cannot be taken back to {n_tokens}")
        keep = -(-(n_tokens - s.gone) // self.block_size)
        self.pages.free(s.blocks[keep:])
        s.blocks = s.blocks[:keep]
        s.n_tokens, s.last_token = n_tokens, last_token

    def evict(self, rid: str, keep: int, recent: int) -> Optional[Tuple[List[int], List[int], int]]:
        """the request's rows are cut back to `keep`, its last `recent` ones among them.  Returns (pages it had, pages that the rows go to, rows it had): shared pages are replaced
        by free ones, the rest stay; or None where there are not enough free ones.  The caller moves the rows and then gives back what `evicted` names."""
        s = self.live[rid]
        assert 0 < recent <= keep < s.rows
        had, n = list(s.blocks), s.rows
        to = had[:-(-keep // self.block_size)]
        shared = [i for i, b in enumerate(to) if self.pages.owners(b) > 1]
        if len(shared) > self.pages.free_blocks:
            return None
        for i, b in zip(shared, self.pages.alloc(len(shared))):
            to[i] = b
        s.blocks, s.gone, s.whole_from = list(to), s.gone + n - keep, s.n_tokens - recent
        return had, to, n

    def evicted(self, had: Sequence[int], to: Sequence[int]) -> None:
        """the pages that an eviction has emptied lose an owner"""
        kept = set(to)
        self.pages.free([b for b in had if b not in kept])

    def compact(self) -> List[Tuple[int, int]]:
        """moves the pages in use to the front of the pool; returns the page copies (from, to) to make"""
        moves = self.pages.compact()
        for s in self.live.values():
            s.blocks = [moves.get(b, b) for b in s.blocks]
        return list(moves.items())

    def release(self, rid: str) -> None:
        s = self.live.pop(rid)
        self.pages.free(s.blocks)
        self.slots.free(s.slot)
        s.blocks = []
