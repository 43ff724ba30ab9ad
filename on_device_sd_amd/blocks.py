"""Blocks of a paged cache between the steps: copied, forked, freed and compacted.

``copy_cache_blocks`` copies blocks within all tensors of a cache (every layer's K, V and scales) by one launch.  ``BlockPool`` is the host
bookkeeping: free blocks, how many sequences hold each, copies where a sequence writes to a block that it shares.  The reference's
``PagedKVCache`` (``demo/src/memory/paged_kv_cache.py:228-683``) allocates and frees; it neither shares nor moves blocks.
"""
from __future__ import annotations

import ctypes as C
import dataclasses
from array import array
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .kv import SequenceSlots
from .kv_fp8 import KVCacheFP8
from .ops import _ptr, _raw_device, _same_device, _stream, _wrote

_TENSORS = 16                                              # ODSD_COPY_TENSORS
Blocks = Union[Sequence[int], torch.Tensor]


def _block_list(blocks: Blocks) -> List[int]:
    if isinstance(blocks, torch.Tensor):
        if blocks.is_cuda:
            raise TypeError("block numbers must be on the host: they are checked, and travel with the launch")
        if blocks.is_floating_point() or blocks.is_complex() or blocks.dtype == torch.bool:
            raise TypeError(f"block numbers must be whole numbers, got {blocks.dtype}")
        return blocks.flatten().tolist()
    return list(blocks)


def _block_pairs(src_blocks: Blocks, dst_blocks: Blocks, moves: bool) -> Tuple[array, array]:
    """Both lists as the library takes them.  They are compared as numbers: two tensors that hold the same number are not equal to a set."""
    try:
        src, dst = (array("i", _block_list(blocks)) for blocks in (src_blocks, dst_blocks))      # (no whole number: TypeError)
    except OverflowError:
        raise ValueError("block numbers must be those of blocks of the caches") from None
    n = len(src)
    if len(dst) != n:
        raise ValueError(f"{n} sources for {len(dst)} destinations")
    places = set(dst)
    if len(places) != n or not places.isdisjoint(src):
        raise ValueError("every destination must be named once, and be no source")
    if moves and len(set(src)) != n:
        raise ValueError("a block that moves has one destination")
    return src, dst


def _tensors_of(caches: Sequence[Union[torch.Tensor, KVCacheFP8]], block_dim: int) -> List[torch.Tensor]:
    if block_dim not in (0, 1):
        raise ValueError("block_dim is 0, or 1 behind a dimension of layers")
    tensors: List[torch.Tensor] = []
    for c in caches:
        tensors += [c.k, c.v, c.scales] if isinstance(c, KVCacheFP8) else [c]
    return tensors


def _check_caches(tensors: Sequence[torch.Tensor], num_blocks: int, block_dim: int) -> None:
    for t in tensors:
        if t.dim() <= block_dim or t.shape[block_dim] != num_blocks or not t.is_contiguous():
            raise ValueError(f"a cache {tuple(t.shape)}: caches must be contiguous, with {num_blocks} blocks along dimension {block_dim}")


def copy_cache_blocks(caches: Sequence[Union[torch.Tensor, KVCacheFP8]], src_blocks: Blocks, dst_blocks: Blocks, block_dim: int = 0,
                      block_tables: Optional[torch.Tensor] = None) -> None:
    """Block ``src_blocks[i]`` of every cache to block ``dst_blocks[i]``, in one launch (16 tensors and 384 pairs of them each).

    ``caches``: contiguous tensors [num_blocks, ...], or with ``block_dim=1`` [layers, num_blocks, ...] (a 16-bit cache of rows viewed by
    blocks), and ``KVCacheFP8``.  The lists are the host's (sequences or CPU tensors) and are read before the call returns: a graph
    that captures it copies these blocks at every replay.  A destination is named once and is no source (else ValueError).
    ``block_tables`` (int32, on the GPU, contiguous): entries that name a source name its destination afterwards: the blocks move."""
    tensors = _tensors_of(caches, block_dim)
    if not tensors:
        raise ValueError("no cache to copy in")
    dev = tensors[0].get_device()
    _same_device(dev, *tensors, block_tables)
    if dev != _raw_device():
        with torch.cuda.device(dev):
            return copy_cache_blocks(tensors, src_blocks, dst_blocks, block_dim, block_tables)
    src, dst = _block_pairs(src_blocks, dst_blocks, block_tables is not None)
    n = len(src)
    if tensors[0].dim() <= block_dim:
        raise ValueError(f"a cache {tuple(tensors[0].shape)} has no dimension {block_dim} of blocks")
    num_blocks = tensors[0].shape[block_dim]
    _check_caches(tensors, num_blocks, block_dim)
    if block_tables is not None and (block_tables.dtype != torch.int32 or not block_tables.is_contiguous()):
        raise ValueError("block_tables must be contiguous int32")
    if n == 0:
        return
    if num_blocks >> 31:
        raise _lib.OdsdError(f"copy_cache_blocks: unsupported sizes: {num_blocks} blocks")
    from_at, to_at = src.buffer_info()[0], dst.buffer_info()[0]
    lib = _lib.load()
    tensors_ = [t for t in tensors if t.numel()]
    for at in range(0, max(len(tensors_), 1), _TENSORS):
        some = tensors_[at:at + _TENSORS]
        k = len(some)
        tables = block_tables if at + _TENSORS >= len(tensors_) else None      # (the last launch has them: where one is refused nothing has moved)
        layers = [t.shape[0] if block_dim else 1 for t in some]
        layer_bytes = [t.numel() // l * t.element_size() for t, l in zip(some, layers)]
        rc = lib.odsd_copy_blocks((C.c_void_p * k)(*[t.data_ptr() for t in some]), (C.c_int64 * k)(*[b // num_blocks for b in layer_bytes]),
                                  (C.c_int64 * k)(*layer_bytes), (C.c_int32 * k)(*layers), k, from_at, to_at, n, num_blocks,
                                  _ptr(tables), 0 if tables is None else tables.numel(), _stream())
        if rc == _lib.ERR_SHAPE:                            # (every number is looked at before anything is launched)
            raise ValueError(f"block numbers must be in [0, {num_blocks})")
        if rc:
            _lib.check(rc, "odsd_copy_blocks")
    _wrote(*tensors, block_tables)


class BlockPool:
    """Which blocks of a cache are free, and which sequences hold the others.  ``caches`` / ``block_dim`` as for ``copy_cache_blocks``: where
    a block has to be copied or moved this is done in all of them (without caches the pool only keeps the books).  The pool owns the
    ``block_table`` and ``num_tokens`` of the ``SequenceSlots`` that it is given.  Every call looks at all blocks of the sequences it is given (``append`` for
    64 sequences of 8192 tokens: 0.7 ms with blocks of 256, 7 ms with blocks of 16)."""

    def __init__(self, num_blocks: int, block_size: int, caches: Sequence[Union[torch.Tensor, KVCacheFP8]] = (), block_dim: int = 0):
        if num_blocks < 0 or block_size <= 0:
            raise ValueError(f"a pool of {num_blocks} blocks of {block_size} tokens")
        tensors = _tensors_of(caches, block_dim)
        _check_caches(tensors, num_blocks, block_dim)
        if len({t.device for t in tensors}) > 1:
            raise ValueError("the caches of a pool are on one device")
        self.num_blocks, self.block_size, self.caches, self.block_dim = num_blocks, block_size, list(caches), block_dim
        self.holders = [0] * num_blocks                    # sequences that hold a block
        self._free = list(range(num_blocks - 1, -1, -1))   # the lowest comes last, and is taken first

    @property
    def num_free(self) -> int:
        return len(self._free)

    def _check(self, seq: SequenceSlots) -> None:
        if seq.block_size != self.block_size:
            raise ValueError(f"a sequence with blocks of {seq.block_size} in a pool with blocks of {self.block_size}")
        if any(not 0 <= b < self.num_blocks or self.holders[b] == 0 for b in seq.block_table):
            raise ValueError("the sequence names blocks that the pool has not given out")

    def _drop(self, blocks: Sequence[int]) -> None:
        for b in blocks:
            self.holders[b] -= 1
            if self.holders[b] == 0:
                self._free.append(b)

    def append(self, seqs: Sequence[SequenceSlots], counts: Sequence[int]) -> None:
        """Room for ``counts[i]`` more tokens of each sequence, whose num_tokens grows by them.  A part-filled last block that another
        sequence holds too is replaced by a copy (all copies in one launch).  Too few free blocks: RuntimeError.  A call that raises, for
        those or for a copy that is refused, changes nothing."""
        if len(seqs) != len(counts) or any(c < 0 for c in counts):
            raise ValueError("every sequence needs a count of new tokens, 0 or more")
        if len({id(s) for s in seqs}) != len(seqs):
            raise ValueError("a sequence is named twice")
        need, held = 0, {}
        plan = []                                          # (sequence, count, copies its last block, new blocks)
        for s, c in zip(seqs, counts):
            self._check(s)
            have = -(-s.num_tokens // self.block_size)
            if len(s.block_table) < have:
                raise ValueError(f"{s.num_tokens} tokens in {len(s.block_table)} blocks")
            new = max(0, -(-(s.num_tokens + c) // self.block_size) - len(s.block_table))
            copies = False
            if c:
                # the blocks that the new tokens are written to and that the sequence has already
                for i in range(s.num_tokens // self.block_size, len(s.block_table)):
                    b = s.block_table[i]
                    if held.get(b, self.holders[b]) > 1:
                        if i >= have:
                            raise ValueError("a block behind the sequence's last token is shared")
                        copies = True
                        held[b] = held.get(b, self.holders[b]) - 1
            plan.append((s, c, copies, new))
            need += new + copies
        if need > len(self._free):
            raise RuntimeError(f"{need} blocks are needed, {len(self._free)} are free")
        free = iter(self._free[:-need - 1:-1])             # in the order in which they are taken
        plan = [(s, c, next(free) if copies else None, [next(free) for _ in range(new)]) for s, c, copies, new in plan]
        copied = [(s.block_table[s.num_tokens // self.block_size], to) for s, _, to, _ in plan if to is not None]
        if copied and self.caches:                         # (before the books change: a copy that is refused leaves them as they were)
            copy_cache_blocks(self.caches, [b for b, _ in copied], [to for _, to in copied], self.block_dim)
        del self._free[len(self._free) - need:]
        for s, c, to, new in plan:
            if to is not None:
                at = s.num_tokens // self.block_size
                self._drop([s.block_table[at]])
                s.block_table[at] = to
                self.holders[to] = 1
            for b in new:
                self.holders[b] = 1
            s.block_table.extend(new)
            s.num_tokens += c

    def fork(self, seq: SequenceSlots) -> SequenceSlots:
        """Another sequence with the same tokens so far, in the same blocks; whichever writes to the last one first gets a copy."""
        self._check(seq)
        table = seq.block_table[:-(-seq.num_tokens // self.block_size)]
        for b in table:
            self.holders[b] += 1
        return dataclasses.replace(seq, block_table=list(table))

    def truncate(self, seq: SequenceSlots, num_tokens: int) -> None:
        """Only the first ``num_tokens`` tokens stay (drafts that were not kept go); blocks behind them are given back."""
        self._check(seq)
        if not 0 <= num_tokens <= seq.num_tokens:
            raise ValueError(f"{num_tokens} of {seq.num_tokens} tokens cannot stay")
        keep = -(-num_tokens // self.block_size)
        self._drop(seq.block_table[keep:])
        del seq.block_table[keep:]
        seq.num_tokens = num_tokens
        seq.draft_start_num_tokens = min(seq.draft_start_num_tokens, num_tokens)

    def free(self, seq: SequenceSlots) -> None:
        """The sequence ends: its blocks are given back."""
        self.truncate(seq, 0)

    def compact(self, seqs: Sequence[SequenceSlots], block_tables: Optional[torch.Tensor] = None) -> Dict[int, int]:
        """Held blocks move down into the free ones, so that they are the lowest numbers of the cache; the tables of ``seqs``, all the
        sequences that hold blocks, follow, and so do ``block_tables`` on the GPU.  Returns {old number: new number} of the moved."""
        count = [0] * self.num_blocks
        for s in {id(s): s for s in seqs}.values():
            self._check(s)
            for b in s.block_table:
                count[b] += 1
        if count != self.holders:
            raise ValueError("blocks are held by sequences that were not named")
        live = self.num_blocks - len(self._free)
        holes = [b for b in range(live) if self.holders[b] == 0]
        moved = dict(zip((b for b in range(live, self.num_blocks) if self.holders[b]), holes))
        if not moved:
            return moved
        if self.caches:
            copy_cache_blocks(self.caches, list(moved), list(moved.values()), self.block_dim, block_tables)
        elif block_tables is not None:
            raise ValueError("block_tables follow the copies of a pool with caches")
        for old, new in moved.items():
            self.holders[new], self.holders[old] = self.holders[old], 0
        for s in {id(s): s for s in seqs}.values():
            s.block_table[:] = [moved.get(b, b) for b in s.block_table]
        self._free = list(range(self.num_blocks - 1, live - 1, -1))
        return moved
