"""Copying, forking, compacting and freeing the blocks of a paged cache.

No counterpart in the reference, whose blocks are only appended to and freed
with their sequence (``src/inference/paged_kv_cache.py:87-169``).  Block
bookkeeping is host work (``BlockTable``, ``BlockAllocator``); the bytes move
in one ``nf_kv_move`` or ``nf_copy_blocks`` launch over every layer's K and V.

A block that several tables (or the prefix index) hold is never written: a
sequence that would append into one gets a copy first.
"""

from __future__ import annotations

from array import array

import numpy as np
import torch

from nifre_b200 import _lib
from nifre_b200.block_allocator import BlockPoolExhaustedError


class PageOps:
    """Page operators of ``PagedKVCache``."""

    # False: the rows of the dense cache own their blocks for good
    _tables_move = True

    # ------------------------------------------------------------------ copies
    def copy_blocks(self, src, dst) -> None:
        """Copy the contents of blocks ``src[i]`` to blocks ``dst[i]``, K and V of every layer.

        Lists of block ids, or int32 CUDA tensors (then read by the kernel:
        ids out of range are skipped and flagged for ``check_status``).  The
        destinations must be distinct and none of them a source.
        """
        if torch.is_tensor(src) != torch.is_tensor(dst):
            raise ValueError("src and dst must both be lists or both be tensors")
        if torch.is_tensor(src):
            for name, t in (("src", src), ("dst", dst)):
                if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                    raise ValueError(f"{name} must be a contiguous one-dimensional int32 tensor")
                _lib.require_cuda(t, name)
                if t.device.index != self._dev_index:
                    raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
            if src.numel() != dst.numel():
                raise ValueError(f"{src.numel()} source blocks, {dst.numel()} destinations")
        else:
            a, b = np.asarray(src, dtype=np.int64).reshape(-1), np.asarray(dst, dtype=np.int64).reshape(-1)
            if len(a) != len(b):
                raise ValueError(f"{len(a)} source blocks, {len(b)} destinations")
            if len(a) and (min(a.min(), b.min()) < 0 or max(a.max(), b.max()) >= self.num_blocks):
                raise ValueError(f"block_id out of range [0, {self.num_blocks})")
            if len(np.unique(b)) != len(b) or np.isin(b, a).any():
                raise ValueError("destination blocks must be distinct and none of them a source")
            if not len(a):
                return
            ids = torch.from_numpy(np.stack([a, b]).astype(np.int32)).pin_memory().to(self.device, non_blocking=True)
            src, dst = ids[0], ids[1]
        self._copy_ids(src, dst)

    def _copy_ids(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        if not src.numel():
            return
        args = (self._k_ptr[0], self._v_ptr[0], self._layer_bytes, self.num_layers, self.block_size * self._row_bytes,
                self.num_blocks, src.data_ptr(), dst.data_ptr(), src.numel(), self._status_ptr, self._stream())
        if torch.cuda.current_device() == self._dev_index:
            rc = _lib.load().nf_copy_blocks(*args)
        else:
            with torch.cuda.device(self._dev_index):
                rc = _lib.load().nf_copy_blocks(*args)
        if rc:
            _lib.check(rc, "nf_copy_blocks")

    def _move_rows(self, moves, pos, most: int) -> None:
        """One launch of row moves (flat: source row, destination row, rows -- at most ``most`` --, continues) and
        position records (flat: slot, value)."""
        if not moves and not pos:
            return
        n_moves, n_pos = len(moves) // 4, len(pos) // 2
        flat = array("i", moves + pos)
        if n_moves <= _lib.MOVE_LIST and n_pos <= _lib.MOVE_LIST:  # read before the call returns
            mp, on_device = flat.buffer_info()[0], 0
        else:
            keep = torch.frombuffer(flat, dtype=torch.int32).pin_memory().to(self.device, non_blocking=True)
            mp, on_device = keep.data_ptr(), 1
        args = (self._k_ptr[0], self._v_ptr[0], self._layer_bytes, self.num_layers, self._row_bytes, self._pool_rows,
                mp if moves else None, n_moves, most, mp + 16 * n_moves if pos else None, n_pos,
                self._pos_ptr, self.batch_size, on_device, self._status_ptr, self._stream())
        if torch.cuda.current_device() == self._dev_index:
            rc = _lib.load().nf_kv_move(*args)
        else:
            with torch.cuda.device(self._dev_index):
                rc = _lib.load().nf_kv_move(*args)
        if rc:
            _lib.check(rc, "nf_kv_move")

    def _slots(self, slots, what: str) -> list[int]:
        got = [int(s) for s in slots]
        if got and (min(got) < 0 or max(got) >= self.batch_size):
            raise IndexError(f"{what} out of range [0, {self.batch_size}): {got}")
        return got

    def _refuse_open(self, slots, what: str) -> None:
        plan = self._plan
        if plan is not None and not plan.closed and np.isin(np.asarray(slots), plan.slots).any():
            raise RuntimeError(f"{what}: the slot is part of a step that is not finished")

    # ------------------------------------------------------------------ forks
    def fork(self, src_slots, dst_slots) -> None:
        """Make slot ``dst_slots[i]`` continue the sequence of slot ``src_slots[i]``.

        The full blocks are shared (reference counts); a partly filled last
        block is copied to a block of the destination's own, in every layer.
        What a destination held is released first; forking again into the slots
        of an earlier fork reuses their own blocks.  Destinations must be
        distinct, and no source.  When the pool cannot hold the copies the
        destinations are left empty and BlockPoolExhaustedError is raised.
        """
        if not self._tables_move:
            raise ValueError("the rows of a dense cache own their storage: they cannot share blocks")
        src, dst = self._slots(src_slots, "source slot"), self._slots(dst_slots, "destination slot")
        if len(src) != len(dst):
            raise ValueError(f"{len(src)} source slots, {len(dst)} destinations")
        if len(set(dst)) != len(dst) or set(dst) & set(src):
            raise ValueError("destination slots must be distinct and none of them a source")
        if not dst:
            return
        self._refuse_open(dst, "fork")
        bs, tables, alloc = self.block_size, self.block_tables, self.block_allocator
        length, counts = self.pos_host.tolist(), alloc._refcount
        held = {}  # per source: length, full blocks, tokens of the last block, its full blocks, its last block
        for s in src:
            if s not in held:
                full, tail = divmod(length[s], bs)
                blocks = tables[s]._physical_blocks
                held[s] = (length[s], full, tail, blocks[:full], blocks[full] * bs if tail else 0)
        changed = []
        for s, d in zip(src, dst):
            # a slot forked before from the same blocks keeps them
            _, full, tail, want, _ = held[s]
            have = tables[d]._physical_blocks
            if tail:
                if len(have) != full + 1 or counts[have[full]] != 1 or have[:full] != want:
                    changed.append((s, d))
            elif have != want:
                changed.append((s, d))
        if changed:
            self._refork(changed, held, dst)
        self.pos_host[dst] = [held[s][0] for s in src]
        if self._hole_end.any():
            self._hole_first[dst], self._hole_end[dst] = self._hole_first[src], self._hole_end[src]
        moves, pos = [], []
        for s, d in zip(src, dst):
            n, full, tail, _, row = held[s]
            if tail:
                moves += (row, tables[d]._physical_blocks[full] * bs, tail, 0)
            pos += (d, n)
        self._move_rows(moves, pos, bs)

    def _refork(self, pairs, held, dst) -> None:
        """Give the destination slots of the pairs their sources' full blocks and a last block of their own.
        ``dst``: all of the call's destinations, which an exhausted pool leaves empty."""
        tables, alloc = self.block_tables, self.block_allocator

        def empty(slots):
            for d in reversed(slots):  # the last released block is the next one allocated
                tables[d].clear()
                self.pos_host[d] = 0
                self._clear_hole(d)

        empty([d for _, d in pairs])
        need, free = sum(held[s][2] > 0 for s, _ in pairs), alloc.free_count
        if need > free:
            empty(dst)
            self._move_rows([], [x for d in dst for x in (d, 0)], 0)
            raise BlockPoolExhaustedError(f"need {need} blocks, only {free} free")
        for s, d in pairs:
            tables[d].share(held[s][3])
            if held[s][2]:
                tables[d].ensure_capacity(held[s][0])

    # ------------------------------------------------------------------ drafted tokens
    def keep_tokens(self, plan, paths) -> None:
        """After a tree step, keep the accepted tokens of each sequence and drop the rest of its draft.

        ``plan``: the step's (closed) plan; ``paths[i]``: the accepted new
        tokens of sequence i, ascending indices into its draft.  Their rows are
        moved together behind the context, in every layer, and the sequence
        ends with the last of them.  Its blocks stay (the next draft needs
        them); ``truncate`` gives them back.
        """
        if not plan.closed:
            raise RuntimeError("keep_tokens: the step is not finished")
        if len(paths) != plan.n_seqs:
            raise ValueError(f"{len(paths)} paths for {plan.n_seqs} sequences")
        slots, ctx, n = plan.slots.tolist(), plan.ctx_before.tolist(), plan.q_lens.tolist()
        self._slots(slots, "cache slot")
        kept = []
        for s, c, q, path in zip(slots, ctx, n, paths):
            path = [int(t) for t in path]
            if any(a >= b for a, b in zip(path, path[1:])) or (path and (path[0] < 0 or path[-1] >= q)):
                raise ValueError(f"a path must be ascending indices of the sequence's {q} new tokens, got {path}")
            if int(self.pos_host[s]) != c + q:
                raise ValueError(f"slot {s} holds {int(self.pos_host[s])} tokens, not the {c + q} of the plan's step")
            kept.append(path)
        self._refuse_open(slots, "keep_tokens")
        bs = self.block_size
        # blocks that the moves, or the next appends, write must be the sequence's own
        for s, c, q, path in zip(slots, ctx, n, kept):
            moved = [j for j, t in enumerate(path) if t != j]
            first = c + (moved[0] if moved else len(path))
            self._own_blocks(s, first // bs, -(-(c + q) // bs))
        moves, pos = [], []
        for s, c, path in zip(slots, ctx, kept):
            pos += (s, c + len(path))
            blocks, started = self.block_tables[s]._physical_blocks, 0
            for j, t in enumerate(path):
                if t == j:
                    continue
                a, b = c + t, c + j
                src, dst = blocks[a // bs] * bs + a % bs, blocks[b // bs] * bs + b % bs
                if started and moves[-2] < bs and src == moves[-4] + moves[-2] and dst == moves[-3] + moves[-2]:
                    moves[-2] += 1  # one record, of bs rows at most (blocks with consecutive ids would make it longer)
                else:
                    moves += (src, dst, 1, started)
                    started = 1
        self._move_rows(moves, pos, bs)
        self.pos_host[slots] = pos[1::2]

    def _own_blocks(self, slot: int, first: int, end: int) -> None:
        """Replace blocks first .. end-1 of the slot's table that others hold too by copies of its own."""
        table, alloc = self.block_tables[slot], self.block_allocator
        blocks = table._physical_blocks
        shared = [i for i in range(first, min(end, len(blocks))) if blocks[i] >= 0 and alloc._refcount[blocks[i]] > 1]
        if not shared:
            return
        if not self._tables_move:
            raise ValueError("the rows of a dense cache own their storage")
        old = [blocks[i] for i in shared]
        new = alloc.allocate_many(len(shared))
        self.copy_blocks(old, new)
        for i, b in zip(shared, new):
            blocks[i] = b
        alloc.release_many(old)
        table.epoch += 1

    # ------------------------------------------------------------------ freeing
    def truncate(self, slot: int, length: int) -> None:
        """Drop the tokens of ``slot`` from position ``length`` on and free the blocks that held only those."""
        (slot,) = self._slots([slot], "cache slot")
        have = int(self.pos_host[slot])
        if not 0 <= length <= have:
            raise ValueError(f"length {length} out of range [0, {have}]")
        if self._hole_first[slot] < length < self._hole_end[slot]:
            raise ValueError(f"the blocks around token {length} were freed behind the sequence's window")
        self._refuse_open([slot], "truncate")
        bs, table = self.block_size, self.block_tables[slot]
        if self._tables_move:
            end = -(-length // bs)
            if length % bs:
                self._own_blocks(slot, end - 1, end)  # the next token goes into the last block
            table.shrink(end)
        if length <= self._hole_first[slot]:
            self._clear_hole(slot)
        self._set_pos(slot, length)

    def free_outside_window(self, slot: int, window: int, sinks: int = 0) -> int:
        """Free the blocks of ``slot`` that no later query with this window and sinks sees; returns their number.

        The sequence can then be attended only through plans of windows (and
        sinks) no larger, and not be read by ``get``, ``attention_step`` or
        tree plans.
        """
        (slot,) = self._slots([slot], "cache slot")
        if window <= 0 or sinks < 0:
            raise ValueError("window must be positive and sinks at least 0")
        if not self._tables_move:
            raise ValueError("the rows of a dense cache own their storage")
        self._refuse_open([slot], "free_outside_window")
        bs, table = self.block_size, self.block_tables[slot]
        # what the kernels read is whole groups of 16 keys from these bounds on
        lo = max(0, int(self.pos_host[slot]) - window + 1) // 16 * 16
        first, end = -(-(-(-sinks // 16) * 16) // bs), lo // bs
        had_first, had_end = int(self._hole_first[slot]), int(self._hole_end[slot])
        if had_end and first * bs > had_first:
            first = had_first // bs  # freed before with fewer sinks: the gap stays one run of blocks
        freed = table.free_blocks(first, end) if end > first else 0
        if freed:
            self._hole_first[slot] = first * bs if not had_end else min(first * bs, had_first)
            self._hole_end[slot] = max(end * bs, had_end)
        return freed

    # runs of freed blocks, in keys: [first, end) of each slot (end 0: none)
    def _init_holes(self, batch_size: int) -> None:
        self._hole_first = np.zeros(batch_size, dtype=np.int64)
        self._hole_end = np.zeros(batch_size, dtype=np.int64)

    def _clear_hole(self, slot: int) -> None:
        self._hole_first[slot] = self._hole_end[slot] = 0

    def _holes_of(self, slots) -> bool:
        return bool(self._hole_end[slots].any())

    def _check_window_holes(self, slots, ctx, window: int, sinks: int) -> None:
        end = self._hole_end[slots]
        if not end.any():
            return
        lo = np.maximum(0, ctx - window + 1) // 16 * 16
        kept = np.minimum(-(-sinks // 16) * 16, lo)
        if ((end > 0) & ((lo < end) | (kept > self._hole_first[slots]))).any():
            raise ValueError(f"blocks that a window of {window} with {sinks} sinks sees were freed")

    # ------------------------------------------------------------------ compaction
    def compact(self) -> int:
        """Move the pool's live blocks to its first ids, so that the rest of the pool is free in one piece; returns the
        number of live blocks.

        Tables, reference counts and the prefix index follow.  Blocks already
        there stay.  Later allocations take the lowest free ids first.
        """
        if not self._tables_move:
            raise ValueError("the rows of a dense cache own their storage")
        if self._plan is not None and not self._plan.closed:
            raise RuntimeError("compact: a step is not finished")
        src, dst = self.block_allocator.compact()
        if len(src):
            to = np.arange(self.num_blocks + 1, dtype=np.int64)  # (index -1, a freed entry, stays -1)
            to[-1] = -1
            to[src] = dst
            for table in self.block_tables:
                table.rename(to)
            if self.prefix_cache is not None:
                for key, block in self.prefix_cache.entries.items():
                    self.prefix_cache.entries[key] = int(to[block])
            self.copy_blocks(src, dst)
        return self.block_allocator.allocated_count
