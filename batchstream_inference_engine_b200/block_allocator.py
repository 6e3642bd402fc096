"""Block allocator with device-resident block tables.

``BlockAllocator`` keeps the reference's semantics exactly
(src/server/block_allocator.py:5-33): a LIFO free list that starts as
``range(num_blocks)``, per-sequence tables that grow to ceil(tokens / block_size)
blocks, all-or-nothing allocation raising ``OutOfBlocks`` (a RuntimeError), and
``free`` returning a table's blocks in table order.  On top of that it mirrors
every table into an int32 tensor ``[max_seqs, max_blocks_per_seq]`` on the GPU
(one row per live sequence), so kernels read block tables and context lengths
from device memory; only new table entries cross PCIe, batched into one copy per
``sync_device()``.

Three operations go beyond the reference: ``fork`` starts a sequence from the
cached tokens of another (whole blocks are shared and reference-counted, the last
partial one is copied), ``trim`` frees the blocks that a sliding window has left
behind, and ``compact`` renumbers the blocks in use to the lowest ids.  ``fork``
and ``compact`` return the (source, destination) block copies that the caller owes
the pool (``ops.copy_blocks``) before the next step.
"""

from __future__ import annotations

import torch


EMPTY_BLOCK = -1  # table entry of a trimmed block


class OutOfBlocks(RuntimeError):
    """The pool (or the device table) cannot hold a sequence's next blocks;
    nothing was taken.  A RuntimeError, as the reference raises it."""


class BlockAllocator:
    def __init__(self, num_blocks: int, block_size: int, max_seqs: int = 0,
                 max_blocks_per_seq: int = 0, device: torch.device | str | None = None):
        self._block_size = block_size
        self._free = list(range(num_blocks))
        self._tables: dict[int, list[int]] = {}
        self._refs: dict[int, int] = {}  # tables that hold a block, where more than one does
        self._trimmed: dict[int, int] = {}  # entries below this were given up by trim,
        self._kept: dict[int, int] = {}  # down to this one (ahead of it are the sinks)
        self.num_blocks = num_blocks
        # Device mirror (optional).
        self._device = torch.device(device) if device is not None else None
        self.max_seqs = max_seqs
        self.max_blocks_per_seq = max_blocks_per_seq
        self._rows: dict[int, int] = {}
        self._free_rows = list(range(max_seqs - 1, -1, -1))
        self._synced: dict[int, int] = {}  # entries of each table already on the device
        self.device_tables: torch.Tensor | None = None
        if self._device is not None:
            if max_seqs <= 0 or max_blocks_per_seq <= 0:
                raise ValueError("a device mirror needs max_seqs and max_blocks_per_seq")
            self.device_tables = torch.full((max_seqs, max_blocks_per_seq), -1,
                                            dtype=torch.int32, device=self._device)

    # ---------------------------------------------------------------- reference API

    @property
    def free_blocks(self) -> int:
        return len(self._free)

    @property
    def block_size(self) -> int:
        return self._block_size

    def allocate(self, seq_id: int, total_tokens: int) -> None:
        """Extends seq_id's table (creating it if new) to ceil(total_tokens /
        block_size) blocks, taking each from the end of the free list; takes
        none and raises OutOfBlocks when the free list is too short."""
        table = self._tables.get(seq_id, [])
        missing = -(-total_tokens // self._block_size) - len(table)
        if missing > len(self._free):
            raise OutOfBlocks(f"sequence {seq_id} needs {missing} more blocks but only "
                              f"{len(self._free)} are free")
        needed = missing
        if self.device_tables is not None:
            if len(table) + max(needed, 0) > self.max_blocks_per_seq:
                raise OutOfBlocks(
                    f"sequence needs {len(table) + needed} blocks, the device table row holds "
                    f"{self.max_blocks_per_seq}")
            if seq_id not in self._rows:
                if not self._free_rows:
                    raise OutOfBlocks(f"all {self.max_seqs} device table rows are in use")
                self._rows[seq_id] = self._free_rows.pop()
                self._synced[seq_id] = 0
        for _ in range(needed):
            table.append(self._free.pop())
        self._tables[seq_id] = table

    def block_table(self, seq_id: int) -> list[int]:
        return self._tables[seq_id]

    def locate(self, seq_id: int, position: int) -> tuple[int, int]:
        block_index, offset = divmod(position, self._block_size)
        return self._tables[seq_id][block_index], offset

    def free(self, seq_id: int) -> None:
        for block in self._tables.pop(seq_id):
            self._release(block)
        self._trimmed.pop(seq_id, None)
        self._kept.pop(seq_id, None)
        row = self._rows.pop(seq_id, None)
        if row is not None:
            self._synced.pop(seq_id, None)
            self._free_rows.append(row)

    # ---------------------------------------------------------------- forks, windows, compaction

    def _release(self, block: int) -> int:
        """Drops one table's hold on a block; 1 when that freed it."""
        if block == EMPTY_BLOCK:
            return 0
        refs = self._refs.get(block, 1)
        if refs > 1:
            if refs == 2:
                del self._refs[block]
            else:
                self._refs[block] = refs - 1
            return 0
        self._free.append(block)
        return 1

    def fork(self, seq_id: int, child_id: int, tokens: int) -> list[tuple[int, int]]:
        """Starts child_id with the first `tokens` tokens of seq_id: its whole
        blocks are shared (neither sequence writes them again), and a last
        partial block is taken from the free list for the child.  Returns that
        block's (source, destination) copy, if any.  Takes nothing and raises
        OutOfBlocks when no block or device table row is free.

        A trimmed sequence is forked where its window ends, at its cached tokens:
        earlier ones would look back on blocks that are gone.  A fork that ends among
        those is refused."""
        table = self._tables[seq_id]
        if child_id in self._tables:
            raise ValueError(f"sequence {child_id} already exists")
        whole, tail = divmod(tokens, self._block_size)
        if tokens < 0 or whole + (tail > 0) > len(table):
            raise ValueError(f"sequence {seq_id} has no blocks for {tokens} tokens")
        if (tokens < self._trimmed.get(seq_id, 0) * self._block_size
                and EMPTY_BLOCK in table[: whole + (tail > 0)]):
            raise ValueError(f"sequence {seq_id} has given up blocks that {tokens} tokens look "
                             "back on")
        copied = tail > 0
        if copied and not self._free:
            raise OutOfBlocks(f"forking sequence {seq_id} needs a block but none is free")
        if self.device_tables is not None:
            if not self._free_rows:
                raise OutOfBlocks(f"all {self.max_seqs} device table rows are in use")
            self._rows[child_id] = self._free_rows.pop()
            self._synced[child_id] = 0
        child = table[:whole]
        for block in child:
            if block != EMPTY_BLOCK:
                self._refs[block] = self._refs.get(block, 1) + 1
        if seq_id in self._trimmed:
            self._trimmed[child_id] = min(self._trimmed[seq_id], whole)
            self._kept[child_id] = self._kept[seq_id]
        pairs = []
        if copied:
            child.append(self._free.pop())
            pairs.append((table[whole], child[-1]))
        self._tables[child_id] = child
        return pairs

    def trim(self, seq_id: int, first_token: int, keep_first: int = 0) -> int:
        """Gives up the blocks of seq_id whose tokens all lie before first_token
        and at or past keep_first (the tokens between the sinks and the window);
        their table entries become EMPTY_BLOCK.  Returns how many blocks that
        freed (a block that a fork still holds stays in use)."""
        table = self._tables[seq_id]
        end = min(first_token // self._block_size, len(table))
        keep = -(-max(keep_first, 0) // self._block_size)
        if keep >= end:
            return 0
        low, high = self._kept.get(seq_id, keep), self._trimmed.get(seq_id, keep)  # given up
        freed = 0
        for i in (*range(keep, min(low, end)), *range(max(keep, high), end)):
            freed += self._release(table[i])
            table[i] = EMPTY_BLOCK
        if keep > high:
            low = keep
        elif end >= low:
            low = min(low, keep)
        self._kept[seq_id], self._trimmed[seq_id] = low, max(high, end)
        return freed

    def moves(self) -> list[tuple[int, int]]:
        """The (source, destination) copies that ``compact`` would return."""
        used = sorted({b for table in self._tables.values() for b in table} - {EMPTY_BLOCK})
        count = len(used)
        return list(zip((b for b in used if b >= count),
                        sorted(b for b in self._free if b < count)))

    def compact(self) -> list[tuple[int, int]]:
        """Renumbers the blocks in use to ids below their count: each block above
        takes the place of a free one below, the lowest first.  Returns the
        (source, destination) copies; no block is both."""
        moved = dict(self.moves())
        count = self.num_blocks - len(self._free)
        for seq_id, table in self._tables.items():
            if any(b in moved for b in table):
                self._tables[seq_id][:] = [moved.get(b, b) for b in table]
                if seq_id in self._synced:
                    self._synced[seq_id] = 0
        self._refs = {moved.get(b, b): n for b, n in self._refs.items()}
        if moved:
            self._free = list(range(count, self.num_blocks))
        return list(moved.items())

    # ---------------------------------------------------------------- device mirror

    def row(self, seq_id: int) -> int:
        """Row of the sequence in ``device_tables``."""
        return self._rows[seq_id]

    def sync_device(self) -> int:
        """Copy table entries added since the last sync to the device; returns how many.

        Stale entries of freed rows are left in place: kernels only read
        ceil(len / block_size) entries of a row, all of which a live sequence owns.
        """
        if self.device_tables is None:
            return 0
        index, value = [], []
        width = self.max_blocks_per_seq
        for seq_id, row in self._rows.items():
            table = self._tables[seq_id]
            done = self._synced[seq_id]
            if done < len(table):
                base = row * width
                index.extend(range(base + done, base + len(table)))
                value.extend(table[done:])
                self._synced[seq_id] = len(table)
        if index:
            packed = torch.tensor([index, value], dtype=torch.int64)
            if self._device.type == "cuda":
                packed = packed.pin_memory()
            packed = packed.to(self._device, non_blocking=True)
            flat = self.device_tables.view(-1)
            flat.index_copy_(0, packed[0], packed[1].to(torch.int32))
        return len(index)
