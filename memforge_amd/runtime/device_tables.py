"""A batch's block tables on the device: requests grow and are cut back there,
and the slots of their new tokens are worked out there, with no step of the host.

The host's allocator (``memforge_c.BlockAllocator``) hands out blocks between
steps; a program whose steps follow each other on the device -- a round of
speculation whose number of accepted tokens only the device knows, steps replayed
as HIP graphs -- keeps its tables here instead and reads them back when it wants
to. One launch a call (mf_tables_extend, two with ``rows``; mf_tables_truncate), every sum in it
whole numbers, so the results do not depend on the order of anything."""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from memforge_amd import _native as nat


@dataclass
class SlotMap:
    """Where a call's new tokens go: ``slot_mapping`` and ``positions`` (int64, one per
    row; slot -1 writes nothing), ``cu_seqlens`` (int32, each request's first row),
    ``kv_lens`` (int32, the requests' lengths now: as before where a request was refused)
    and ``refused`` (int32 of one, how many could not grow)."""

    slot_mapping: torch.Tensor
    positions: torch.Tensor
    cu_seqlens: torch.Tensor
    kv_lens: torch.Tensor
    refused: torch.Tensor


@dataclass
class DeviceBlockTables:
    """``tables`` (int32 (requests, max_blocks)), of whose rows the first ``held[s]``
    entries are blocks of request s; ``lens`` its tokens; ``free`` (int32) a stack of
    unused blocks of which the first ``free_count`` (int32 of one) are on it, the last
    on top. All contiguous on one device and changed in place by ``extend`` and
    ``truncate``, on the current stream and in their order on it."""

    tables: torch.Tensor
    lens: torch.Tensor
    held: torch.Tensor
    free: torch.Tensor
    free_count: torch.Tensor
    block_size: int

    @classmethod
    def allocate(cls, num_requests: int, max_blocks: int, num_blocks: int, block_size: int,
                 device) -> "DeviceBlockTables":
        """Empty requests over blocks 0 .. ``num_blocks`` - 1, block 0 to be taken first."""
        def zeros(*shape):
            return torch.zeros(shape, dtype=torch.int32, device=device)

        return cls(zeros(num_requests, max_blocks), zeros(num_requests), zeros(num_requests),
                   torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device),
                   torch.full((1,), num_blocks, dtype=torch.int32, device=device), block_size)

    def _state(self, name: str, want: torch.Tensor):
        """The tensors' checks, and the C arguments that both entry points begin with."""
        tables = self.tables
        nat.require_device(tables, want)
        if tables.dim() != 2:
            raise ValueError(f"tables must be (requests, max_blocks), got {tuple(tables.shape)}")
        (n, width), dev = tables.shape, tables.device
        shape = (n,)
        nat.check_index("tables", tables, torch.int32, dev)
        nat.check_index("lens", self.lens, torch.int32, dev, shape)
        nat.check_index("held", self.held, torch.int32, dev, shape)
        nat.check_index("free", self.free, torch.int32, dev)
        nat.check_index("free_count", self.free_count, torch.int32, dev, (1,))
        nat.check_index(name, want, torch.int32, dev, shape)
        return dev, n, (tables.data_ptr(), width, width, self.lens.data_ptr(), self.held.data_ptr(),
                                  self.free.data_ptr(), self.free.numel(), self.free_count.data_ptr(), want.data_ptr(), n,
                                  self.block_size)

    def extend(self, new_tokens: torch.Tensor, max_rows: int, rows: Optional[torch.Tensor] = None) -> SlotMap:
        """Grow request s by ``new_tokens[s]`` (int32, on the device). In request order each
        takes the blocks it lacks from the stack; one whose table row, whose rows within
        ``max_rows`` or whose blocks do not suffice is refused and keeps what it has, its
        rows get slot -1, and so does every later one that lacks blocks when it was the
        blocks. The new tokens are packed: row ``cu_seqlens[s] + i`` is token i of request
        s, rows past the last get slot -1. With ``rows`` (int32 (requests, most)) token i of
        request s is row ``rows[s, i]`` of ``max_rows`` instead, negative entries none, and
        no row named twice: the accepted path of a tree's rows, whose keys and values ``_native.kv_write`` then
        puts into the pool as they lie."""
        dev, n, state = self._state("new_tokens", new_tokens)
        if max_rows < 0:
            raise ValueError(f"max_rows must not be negative, got {max_rows}")
        if rows is not None:
            nat.check_index("rows", rows, torch.int32, dev)
            if rows.dim() != 2 or rows.shape[0] != n:
                raise ValueError(f"rows must be ({n}, most new tokens), got {tuple(rows.shape)}")
            # (an empty tensor has no address, and no address means packed rows; nothing is read of no columns)
            at, width = rows.data_ptr() or self.lens.data_ptr(), rows.shape[1]
        else:
            at, width = None, 0
        slots = torch.empty(max_rows, dtype=torch.int64, device=dev)
        positions = torch.empty(max_rows, dtype=torch.int64, device=dev)
        cu = torch.empty(n + 1, dtype=torch.int32, device=dev)
        lens = torch.empty(n, dtype=torch.int32, device=dev)
        refused = torch.empty(1, dtype=torch.int32, device=dev)
        nat._launch(dev, "mf_tables_extend", nat.lib().mf_tables_extend, *state, max_rows, at, width, width,
                    slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), lens.data_ptr(), refused.data_ptr(),
                    nat._WORKSPACE.counters(1, dev).data_ptr())
        return SlotMap(slots, positions, cu, lens, refused)

    def truncate(self, lengths: torch.Tensor) -> None:
        """Cut request s back to ``min(lens[s], lengths[s])`` tokens (int32, on the device;
        negative as 0) and give back the blocks that it then does not need: all of a
        finished request's with 0. A block belongs to one request; one that stood in two tables
        would be given back twice. Their table entries become 0. After ``extend`` and
        ``truncate`` to the lengths before, tables and stack are as they were."""
        dev, n, state = self._state("lengths", lengths)
        nat._launch(dev, "mf_tables_truncate", nat.lib().mf_tables_truncate, *state,
                    nat._WORKSPACE.counters(1, dev).data_ptr())
