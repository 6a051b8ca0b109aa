"""A serving step's tables, built on the GPU: block table, slot map, positions, lengths.

`reshape_and_cache` takes the slots of a step's tokens, the decode and the prefill
a block table and lengths. `build_step_tables` makes them from what a step adds
to each row, with no copy of a length to the host, so a captured step can be
replayed while sequences grow, finish and enter. The launch goes through
`pa_step_tables` (include/pagedattn.h); there is no CPU path.
"""

from __future__ import annotations

import dataclasses

import torch

from . import _abi
from .hip_decode import _launch


@dataclasses.dataclass
class StepTables:
    """What a step hands to the cache writer and the attention."""

    query_start_loc: torch.Tensor  # [batch + 1] int32: row b's tokens are packed from [b] to [b + 1]
    slot_mapping: torch.Tensor     # [max_tokens] int64, -1 past the last token
    positions: torch.Tensor        # [max_tokens] int64, 0 past the last token
    seq_lens: torch.Tensor         # [batch] int32: tokens after the step
    free_count: torch.Tensor       # [1] int32: pages left on the stack


# Geometries (shapes, strides, types, devices) that have been checked; nothing of a
# tensor's identity or address.
_CHECKED: set[tuple] = set()
_CHECKED_MAX = 512


def _check(block_table, vectors, max_tokens) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError(f"block_table must be int32 [B, max_blocks], got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    dev = block_table.device
    b, blocks = block_table.shape
    if blocks < 1 or (blocks > 1 and b and block_table.stride(1) != 1):
        raise ValueError("block_table rows must be contiguous and not empty")
    if max_tokens < 0:
        raise ValueError(f"max_tokens {max_tokens} < 0")
    sizes = {"seq_lens": b, "new_lens": b, "finished": b, "free_pages": None, "free_count": 1, "seq_lens_out": b,
             "free_count_out": 1, "query_start_loc": b + 1, "slot_mapping": max_tokens, "positions": max_tokens}
    types = {"finished": torch.bool, "slot_mapping": torch.int64, "positions": torch.int64}
    for (name, n), t in zip(sizes.items(), vectors):
        if t is None:
            continue
        dtype = types.get(name, torch.int32)
        if t.dtype != dtype or t.dim() != 1 or (n is not None and t.shape[0] != n):
            raise ValueError(f"{name} must be {dtype} [{'n' if n is None else n}], got {t.dtype} {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, block_table on {dev}")
    if dev.type != "cuda":
        raise ValueError(f"block_table is on {dev}: the tables are built on the GPU")


def build_step_tables(
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    new_lens: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    block_size: int,
    max_tokens: int,
    finished: torch.Tensor | None = None,
    seq_lens_out: torch.Tensor | None = None,
    free_count_out: torch.Tensor | None = None,
    query_start_loc: torch.Tensor | None = None,
    slot_mapping: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
) -> StepTables:
    """Grow every row b by new_lens[b] tokens; asynchronous on the current stream.

    block_table [B, max_blocks] int32 is changed in place: the row's new pages
    are popped from the top of the stack free_pages[0 .. free_count[0] - 1]
    (int32), rows in order. `finished` [B] bool: those rows first push their
    pages (free_pages must have room for the pool) and start empty, so a new
    sequence can enter a row in the step that ends the old one. Lengths and the
    count are written to seq_lens_out and free_count_out, by default in place.
    The other outputs are allocated unless given (a captured step gives them).

    A row that does not fit gets nothing and keeps its length: one past its
    table row (max_blocks * block_size tokens), and, in row order, those from
    the first on that max_tokens (for rows that add tokens) or the stack (for
    rows that need a page) does not hold. Its query_start_loc range is then
    empty although new_lens[b] > 0. Values <= 0 in new_lens add nothing. A row
    owns its pages: pages shared between rows must not be returned through
    `finished`.
    """
    max_tokens, block_size = int(max_tokens), int(block_size)
    # (outputs that are not given need no check)
    vectors = (seq_lens, new_lens, finished, free_pages, free_count, seq_lens_out, free_count_out, query_start_loc,
               slot_mapping, positions)
    key = (block_table.shape, block_table.stride(), block_table.dtype, block_table.get_device(), max_tokens,
           *[None if t is None else (t.shape, t.dtype, t.get_device(), t.is_contiguous()) for t in vectors])
    if key not in _CHECKED:
        _check(block_table, vectors, max_tokens)
        if len(_CHECKED) >= _CHECKED_MAX:
            _CHECKED.clear()
        _CHECKED.add(key)
    b, blocks = block_table.shape
    if seq_lens_out is None:
        seq_lens_out = seq_lens
    if free_count_out is None:
        free_count_out = free_count
    dev = block_table.device
    if query_start_loc is None:
        query_start_loc = torch.empty((b + 1,), dtype=torch.int32, device=dev)
    if slot_mapping is None and positions is None:
        slot_mapping, positions = torch.empty((2, max_tokens), dtype=torch.int64, device=dev).unbind(0)
    elif slot_mapping is None:
        slot_mapping = torch.empty((max_tokens,), dtype=torch.int64, device=dev)
    elif positions is None:
        positions = torch.empty((max_tokens,), dtype=torch.int64, device=dev)
    args = _abi.PaStepTablesArgs(
        block_table.data_ptr(), seq_lens.data_ptr(), new_lens.data_ptr(),
        None if finished is None else finished.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
        seq_lens_out.data_ptr(), free_count_out.data_ptr(), query_start_loc.data_ptr(), slot_mapping.data_ptr(),
        positions.data_ptr(), b, blocks, block_size, free_pages.shape[0], max_tokens,
        block_table.stride(0) if b > 1 else blocks)
    rc = _launch(block_table, _abi.load().pa_step_tables, args)
    if rc:
        _abi.check(rc, "pa_step_tables")
    return StepTables(query_start_loc, slot_mapping, positions, seq_lens_out, free_count_out)


__all__ = ["StepTables", "build_step_tables"]
