"""A step's index tensors, built on the GPU from its rows' lengths.

The reference's runner fills them on the host for every step and copies them over
(``ModelRunner.prepare``, miniagentserve/engine/model_runner.py:176-225), its block manager having handed out the pages
(miniagentserve/engine/block_manager.py:43-73). ``plan_step`` does both in one launch from lengths that are already on
the device, with no host synchronisation: a captured decode step can plan itself from the one before.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._tensors import error_word, require_dtype, require_gpu, require_same_device

__all__ = ["StepTables", "step_tables", "plan_step"]


class StepTables(NamedTuple):
    """What ``plan_step`` writes (besides the block tables)."""
    positions: torch.Tensor      # int32 [num_tokens]: each token's position, 0 for padding
    batch_indices: torch.Tensor  # int32 [num_tokens]: its row, -1 for padding
    slot_mapping: torch.Tensor   # int64 [num_tokens]: its cache slot, -1 for padding
    cu_seqlens_q: torch.Tensor   # int32 [rows + 1]: the rows' first tokens
    seq_lens: torch.Tensor       # int32 [rows]: cached + new positions
    free_range: torch.Tensor     # int64 [2]: what is left of the free ring


def step_tables(rows: int, num_tokens: int, device) -> StepTables:
    """Empty tensors for steps of ``rows`` rows and ``num_tokens`` tokens, padding included."""
    def empty(n, dtype):
        return torch.empty(n, dtype=dtype, device=device)

    return StepTables(empty(num_tokens, torch.int32), empty(num_tokens, torch.int32), empty(num_tokens, torch.int64),
                      empty(rows + 1, torch.int32), empty(rows, torch.int32), empty(2, torch.int64))


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, length: int | None = None) -> None:
    require_gpu(t, name)
    require_dtype(t, name, dtype)
    if t.dim() != 1 or not t.is_contiguous() or (length is not None and t.shape[0] != length):
        raise ValueError(f"{name} must be a contiguous 1-D tensor" + ("" if length is None else f" of {length} elements")
                         + f", got shape {tuple(t.shape)}")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    return (a.numel() > 0 and b.numel() > 0 and a.data_ptr() < b.data_ptr() + b.numel() * b.element_size()
            and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())


def _plan(new_lens, cached_lens, block_tables, free_pages, free_range, page_size: int, out, error_flags) -> None:
    rows = new_lens.shape[0] if new_lens.dim() else 0
    _vector(new_lens, "new_lens", torch.int32)
    _vector(cached_lens, "cached_lens", torch.int32, rows)
    _vector(free_pages, "free_pages", torch.int32)
    _vector(free_range, "free_range", torch.int64, 2)
    require_gpu(block_tables, "block_tables")
    require_dtype(block_tables, "block_tables", torch.int32)
    if block_tables.dim() != 2 or block_tables.shape[0] < rows or (block_tables.shape[1] > 1 and
                                                                   block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [rows, max_blocks] int32 with a contiguous last dimension")
    if rows > 1 and block_tables.stride(0) < block_tables.shape[1]:
        raise ValueError("block_tables' rows must not overlap")
    tokens = out[0].shape[0] if out[0].dim() else 0
    for name, t, dtype, n in (("positions", out[0], torch.int32, tokens), ("batch_indices", out[1], torch.int32, tokens),
                              ("slot_mapping", out[2], torch.int64, tokens),
                              ("cu_seqlens_q", out[3], torch.int32, rows + 1), ("seq_lens", out[4], torch.int32, rows),
                              ("free_range", out[5], torch.int64, 2)):
        _vector(t, f"out.{name}", dtype, n)
    device = require_same_device(("new_lens", new_lens), ("cached_lens", cached_lens), ("block_tables", block_tables),
                                 ("free_pages", free_pages), ("free_range", free_range), *zip(StepTables._fields, out))
    if page_size < 1:
        raise ValueError(f"page_size must be positive, got {page_size}")
    # every workgroup reads the lengths and the range while others write
    for name, t in zip(StepTables._fields, out):
        for read_name, read in (("new_lens", new_lens), ("cached_lens", cached_lens), ("free_pages", free_pages),
                                ("free_range", free_range)):
            if _overlap(t, read):
                raise ValueError(f"out.{name} shares memory with {read_name}: a step's outputs need their own")
    err = error_word(error_flags, device)
    with _lib.on_device(device):
        st = _lib.load().mas_plan_step(
            *(t.data_ptr() for t in out), block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1],
            new_lens.data_ptr(), cached_lens.data_ptr(), rows, free_pages.data_ptr(), free_pages.shape[0],
            free_range.data_ptr(), page_size, tokens, err, _lib.stream_handle(device))
    _lib.check(st, "plan_step")


def plan_step(new_lens: torch.Tensor, cached_lens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
              free_range: torch.Tensor, page_size: int, num_tokens: int, *, out: StepTables | None = None,
              error_flags: torch.Tensor | None = None) -> StepTables:
    """The index tensors of a step in which row r, holding ``cached_lens[r]`` positions, gets ``new_lens[r]`` tokens
    (int32 ``[rows]`` each, rows in order; a row may get none).

    Token t of row r sits at position ``p = cached_lens[r] + t - cu_seqlens_q[r]``, slot ``page * page_size + p %
    page_size`` of page ``block_tables[r, p // page_size]``; ``seq_lens`` is cached + new. Blocks that the row does
    not hold yet get pages from the free ring, in row order, written to ``block_tables`` (int32
    ``[rows, max_blocks]``, in place). The ring: ``free_pages`` int32 ``[n]``, entry i of it at ``free_pages[i % n]``;
    ``free_range`` int64 ``[2]``, entries ``free_range[0]`` up to ``free_range[1]`` are free. A host that frees pages
    writes them at the end and raises ``free_range[1]``. ``num_tokens`` (the captured step's token count, say) is at
    least the rows' tokens; the rest are padding: position 0, row -1, slot -1, which the slot form of the stores skips.

    From the first row on whose tokens do not fit ``num_tokens`` or whose pages are not there, rows get no token: their
    ``cu_seqlens_q`` span is empty, ``seq_lens`` is ``cached_lens``, and bit 64 of ``error_flags`` is set. A row with
    a negative length, or one past its table, is passed over alone (bit 2). ``out`` (``step_tables``) is written when
    given; a loop of steps feeds ``out.seq_lens`` and ``out.free_range`` of one step to the next, whose outputs
    must be other tensors.
    """
    if num_tokens < 0:
        raise ValueError(f"num_tokens must not be negative, got {num_tokens}")
    if out is None:
        out = step_tables(new_lens.shape[0], num_tokens, new_lens.device)
    elif len(out) != 6 or out[0].shape[0] != num_tokens:
        raise ValueError(f"out must be StepTables of {num_tokens} tokens")
    if torch.compiler.is_compiling():
        torch.ops.mas.plan_step(new_lens, cached_lens, block_tables, free_pages, free_range, int(page_size), *out,
                                error_flags)
        return StepTables(*out)
    if _lib.direct is not None and (st := _lib.direct.plan_step(new_lens, cached_lens, block_tables, free_pages,
                                                                free_range, page_size, out, error_flags)) is not None:
        if st:
            _lib.check(st, "plan_step")
        return out if type(out) is StepTables else StepTables(*out)
    _plan(new_lens, cached_lens, block_tables, free_pages, free_range, page_size, out, error_flags)
    return StepTables(*out)
