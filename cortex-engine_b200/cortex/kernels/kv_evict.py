"""Eviction from a paged row pool by accumulated attention weight.

``paged_attention`` adds up how much attention each position of a sequence has
received; ``evict_by_weight`` keeps every sequence inside a budget of rows by
dropping those that received least, the newest excepted. It has no counterpart
in the reference, whose cache drops whole entries only
(cortex/cache/streaming.py:186-195). CUDA tensors only. Launches on the current
stream of the tensors' device, never synchronises, and allocates its workspace
per call.
"""

from __future__ import annotations

import torch

from cortex import _lib as L
from cortex.kernels.paged_attention import check_pages, rows_contiguous

_pack = L.EVICT_ARGS.pack


def _table(what: str, t: torch.Tensor, dtype: torch.dtype, B: int, width: int) -> tuple[int, int]:
    """(row stride, columns) of a (B, >= width) table."""
    if t.dtype is not dtype:
        raise TypeError(f"evict_by_weight: {what} must be {dtype}, got {t.dtype}")
    shape = t.shape
    if len(shape) != 2 or shape[0] != B or shape[1] < width:
        raise ValueError(f"evict_by_weight: {what} must be ({B}, >= {width}), got {tuple(shape)}")
    ld, step = t.stride()
    if step != 1 and shape[1] > 1:
        raise ValueError(f"evict_by_weight: {what} rows must be contiguous")
    return ld, shape[1]


def evict_by_weight(pool: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    weights: torch.Tensor, positions: torch.Tensor, *, budget: int,
                    recent: int = 0, out: tuple | None = None):
    """Drop the rows with the least weight of every sequence over its budget.

    Args:
        pool: (num_pages, page_size, width) rows, changed in place (float32 or
            bfloat16).
        page_table: (B, pages) int32; slot j of sequence b is row j % page_size of
            page ``page_table[b, j // page_size]``. A sequence's pages must be its
            own: with a page in two places of the table, the rows in it are
            unspecified afterwards.
        lengths: (B,) int32 rows per sequence.
        weights: (B, W) float32, W >= pages * page_size: the weight of each slot.
        positions: (B, W) int32: the position of the row in each slot. Rows move, so
            slots are not positions once a sequence has been through an eviction.
        budget: rows a sequence may keep (>= 1).
        recent: rows whose position is among the newest ``recent`` (position >
            newest - recent) are kept before all others; 0 <= recent <= budget.
        out: optional (lengths, weights, positions) to write to, each of which may be
            the input itself (in place) and is apart from all other inputs; slots
            behind the new lengths are left as they were. Without it new tensors:
            weights and positions (B, budget), 0 and -1 behind the new lengths.

    Of a sequence of n > budget rows the ``budget`` best stay: the newest, then by
    weight, largest first (NaN last), equal ones by lower slot. The kept rows in
    slots from ``budget`` on move into the freed slots before it, both in
    ascending order, with their weight and position. Returns (lengths, weights,
    positions); pages behind ``budget`` are free afterwards.

    A length outside [0, pages * page_size] (its sequence is left alone) or a page
    outside the pool (its rows are not copied) is recorded in the device status.
    """
    d = pool.get_device()
    if d < 0 or page_table.get_device() != d or lengths.get_device() != d or \
            weights.get_device() != d or positions.get_device() != d or out is not None:
        L.require_cuda(pool, page_table, lengths, weights, positions, *(out or ()),
                       what="evict_by_weight")
    if d != L.current_device():
        with torch.cuda.device(d):
            return evict_by_weight(pool, page_table, lengths, weights, positions, budget=budget,
                                   recent=recent, out=out)
    B, table_width, pages, page_size, width = check_pages("evict_by_weight", pool, page_table, lengths)
    if pool.dtype is not torch.bfloat16 and pool.dtype is not torch.float32:
        raise NotImplementedError(f"evict_by_weight: rows of {pool.dtype}")
    if not 1 <= budget < 2 ** 31 or not 0 <= recent <= budget:
        raise ValueError(f"evict_by_weight: needs 1 <= budget and 0 <= recent <= budget, "
                         f"got {budget} and {recent}")
    cap = table_width * page_size
    w_ld, w_cols = _table("weights", weights, torch.float32, B, cap)
    pos_ld, pos_cols = _table("positions", positions, torch.int32, B, cap)
    dev = pool.device
    fill = out is None
    if fill:
        new_len = torch.empty_like(lengths, memory_format=torch.contiguous_format)
        new_w = torch.empty(B, budget, dtype=torch.float32, device=dev)
        new_pos = torch.empty(B, budget, dtype=torch.int32, device=dev)
        new_w_ld = new_pos_ld = new_cols = budget
        if not rows_contiguous(lengths):
            lengths = lengths.contiguous()
    else:
        new_len, new_w, new_pos = out
        if new_len.dtype != torch.int32 or new_len.shape != lengths.shape:
            raise ValueError("evict_by_weight: out lengths must be like lengths")
        if not rows_contiguous(new_len) or not rows_contiguous(lengths):
            raise ValueError("evict_by_weight: lengths must be contiguous")
        new_w_ld, new_cols = _table("out weights", new_w, torch.float32, B, min(budget, cap))
        new_pos_ld, n = _table("out positions", new_pos, torch.int32, B, min(budget, cap))
        new_cols = min(new_cols, n)
        for name, given, own in (("out lengths", new_len, lengths), ("out weights", new_w, weights),
                                 ("out positions", new_pos, positions)):
            if given is not own:
                L.check_output("evict_by_weight", name, given, pool, page_table, lengths, weights,
                               positions, *(t for t in out if t is not given))
            elif not given.is_contiguous():
                L.check_output("evict_by_weight", name, given)
    if not rows_contiguous(page_table):
        page_table = page_table.contiguous()
    page_ld, row_ld, _ = pool.stride()
    if row_ld < width or page_ld < page_size * row_ld:
        L.check_output("evict_by_weight", "pool", pool)
    block = _pack(pool.element_size(), B, pool.data_ptr(), pages, page_ld, row_ld, page_size, width,
                  page_table.data_ptr(), page_table.stride()[0], table_width, budget, recent, fill,
                  lengths.data_ptr(), new_len.data_ptr(), weights.data_ptr(), new_w.data_ptr(),
                  positions.data_ptr(), new_pos.data_ptr(), w_ld, new_w_ld, pos_ld, new_pos_ld,
                  min(w_cols, pos_cols, 2 ** 31 - 1), min(new_cols, 2 ** 31 - 1))
    lib = L.load()
    L.launch("ck_evict_by_weight", lib.ck_evict_by_weight, lib.ck_evict_workspace_bytes,
             ("evict", d, B, cap, budget, width, pool.dtype), block, dev, L.raw_stream(d))
    return new_len, new_w, new_pos


__all__ = ["evict_by_weight"]
