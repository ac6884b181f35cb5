"""Attention of one new token per sequence over a paged K|V pool.

``paged_attention`` reads K and V where ``StreamingKVCache`` keeps them: pool
rows of K | V (kv_proj's output), gathered by page table, never copied into a
packed buffer. It has no counterpart in the reference, whose cache
(cortex/cache/streaming.py:79-236) feeds no attention; semantics follow
``sparse_cross_attention`` (fp32 statistics; a query without any key gives 0).
CUDA tensors only; float32 and bfloat16; forward only, as the rest of the
package. Launches on the current stream of the tensors' device, never
synchronises, and allocates its workspace per call, so calls on several streams
and captured graphs do not share memory.
"""

from __future__ import annotations

import torch

from cortex import _lib as L

_pack = L.PAGED_ATTENTION_ARGS.pack


def check_pages(what: str, pool: torch.Tensor, page_table: torch.Tensor,
                lengths: torch.Tensor) -> tuple[int, int, int, int, int]:
    """Checks shared by the operators over a paged pool: (sequences, pages of a
    table row, pages, page size, row width)."""
    shape, table, count = pool.shape, page_table.shape, lengths.shape
    if len(shape) != 3:
        raise ValueError(f"{what}: pool must be (num_pages, page_size, width), "
                         f"got {tuple(shape)}")
    if page_table.dtype is not torch.int32 or lengths.dtype is not torch.int32:
        raise TypeError(f"{what}: page_table and lengths must be int32, got "
                        f"{page_table.dtype} and {lengths.dtype}")
    if len(table) != 2 or len(count) != 1 or table[0] != count[0]:
        raise ValueError(f"{what}: page_table must be (B, pages) beside lengths (B,), got "
                         f"{tuple(table)} and {tuple(count)}")
    pages, page_size, width = shape
    if page_size < 1 or width < 1:
        raise ValueError(f"{what}: pages must hold at least one row of one element")
    if pool.stride()[2] != 1 and width > 1:
        raise ValueError(f"{what}: pool rows must be contiguous")
    return table[0], table[1], pages, page_size, width


def rows_contiguous(t: torch.Tensor) -> bool:
    """Whether the elements of a row (the last dimension) lie next to each other."""
    return t.is_contiguous() or t.stride()[-1] == 1 or t.shape[-1] <= 1


def paged_attention(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None,
                    weights: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    weights_out: torch.Tensor | None = None):
    """softmax(scale q k^T) v of one query token per sequence.

    Args:
        q: (B, H, Dh) queries, the pool's dtype; Dh <= 256, H <= 4096.
        pool: (num_pages, page_size, 2 * Hkv * Dh) rows of K of every head, then V
            of every head; H must be a multiple of Hkv (grouped queries).
        page_table: (B, pages) int32; position j of sequence b is row
            j % page_size of page ``page_table[b, j // page_size]``. Entries past a
            sequence's last page are not read. Sequences may share pages.
        lengths: (B,) int32 positions per sequence; 0 gives a zero output.
        scale: default Dh ** -0.5.
        weights: optional (B, W) float32, W >= pages * page_size: attention weight
            each position has received so far. The call then returns
            (out, weights_out) with weights_out[b, j] = weights[b, j] + the sum over
            heads of position j's probability (what ``evict_by_weight`` reads).
        out, weights_out: optional outputs, outside the memory that the inputs
            span; only ``weights_out`` may be ``weights`` itself (in place).

    With weights the workspace holds every score, 4 bytes a head and slot of the table,
    whatever the lengths (268 MB at 64 sequences of 32 heads and 32768 slots).

    A page outside the pool (its rows count as absent) or a length outside
    [0, pages * page_size] (clamped) is recorded in the device status
    (``_lib.check_device_status`` raises IndexError), as for event indices.
    """
    d = q.get_device()
    if d < 0 or pool.get_device() != d or page_table.get_device() != d or \
            lengths.get_device() != d or (weights is not None and weights.get_device() != d) or \
            out is not None or weights_out is not None:
        L.require_cuda(q, pool, page_table, lengths, weights, out, weights_out,
                       what="paged_attention")
    if d != L.current_device():
        with torch.cuda.device(d):
            return paged_attention(q, pool, page_table, lengths, scale=scale, weights=weights,
                                   out=out, weights_out=weights_out)
    B, table_width, pages, page_size, width = check_pages("paged_attention", pool, page_table, lengths)
    dtype = q.dtype
    if dtype is not pool.dtype:
        raise TypeError(f"paged_attention: q is {dtype}, the pool {pool.dtype}")
    shape = q.shape
    if len(shape) != 3 or shape[0] != B:
        raise ValueError(f"paged_attention: q must be (B, H, Dh) with B = {B}, got {tuple(shape)}")
    _, H, Dh = shape
    if Dh == 0 or width % (2 * Dh) != 0:
        raise ValueError(f"paged_attention: rows of {width} are not K | V of heads of {Dh}")
    Hkv = width // (2 * Dh)
    if H == 0 or H % Hkv != 0:
        raise ValueError(f"paged_attention: {H} query heads over {Hkv} K|V heads")
    if not rows_contiguous(q):
        q = q.contiguous()
    if not rows_contiguous(page_table):
        page_table = page_table.contiguous()
    if not rows_contiguous(lengths):
        lengths = lengths.contiguous()
    dev = q.device
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(B, H, Dh, dtype=dtype, device=dev)
    elif out.shape != q.shape or out.dtype != dtype or not rows_contiguous(out):
        raise ValueError("paged_attention: out must be like q with contiguous heads")
    else:
        L.check_output("paged_attention", "out", out, q, pool, page_table, lengths, weights,
                       weights_out)
    W = w_in = w_out = w_in_ld = w_out_ld = 0
    if weights is not None:
        if weights.dtype != torch.float32 or weights.dim() != 2 or weights.shape[0] != B or \
                weights.shape[1] < table_width * page_size:
            raise ValueError("paged_attention: weights must be float32 (B, >= pages * page_size)")
        if weights_out is None:
            weights_out = torch.empty_like(weights, memory_format=torch.contiguous_format)
        elif weights_out.shape != weights.shape or weights_out.dtype != torch.float32:
            raise ValueError("paged_attention: weights_out must be like weights")
        elif weights_out is weights:
            L.check_output("paged_attention", "weights_out", weights_out, q, pool, page_table, lengths)
        else:
            L.check_output("paged_attention", "weights_out", weights_out, q, pool, page_table,
                           lengths, weights)
        if not rows_contiguous(weights) or not rows_contiguous(weights_out):
            raise ValueError("paged_attention: weights rows must be contiguous")
        W, w_in, w_out = weights.shape[1], weights.data_ptr(), weights_out.data_ptr()
        w_in_ld, w_out_ld = weights.stride()[0], weights_out.stride()[0]
    elif weights_out is not None:
        raise ValueError("paged_attention: weights_out without weights")
    qb, qh, _ = q.stride()
    pb, pr, _ = pool.stride()
    ob, oh, _ = out.stride()
    if B == 1:  # the stride of a single row says nothing
        qb = 0
    if H == 1:
        qh = 0
    if pages == 1:
        pb = 0
    if page_size == 1:
        pr = 0
    q_ptr, pool_ptr = q.data_ptr(), pool.data_ptr()
    block = _pack(L.dtype_code(dtype), B, H, Hkv, Dh, q_ptr, qb, qh, pool_ptr, pages, pb, pr,
                  page_size, table_width, page_table.data_ptr(), page_table.stride()[0],
                  lengths.data_ptr(), out.data_ptr(), ob, oh, w_in, w_out, w_in_ld, w_out_ld, W,
                  Dh ** -0.5 if scale is None else scale)
    lib = L.load()
    # everything the size depends on, alignment included
    key = ("attention", d, dtype, B, H, Hkv, Dh, page_size, table_width, W, (pb | pr | qb | qh) & 7,
           (q_ptr | pool_ptr) & 15)
    L.launch("ck_paged_attention", lib.ck_paged_attention, lib.ck_paged_attention_workspace_bytes, key,
             block, dev, L.raw_stream(d))
    return out if weights is None else (out, weights_out)


__all__ = ["paged_attention"]
