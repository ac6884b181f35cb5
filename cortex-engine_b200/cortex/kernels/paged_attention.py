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

import ctypes

import torch

from cortex import _lib as L


def check_pages(what: str, pool: torch.Tensor, page_table: torch.Tensor,
                lengths: torch.Tensor) -> int:
    """Shape checks shared by the operators over a paged pool; returns B."""
    if pool.dim() != 3:
        raise ValueError(f"{what}: pool must be (num_pages, page_size, width), "
                         f"got {tuple(pool.shape)}")
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError(f"{what}: page_table and lengths must be int32, got "
                        f"{page_table.dtype} and {lengths.dtype}")
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    if page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError(f"{what}: page_table must be (B, pages) beside lengths (B,), got "
                         f"{tuple(page_table.shape)} and {tuple(lengths.shape)}")
    if pool.shape[1] < 1:
        raise ValueError(f"{what}: pages must hold at least one row")
    if pool.stride(2) != 1 and pool.shape[2] > 1:
        raise ValueError(f"{what}: pool rows must be contiguous")
    return B


def paged_attention(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None,
                    weights: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    weights_out: torch.Tensor | None = None):
    """softmax(scale q k^T) v of one query token per sequence.

    Args:
        q: (B, H, Dh) queries, the pool's dtype; Dh <= 256.
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
        out, weights_out: optional outputs; ``weights_out`` may be ``weights``
            itself (in place), otherwise the two must not overlap.

    A page outside the pool (its rows count as absent) or a length outside
    [0, pages * page_size] (clamped) is recorded in the device status
    (``_lib.check_device_status`` raises IndexError), as for event indices.
    """
    dev = L.require_cuda(q, pool, page_table, lengths, weights, out, weights_out,
                         what="paged_attention")
    B = check_pages("paged_attention", pool, page_table, lengths)
    if q.dim() != 3 or q.shape[0] != B:
        raise ValueError(f"paged_attention: q must be (B, H, Dh) with B = {B}, got {tuple(q.shape)}")
    if q.dtype != pool.dtype:
        raise TypeError(f"paged_attention: q is {q.dtype}, the pool {pool.dtype}")
    _, H, Dh = q.shape
    width = pool.shape[2]
    if Dh == 0 or width == 0 or width % (2 * Dh) != 0:
        raise ValueError(f"paged_attention: rows of {width} are not K | V of heads of {Dh}")
    Hkv = width // (2 * Dh)
    if H == 0 or H % Hkv != 0:
        raise ValueError(f"paged_attention: {H} query heads over {Hkv} K|V heads")
    if q.stride(2) != 1:
        q = q.contiguous()
    table_ld = page_table.stride(0)
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        page_table = page_table.contiguous()
        table_ld = page_table.stride(0)
    if B > 1 and lengths.stride(0) != 1:
        lengths = lengths.contiguous()
    if out is None:
        out = torch.empty(B, H, Dh, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("paged_attention: out must be like q with contiguous heads")
    a = L.PagedAttentionArgs(
        L.dtype_code(q.dtype), B, H, Hkv, Dh, q.data_ptr(), q.stride(0), q.stride(1),
        pool.data_ptr(), pool.shape[0], pool.stride(0), pool.stride(1), pool.shape[1],
        page_table.shape[1], page_table.data_ptr(), table_ld, lengths.data_ptr(),
        out.data_ptr(), out.stride(0), out.stride(1))
    a.scale = Dh ** -0.5 if scale is None else scale
    if weights is not None:
        if weights.dtype != torch.float32 or weights.dim() != 2 or weights.shape[0] != B or \
                weights.shape[1] < page_table.shape[1] * pool.shape[1]:
            raise ValueError("paged_attention: weights must be float32 (B, >= pages * page_size)")
        if weights.shape[1] > 1 and weights.stride(1) != 1:
            raise ValueError("paged_attention: weights rows must be contiguous")
        if weights_out is None:
            weights_out = torch.empty(weights.shape, dtype=torch.float32, device=dev)
        elif weights_out.shape != weights.shape or weights_out.dtype != torch.float32 or \
                (weights.shape[1] > 1 and weights_out.stride(1) != 1):
            raise ValueError("paged_attention: weights_out must be like weights")
        a.w_in, a.w_out = weights.data_ptr(), weights_out.data_ptr()
        a.w_in_ld, a.w_out_ld, a.w_width = weights.stride(0), weights_out.stride(0), weights.shape[1]
    elif weights_out is not None:
        raise ValueError("paged_attention: weights_out without weights")
    lib = L.load()
    ref = ctypes.byref(a)
    with L.on_device(dev):
        n = lib.ck_paged_attention_workspace_bytes(ref)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        rc = lib.ck_paged_attention(ref, None if ws is None else ws.data_ptr(), n,
                                    L.stream_of(dev))
    if rc != L.CK_OK:
        L.check(rc, "ck_paged_attention")
    return out if weights is None else (out, weights_out)


__all__ = ["paged_attention"]
