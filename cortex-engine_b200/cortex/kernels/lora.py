"""A projection shared by many requests, beside each request's low-rank adapter.

Sessions served from one set of weights differ by small adapters; ``lora_linear``
runs a batch whose rows belong to different sessions as one call:
``y[m] = W x[m] + scaling[i] B_i (A_i x[m]) + bias`` with ``i = adapter_ids[m]``.
No reference counterpart; the shared part is ``nn.Linear``'s
(cortex/models/perceiver.py:44-49). CUDA tensors only; float32 and bfloat16;
forward only. Launches on the current stream of the tensors' device, never
synchronises, and allocates its workspace per call.
"""

from __future__ import annotations

import torch

from cortex import _lib as L
from cortex.kernels.paged_attention import rows_contiguous

_pack = L.LORA_ARGS.pack


def lora_linear(x: torch.Tensor, w: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                adapter_ids: torch.Tensor, *, scaling: torch.Tensor | None = None,
                bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ w.T (+ bias)`` plus every row's own adapter.

    Args:
        x: (..., K) rows.
        w: (N, K) shared weight, x's dtype (``nn.Linear.weight``).
        lora_a, lora_b: (n, rank, K) and (n, N, rank) adapters, x's dtype,
            rank <= 256.
        adapter_ids: int32, one per row of x (its leading shape); negative for a
            row without an adapter.
        scaling: optional (n,) float32 factor of each adapter's part.
        bias: optional (N,), x's dtype.
        out: optional output, (..., N), outside the memory that the inputs span.

    Sums are fp32 and the result is rounded once. bf16 calls of many rows (from 33 on,
    by rows, rank and N) carry h = scaling[i] A_i x as the sum of two bf16 numbers to the
    product with B_i, an error of at most 2^-15 |B_i||h|. An id >= n is recorded in the
    device status (IndexError from ``_lib.check_device_status``) and its row gets
    no adapter.
    """
    d = x.get_device()
    if d < 0 or w.get_device() != d or lora_a.get_device() != d or lora_b.get_device() != d or \
            adapter_ids.get_device() != d or \
            (scaling is not None and scaling.get_device() != d) or \
            (bias is not None and bias.get_device() != d) or out is not None:
        L.require_cuda(x, w, lora_a, lora_b, adapter_ids, scaling, bias, out, what="lora_linear")
    if d != L.current_device():
        with torch.cuda.device(d):
            return lora_linear(x, w, lora_a, lora_b, adapter_ids, scaling=scaling, bias=bias, out=out)
    dtype, xs, ws, a_shape = x.dtype, x.shape, w.shape, lora_a.shape
    K = xs[-1] if len(xs) > 0 else -1
    lead = xs[:-1]
    if len(ws) != 2 or ws[1] != K or K < 1:
        raise ValueError(f"lora_linear: w must be (N, K) with K = {K}, got {tuple(ws)}")
    N = ws[0]
    if len(a_shape) != 3 or a_shape[2] != K or a_shape[1] < 1:
        raise ValueError(f"lora_linear: lora_a must be (n, rank, {K}), got {tuple(a_shape)}")
    n, rank, _ = a_shape
    if lora_b.shape != (n, N, rank):
        raise ValueError(f"lora_linear: lora_b must be {(n, N, rank)}, got {tuple(lora_b.shape)}")
    if dtype is not w.dtype or dtype is not lora_a.dtype or dtype is not lora_b.dtype:
        raise TypeError(f"lora_linear: x, w, lora_a and lora_b differ in dtype ({dtype}, "
                        f"{w.dtype}, {lora_a.dtype}, {lora_b.dtype})")
    if adapter_ids.dtype is not torch.int32:
        raise TypeError(f"lora_linear: adapter_ids must be int32, got {adapter_ids.dtype}")
    if adapter_ids.shape != lead:
        raise ValueError(f"lora_linear: adapter_ids must be {tuple(lead)}, "
                         f"got {tuple(adapter_ids.shape)}")
    ids, x2 = adapter_ids, x
    if len(lead) != 1:
        ids, x2 = ids.reshape(-1), x.reshape(-1, K)
    M, ldx, ldw = x2.shape[0], x2.stride()[0], w.stride()[0]
    if not rows_contiguous(x2) or (ldx < K and M > 1):  # (rows that share memory: expanded)
        x2, ldx = x2.contiguous(), K
    if not rows_contiguous(w) or (ldw < K and N > 1):
        w, ldw = w.contiguous(), K
    if M <= 1:
        ldx = K  # the stride of a single row says nothing
    if N <= 1:
        ldw = K
    if not rows_contiguous(ids):
        ids = ids.contiguous()
    if not lora_a.is_contiguous():
        lora_a = lora_a.contiguous()
    if not lora_b.is_contiguous():
        lora_b = lora_b.contiguous()
    scaling_ptr = bias_ptr = 0
    if scaling is not None:
        if scaling.dtype is not torch.float32 or scaling.shape != (n,):
            raise ValueError(f"lora_linear: scaling must be float32 ({n},)")
        if not scaling.is_contiguous():
            scaling = scaling.contiguous()
        scaling_ptr = scaling.data_ptr()
    if bias is not None:
        if bias.dtype != dtype or bias.shape != (N,):
            raise ValueError(f"lora_linear: bias must be {dtype} ({N},)")
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    dev, ldy = x.device, N
    if out is None:
        y = torch.empty(M, N, dtype=dtype, device=dev)
    else:
        if out.shape != (*lead, N) or out.dtype != dtype:
            raise ValueError(f"lora_linear: out must be {dtype} {(*lead, N)}")
        y = out if out.dim() == 2 else out.view(M, N)
        if not rows_contiguous(y):
            raise ValueError("lora_linear: out rows must be contiguous")
        L.check_output("lora_linear", "out", y, x, w, lora_a, lora_b, adapter_ids, scaling, bias)
        if M > 1:
            ldy = y.stride()[0]
    x_ptr, w_ptr, y_ptr = x2.data_ptr(), w.data_ptr(), y.data_ptr()
    a_ptr, b_ptr = lora_a.data_ptr(), lora_b.data_ptr()
    block = _pack(L.dtype_code(dtype), n, rank, M, K, N, x_ptr, ldx, w_ptr, ldw, a_ptr, b_ptr,
                  ids.data_ptr(), scaling_ptr, bias_ptr, y_ptr, ldy)
    lib = L.load()
    # everything the size depends on, alignment included
    key = ("lora", d, dtype, M, K, N, rank, n, (ldx | ldw) & 7, ldy & 7,
           (x_ptr | w_ptr | a_ptr | b_ptr) & 15, y_ptr & 15)
    L.launch("ck_lora_linear", lib.ck_lora_linear, lib.ck_lora_workspace_bytes, key, block, dev,
             L.raw_stream(d))
    if out is not None:
        return out
    return y if len(lead) == 1 else y.reshape(*lead, N)


__all__ = ["lora_linear"]
