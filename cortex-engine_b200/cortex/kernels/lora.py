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

import ctypes

import torch

from cortex import _lib as L


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
        out: optional output, (..., N); it must not overlap an input.

    Sums are fp32 and the result is rounded once. An id >= n is recorded in the
    device status (IndexError from ``_lib.check_device_status``) and its row gets
    no adapter.
    """
    dev = L.require_cuda(x, w, lora_a, lora_b, adapter_ids, scaling, bias, out,
                         what="lora_linear")
    K = x.shape[-1] if x.dim() > 0 else -1
    if w.dim() != 2 or w.shape[1] != K or K < 1:
        raise ValueError(f"lora_linear: w must be (N, K) with K = {K}, got {tuple(w.shape)}")
    N = w.shape[0]
    if lora_a.dim() != 3 or lora_a.shape[2] != K or lora_a.shape[1] < 1:
        raise ValueError(f"lora_linear: lora_a must be (n, rank, {K}), got {tuple(lora_a.shape)}")
    n, rank = lora_a.shape[0], lora_a.shape[1]
    if lora_b.shape != (n, N, rank):
        raise ValueError(f"lora_linear: lora_b must be {(n, N, rank)}, got {tuple(lora_b.shape)}")
    if not x.dtype == w.dtype == lora_a.dtype == lora_b.dtype:
        raise TypeError(f"lora_linear: x, w, lora_a and lora_b differ in dtype ({x.dtype}, "
                        f"{w.dtype}, {lora_a.dtype}, {lora_b.dtype})")
    if adapter_ids.dtype != torch.int32:
        raise TypeError(f"lora_linear: adapter_ids must be int32, got {adapter_ids.dtype}")
    lead = x.shape[:-1]
    if adapter_ids.shape != lead:
        raise ValueError(f"lora_linear: adapter_ids must be {tuple(lead)}, "
                         f"got {tuple(adapter_ids.shape)}")
    if scaling is not None and (scaling.dtype != torch.float32 or scaling.shape != (n,)):
        raise ValueError(f"lora_linear: scaling must be float32 ({n},)")
    if bias is not None and (bias.dtype != x.dtype or bias.shape != (N,)):
        raise ValueError(f"lora_linear: bias must be {x.dtype} ({N},)")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    if w.stride(1) != 1:
        w = w.contiguous()
    M = x2.shape[0]
    ids = adapter_ids.reshape(-1).contiguous()
    lora_a, lora_b = lora_a.contiguous(), lora_b.contiguous()
    if scaling is not None:
        scaling = scaling.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if out is None:
        y = torch.empty(M, N, dtype=x.dtype, device=dev)
    else:
        if out.shape != (*lead, N) or out.dtype != x.dtype:
            raise ValueError(f"lora_linear: out must be {x.dtype} {(*lead, N)}")
        y = out if out.dim() == 2 else out.view(M, N)
        if N > 1 and y.stride(1) != 1:
            raise ValueError("lora_linear: out rows must be contiguous")
    a = L.LoraArgs(
        L.dtype_code(x.dtype), n, rank, M, K, N, x2.data_ptr(), x2.stride(0), w.data_ptr(),
        w.stride(0), lora_a.data_ptr(), lora_b.data_ptr(), ids.data_ptr(), L.ptr(scaling),
        L.ptr(bias), y.data_ptr(), y.stride(0))
    lib = L.load()
    ref = ctypes.byref(a)
    with L.on_device(dev):
        nb = lib.ck_lora_workspace_bytes(ref)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        rc = lib.ck_lora_linear(ref, None if ws is None else ws.data_ptr(), nb, L.stream_of(dev))
    if rc != L.CK_OK:
        L.check(rc, "ck_lora_linear")
    return out if out is not None else (y if x.dim() == 2 else y.reshape(*lead, N))


__all__ = ["lora_linear"]
