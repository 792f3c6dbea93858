"""Clipping gradients by their global norm, on the device.

The step between ``loss.backward()`` through the head and the optimizer: the same call and
result as ``torch.nn.utils.clip_grad_norm_`` with the 2-norm (TRL's trainer, which drives
the reference's patched forward, calls that with ``max_grad_norm`` and logs the norm), in two
launches for up to 1024 gradients of any mix of fp16, bf16 and fp32.
"""
from __future__ import annotations

from array import array

import torch

from . import _lib

_GRAD_DTYPES = {torch.float16: _lib.LMCE_DTYPE_F16, torch.bfloat16: _lib.LMCE_DTYPE_BF16,
                torch.float32: _lib.LMCE_DTYPE_F32}


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place so that their global 2-norm is at most
    ``max_norm``; returns the norm they had (fp32 scalar on their device).

    ``parameters`` is a tensor or an iterable of tensors; those without a gradient are
    skipped, one that is listed twice counts once. Gradients: fp16, bf16 or fp32, mixed, on
    one CUDA device, of any alignment (a non-contiguous one goes through a copy). They are
    multiplied by ``max_norm / (norm + 1e-6)`` where that is below 1 and left as they are
    otherwise; a norm that is not a number makes them all so, an infinite one zeroes the
    finite ones, as in torch; ``max_norm=inf`` only measures. Nothing is read back to the host unless ``error_if_nonfinite``
    asks for an error in those two cases (before any gradient changes)."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"clip_grad_norm_: max_norm {max_norm}")
    grads = [g for g in [p.grad for p in params] if g is not None]
    if not grads:
        return torch.zeros((), device=params[0].device if params else None)
    # one attribute of all gradients at a time: with hundreds of small gradients the host's work
    # on them is what the call costs
    dev = grads[0].device
    if dev.type != "cuda":
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, "clip_grad_norm_ runs on CUDA gradients only (no CPU path)")
    if {g.layout for g in grads} != {torch.strided}:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, "clip_grad_norm_: a sparse gradient (need dense ones)")
    if {g.device for g in grads} != {dev}:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, "clip_grad_norm_: gradients on several devices")
    kinds = [g.dtype for g in grads]
    if not _GRAD_DTYPES.keys() >= set(kinds):
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                             f"clip_grad_norm_: gradients of {set(kinds) - _GRAD_DTYPES.keys()} (need fp16, bf16, fp32)")
    ptrs = [g.data_ptr() for g in grads]
    if len(set(ptrs)) < len(ptrs):  # a parameter listed twice counts once (empty gradients share address 0)
        grads = [p.grad for p in dict.fromkeys(params) if p.grad is not None]
        kinds, ptrs = [g.dtype for g in grads], [g.data_ptr() for g in grads]
    copies = []
    if not all([g.is_contiguous() for g in grads]):
        for i, g in enumerate(grads):
            if not g.is_contiguous():
                c = g.contiguous()
                copies.append((g, c))
                ptrs[i] = c.data_ptr()
    count = len(grads)
    table = array("q", ptrs + [g.numel() for g in grads])
    codes = array("i", [_GRAD_DTYPES[k] for k in kinds])
    at = table.buffer_info()[0]
    total = torch.empty((), dtype=torch.float32, device=dev)
    ws_bytes = int(_lib.load().lmce_clip_grad_workspace_bytes(count))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)

    def run(limit):
        _lib.launch(dev, "lmce_clip_grad_norm", at, at + 8 * count, codes.buffer_info()[0], count, limit,
                    total.data_ptr(), ws.data_ptr(), ws_bytes)

    if error_if_nonfinite:
        run(float("inf"))  # measures only
        if not torch.isfinite(total):
            raise RuntimeError(f"clip_grad_norm_: the gradients' norm is {total.item()}, nothing was scaled")
    run(max_norm)
    for g, c in copies:
        g.copy_(c)
    return total
