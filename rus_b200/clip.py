"""Clipping gradients by their global norm, on the device.

The step between ``loss.backward()`` through the head and the optimizer: the same call and
result as ``torch.nn.utils.clip_grad_norm_`` with the 2-norm (TRL's trainer, which drives
the reference's patched forward, calls that with ``max_grad_norm`` and logs the norm), in two
launches for up to 1024 gradients of any mix of fp16, bf16 and fp32.
"""
from __future__ import annotations

import torch

from . import _lib

_GRAD_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


@torch.no_grad()
def _clip_any(params: list[torch.Tensor], max_norm: float, error_if_nonfinite: bool) -> torch.Tensor:
    """Distinct parameters with gradients of any kind: what is refused is said here, and strided
    gradients go through copies."""
    grads = [g for p in params if (g := p.grad) is not None]
    if not grads:
        return torch.zeros((), device=params[0].device if params else None)
    for g in grads:
        if g.device.type != "cuda":
            raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                                 "clip_grad_norm_ runs on CUDA gradients only (no CPU path)")
        if g.device != grads[0].device:
            raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, "clip_grad_norm_: gradients on several devices")
        if g.layout != torch.strided or g.dtype not in _GRAD_DTYPES:
            raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"clip_grad_norm_: gradient {g.dtype}, {g.layout} "
                                                            "(need dense fp16, bf16 or fp32)")
        if any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)):
            raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT,
                                 "clip_grad_norm_: an expanded gradient (its elements share memory)")
    # the copies of strided gradients hide from the library what shares memory
    starts = [g.data_ptr() for g in grads if g.numel() > 0]
    if len(set(starts)) < len(starts):
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, "clip_grad_norm_: gradients overlap in memory")
    flat = [g.contiguous() for g in grads]

    def run(limit):
        return _lib.host().clip_grad_norm(flat, limit, False)

    if error_if_nonfinite:
        total = run(float("inf"))  # measures only
        if not torch.isfinite(total):
            raise RuntimeError(f"clip_grad_norm_: the gradients' norm is {total.item()}, nothing was scaled")
    total = run(max_norm)
    if max_norm != float("inf"):
        for g, c in zip(grads, flat):
            if c is not g:
                g.copy_(c)
    return total


def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place so that their global 2-norm is at most
    ``max_norm``; returns the norm they had (fp32 scalar on their device).

    ``parameters`` is a tensor or an iterable of tensors; those without a gradient are
    skipped, one that is listed twice counts once. Gradients: fp16, bf16 or fp32, mixed, on
    one CUDA device, of any alignment (a non-contiguous one goes through a copy), none
    overlapping another in memory. The norm is over this process's gradients: for a
    vocabulary shard it covers the shard. They are multiplied by ``max_norm / (norm + 1e-6)``
    where that is below 1 and left as they are otherwise; a norm that is not a number makes
    them all so, an infinite one zeroes the finite ones, as in torch; ``max_norm=inf`` only
    measures. With any other limit autograd sees an in-place change of each gradient, scaled or
    not. Nothing is read back to the host unless ``error_if_nonfinite`` asks for an error in
    those two cases (before any gradient changes)."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"clip_grad_norm_: max_norm {max_norm}")
    if params and params[0].is_cuda and not error_if_nonfinite:
        total = (_lib._host or _lib.host()).clip_grad_norm(params, max_norm, True)
        if total is not None:  # contiguous gradients, each listed once
            return total
    return _clip_any(list(dict.fromkeys(params)), max_norm, error_if_nonfinite)
