"""Clipping gradients by their global norm, on the device.

The step between ``loss.backward()`` through the head and the optimizer: the same call and
result as ``torch.nn.utils.clip_grad_norm_`` with the 2-norm (TRL's trainer, which drives
the reference's patched forward, calls that with ``max_grad_norm`` and logs the norm), in two
launches for up to 1024 gradients of any mix of fp16, bf16 and fp32.
"""
from __future__ import annotations

from array import array
from operator import attrgetter

import torch

from . import _lib

_GRAD_DTYPES = {torch.float16: _lib.LMCE_DTYPE_F16, torch.bfloat16: _lib.LMCE_DTYPE_BF16,
                torch.float32: _lib.LMCE_DTYPE_F32}
_dtype_of = attrgetter("dtype")


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place so that their global 2-norm is at most
    ``max_norm``; returns the norm they had (fp32 scalar on their device).

    ``parameters`` is a tensor or an iterable of tensors; those without a gradient are
    skipped, one that is listed twice counts once. Gradients: fp16, bf16 or fp32, mixed, on
    one CUDA device, of any alignment (a non-contiguous one goes through a copy), none
    overlapping another in memory. The norm is over this process's gradients: for a
    vocabulary shard it covers the shard. They are
    multiplied by ``max_norm / (norm + 1e-6)`` where that is below 1 and left as they are
    otherwise; a norm that is not a number makes them all so, an infinite one zeroes the
    finite ones, as in torch; ``max_norm=inf`` only measures. Nothing is read back to the host
    unless ``error_if_nonfinite`` asks for an error in those two cases (before any gradient
    changes)."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"clip_grad_norm_: max_norm {max_norm}")
    grads = [g for p in params if (g := p.grad) is not None]
    if not grads:
        return torch.zeros((), device=params[0].device if params else None)
    # one attribute of all gradients at a time, through C-level maps: with hundreds of small
    # gradients the host's work on them is what the call costs
    dev = grads[0].device
    if dev.type != "cuda":
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, "clip_grad_norm_ runs on CUDA gradients only (no CPU path)")
    if set(map(torch.Tensor.get_device, grads)) != {dev.index}:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, "clip_grad_norm_: gradients on several devices")
    kinds = list(map(_dtype_of, grads))
    distinct = set(kinds)
    if not _GRAD_DTYPES.keys() >= distinct:
        other = distinct - _GRAD_DTYPES.keys()
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                             f"clip_grad_norm_: gradients of {other} (need fp16, bf16 or fp32)")
    try:
        table = array("q", map(torch.Tensor.data_ptr, grads))
    except RuntimeError as e:  # no storage
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"clip_grad_norm_: a gradient that is not dense ({e})") from e
    copies = []
    if not all(map(torch.Tensor.is_contiguous, grads)):
        # the copies hide from the library what shares memory
        if len(set(map(id, params))) < len(params):
            return clip_grad_norm_(dict.fromkeys(params), max_norm, error_if_nonfinite)
        starts = [a for a, g in zip(table, grads) if g.numel() > 0]
        if len(set(starts)) < len(starts):
            raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, "clip_grad_norm_: gradients overlap in memory")
        for i, g in enumerate(grads):
            if not g.is_contiguous():
                if any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)):
                    raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT,
                                         "clip_grad_norm_: an expanded gradient (its elements share memory)")
                c = g.contiguous()
                copies.append((g, c))
                table[i] = c.data_ptr()
    count = len(grads)
    table.extend(map(torch.Tensor.numel, grads))
    if len(distinct) == 1:
        codes = array("i", [_GRAD_DTYPES[kinds[0]]]) * count
    else:
        codes = array("i", map(_GRAD_DTYPES.__getitem__, kinds))
    at = table.buffer_info()[0]
    total = grads[0].new_empty((), dtype=torch.float32)
    ws_bytes = int(_lib.load().lmce_clip_grad_workspace_bytes(count))
    ws = total.new_empty(ws_bytes, dtype=torch.uint8)

    def run(limit):
        _lib.launch(dev, "lmce_clip_grad_norm", at, at + 8 * count, codes.buffer_info()[0], count, limit,
                    total.data_ptr(), ws.data_ptr(), ws_bytes)

    try:
        if error_if_nonfinite:
            run(float("inf"))  # measures only
            if not torch.isfinite(total):
                raise RuntimeError(f"clip_grad_norm_: the gradients' norm is {total.item()}, nothing was scaled")
        run(max_norm)
    except _lib.LmceError as e:
        # refused before any launch; a parameter listed twice counts once
        if e.code == _lib.LMCE_ERR_INVALID_ARGUMENT and len(set(map(id, params))) < len(params):
            return clip_grad_norm_(dict.fromkeys(params), max_norm, error_if_nonfinite)
        raise
    for g, c in copies:
        g.copy_(c)
    return total
