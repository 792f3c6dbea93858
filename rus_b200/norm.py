"""Residual addition with its RMSNorm, and the same with an e4m3 output for 8-bit products.

What a decoder block runs in front of its attention and its feed-forward projections; the
reference fuses the pair in ``rms_norm_fwd`` (``solution/kernels.py:124-164``) with the
backward ``rms_norm_bwd`` (``kernels.py:167-190``, no weight gradient). ``rms_norm_pack``
(``packing.py``) is the final norm in front of the head; these stand in front of every
block. Allocation and the autograd node are in ``csrc/lmce_host.cpp``. CUDA tensors only:
there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import _DTYPES


def _refuse(x, residual, weight, who: str) -> None:
    """Raise what is wrong with arguments that the host side did not take."""
    if not x.is_cuda or not weight.is_cuda or (residual is not None and not residual.is_cuda):
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who} runs on CUDA tensors only (no CPU path)")
    if x.dtype not in _DTYPES:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: dtype {x.dtype} (need fp16 or bf16)")
    if x.dim() == 0 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: weight must be [H] with H = x.shape[-1]")
    if weight.dtype != x.dtype or (residual is not None and residual.dtype != x.dtype):
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: x, residual and weight must have the same dtype")
    if residual is not None and residual.shape != x.shape:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: residual must have the shape of x")
    if weight.device != x.device or (residual is not None and residual.device != x.device):
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: all tensors must be on the same device")
    if x.shape[-1] % 8 != 0 or not 0 < x.shape[-1] <= 16384:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                             f"{who}: hidden size {x.shape[-1]} (need a multiple of 8, at most 16384)")
    raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: need dense tensors, and torch.no_grad() where "
                                                    "the operator has no backward")


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6):
    """The residual stream ``s = x + residual`` and its RMSNorm ``y``: returns ``(y, s)``.

    ``x`` and ``residual`` [..., H] fp16 or bf16 of one shape (``residual=None``: the first
    block, ``s`` is ``x``), ``weight`` [H] in the same dtype, H a multiple of 8. ``s`` is
    rounded to the inputs' dtype and ``y = s / sqrt(mean(s^2) + eps) * weight`` is computed
    from that ``s`` in fp32 and rounded once. Differentiable in all three tensors; the
    gradient of ``x`` and of ``residual`` is the same tensor. A row that holds an infinity or
    a NaN affects no other row of the outputs (it does reach the weight's gradient)."""
    if x.is_cuda:
        out = (_lib._host or _lib.host()).add_rms_norm(x, residual, weight, eps)
        if out is not None:
            return out
    _refuse(x, residual, weight, "add_rms_norm")


def add_rms_norm_e4m3(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6):
    """``add_rms_norm`` with the norm's output in 8 bits: returns ``(q, scale, s)``.

    ``q`` [..., H] ``torch.float8_e4m3fn`` and ``scale`` [...] fp32 stand for ``q * scale``:
    each row's scale maps its largest magnitude to e4m3's largest value, 448 (scale 1 for a
    row of zeros). They are the operand ``gated_linear_e4m3`` takes. Serving only: a call
    that autograd would have to record is refused."""
    if x.is_cuda:
        out = (_lib._host or _lib.host()).add_rms_norm_e4m3(x, residual, weight, eps)
        if out is not None:
            return out
    _refuse(x, residual, weight, "add_rms_norm_e4m3")
