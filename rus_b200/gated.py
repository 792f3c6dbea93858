"""Gated projection of a feed-forward block: both projections, the activation and the product
in one kernel, with its backward; and the same on e4m3 operands for serving.

The reference computes it as two cuBLAS products and its SwiGLU kernels
(``solution/kernels.py:355-446``, ``FusedMLPGLUFn`` in ``solution/ops.py:57-85``) around
frozen weights; here the weights get their gradients as well. The down projection that
follows is one plain product. Allocation and the autograd node are in
``csrc/lmce_host.cpp``. CUDA tensors only: there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import _DTYPES

ACTIVATIONS = {"silu": _lib.LMCE_ACT_SILU, "gelu_tanh": _lib.LMCE_ACT_GELU_TANH}


def _refuse(x, w_gate, w_up, activation, who: str, step: int) -> None:
    """Raise what is wrong with arguments that the host side did not take."""
    if activation not in ACTIVATIONS:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                             f"{who}: activation {activation!r} (need one of {sorted(ACTIVATIONS)})")
    if not (x.is_cuda and w_gate.is_cuda and w_up.is_cuda):
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who} runs on CUDA tensors only (no CPU path)")
    if x.dim() == 0 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_gate.shape[1] != x.shape[-1]:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT,
                             f"{who}: both weights must be [F, H] with H = x.shape[-1]")
    if w_gate.dtype != x.dtype or w_up.dtype != x.dtype:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: x and both weights must have the same dtype")
    if w_gate.device != x.device or w_up.device != x.device:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: all tensors must be on the same device")
    f, h = w_gate.shape
    if f <= 0 or f % 64 or h <= 0 or h % step:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                             f"{who}: sizes H={h}, F={f} (need H a multiple of {step}, F of 64)")


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu"):
    """``act(x @ w_gate.T) * (x @ w_up.T)`` without either product in memory.

    ``x`` [..., H] and both weights [F, H] in one dtype, fp16 or bf16; H and F multiples of
    64, any number of tokens. ``activation``: ``"silu"`` or ``"gelu_tanh"``. Products
    accumulate and the activation runs in fp32; the result is rounded once. Differentiable in
    ``x`` and both weights (each gradient is computed only if its tensor wants it). When a
    gradient is wanted the forward keeps both products, 24 bits of each, 6 bytes per token
    and feature, for the backward; ``torch.utils.checkpoint`` around the block trades that for a
    second forward."""
    act = ACTIVATIONS.get(activation)
    if act is not None and x.is_cuda:
        out = (_lib._host or _lib.host()).gated_linear(x, w_gate, w_up, act)
        if out is not None:
            return out
    _refuse(x, w_gate, w_up, activation, "gated_linear", 64)
    raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"gated_linear: dtype {x.dtype} (need dense fp16 or bf16)")


def gated_linear_e4m3(x: torch.Tensor, x_scale: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor,
                      w_up: torch.Tensor, up_scale: torch.Tensor, activation: str = "silu",
                      out_dtype: torch.dtype = torch.bfloat16):
    """``gated_linear`` on ``torch.float8_e4m3fn`` operands with fp32 scales, for serving.

    ``x`` [..., H] and ``x_scale`` [...] as ``add_rms_norm_e4m3`` returns them; each weight
    [F, H] with one scale per row [F], laid out once when the weights are loaded::

        scale = w.float().abs().amax(1).clamp(min=1e-12) / 448
        w8 = (w.float() / scale[:, None]).to(torch.float8_e4m3fn)

    H a multiple of 128, F of 64. Products accumulate in fp32, are scaled there, and the
    result is rounded once to ``out_dtype`` (fp16 or bf16). No backward: a call that autograd
    would have to record is refused (an e4m3 ``nn.Parameter`` requires a gradient unless it is
    made with ``requires_grad=False``)."""
    act = ACTIVATIONS.get(activation)
    if act is not None and x.is_cuda:
        out = (_lib._host or _lib.host()).gated_linear_e4m3(x, x_scale, w_gate, gate_scale, w_up, up_scale, act,
                                                            out_dtype)
        if out is not None:
            return out
    who = "gated_linear_e4m3"
    _refuse(x, w_gate, w_up, activation, who, 128)
    if x.dtype != torch.float8_e4m3fn:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: dtype {x.dtype} (need float8_e4m3fn)")
    if out_dtype not in _DTYPES:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: out_dtype {out_dtype} (need fp16 or bf16)")
    f = w_gate.shape[0]
    for name, t, shape in (("x_scale", x_scale, x.shape[:-1]), ("gate_scale", gate_scale, (f,)),
                           ("up_scale", up_scale, (f,))):
        if t.dtype != torch.float32 or t.shape != shape or t.device != x.device:
            raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT,
                                 f"{who}: {name} must be fp32 {tuple(shape)} on the device of x")
    raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                         f"{who} has no backward and takes dense tensors: call it under torch.no_grad()")
