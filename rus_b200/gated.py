"""Gated projection of a feed-forward block: both projections, the activation and the product
in one kernel, with its backward; and the same on e4m3 operands for serving.

The reference computes it as two cuBLAS products and its SwiGLU kernels
(``solution/kernels.py:355-446``, ``FusedMLPGLUFn`` in ``solution/ops.py:57-85``) around
frozen weights; here the weights get their gradients as well. The down projection that
follows is one plain product. CUDA tensors only: there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .norm import _rows, no_second_order
from .ops import _DTYPES, _debug_sync, _ptr, _raise_device_error

ACTIVATIONS = {"silu": _lib.LMCE_ACT_SILU, "gelu_tanh": _lib.LMCE_ACT_GELU_TANH}


def _check(x, w_gate, w_up, activation, who: str, step: int) -> None:
    dt, dev, shape = x.dtype, x.device, w_gate.shape
    if (activation in ACTIVATIONS and dev.type == "cuda" and w_gate.device == dev and w_up.device == dev
            and w_gate.dtype == dt and w_up.dtype == dt and len(shape) == 2 and w_up.shape == shape and x.dim() > 0
            and x.shape[-1] == shape[1] and shape[0] > 0 and shape[0] % 64 == 0 and shape[1] > 0
            and shape[1] % step == 0):
        return
    if activation not in ACTIVATIONS:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                             f"{who}: activation {activation!r} (need one of {sorted(ACTIVATIONS)})")
    if not (x.is_cuda and w_gate.is_cuda and w_up.is_cuda):
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who} runs on CUDA tensors only (no CPU path)")
    if x.dim() == 0 or w_gate.dim() != 2 or w_up.shape != shape or shape[1] != x.shape[-1]:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT,
                             f"{who}: both weights must be [F, H] with H = x.shape[-1]")
    if w_gate.dtype != dt or w_up.dtype != dt:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: x and both weights must have the same dtype")
    if w_gate.device != dev or w_up.device != dev:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: all tensors must be on the same device")
    raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                         f"{who}: sizes H={shape[1]}, F={shape[0]} (need H a multiple of {step}, F of 64)")


def _forward(x, w_gate, w_up, activation, save: bool):
    f, h = w_gate.shape
    xc, wg, wu = _rows(x), _rows(w_gate), _rows(w_up)
    n = xc.numel() // h
    out = xc.new_empty((*x.shape[:-1], f))
    saved = None
    if n > 0:
        if save:
            saved = xc.new_empty(int(_lib.load().lmce_gated_saved_bytes(n, f)), dtype=torch.uint8)
        _lib.launch(x.device, "lmce_gated_linear", xc.data_ptr(), wg.data_ptr(), wu.data_ptr(), n, h, f,
                    _DTYPES[x.dtype], ACTIVATIONS[activation], out.data_ptr(), _ptr(saved))
        if _debug_sync():
            _raise_device_error()
    return out, xc, wg, wu, saved


class GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        out, xc, wg, wu, saved = _forward(x, w_gate, w_up, activation, True)
        ctx.save_for_backward(xc, wg, wu, saved)
        ctx.activation = activation
        return out

    @staticmethod
    def backward(ctx, dh):
        no_second_order("gated_linear")
        x, wg, wu, saved = ctx.saved_tensors
        want_x, want_g, want_u = ctx.needs_input_grad[:3]
        f, h = wg.shape
        n = x.numel() // h
        dev = x.device
        new = torch.empty_like if n > 0 else torch.zeros_like
        dx = new(x) if want_x else None
        dg = new(wg) if want_g else None
        du = new(wu) if want_u else None
        if n > 0:
            g = _rows(dh)
            ws_bytes = int(_lib.load().lmce_gated_bwd_workspace_bytes(n, h, f, want_x, want_g + want_u))
            ws = x.new_empty(ws_bytes, dtype=torch.uint8)
            _lib.launch(dev, "lmce_gated_backward", g.data_ptr(), saved.data_ptr(), x.data_ptr(), wg.data_ptr(),
                        wu.data_ptr(), n, h, f, _DTYPES[x.dtype], ACTIVATIONS[ctx.activation], _ptr(dx), _ptr(dg),
                        _ptr(du), ws.data_ptr(), ws_bytes)
            if _debug_sync():
                _raise_device_error()
        return dx, dg, du, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu"):
    """``act(x @ w_gate.T) * (x @ w_up.T)`` without either product in memory.

    ``x`` [..., H] and both weights [F, H] in one dtype, fp16 or bf16; H and F multiples of
    64, any number of tokens. ``activation``: ``"silu"`` or ``"gelu_tanh"``. Products
    accumulate and the activation runs in fp32; the result is rounded once. Differentiable in
    ``x`` and both weights (each gradient is computed only if its tensor wants it). When a
    gradient is wanted the forward keeps both products, 24 bits of each, 6 bytes per token
    and feature, for the backward; ``torch.utils.checkpoint`` around the block trades that for a
    second forward."""
    _check(x, w_gate, w_up, activation, "gated_linear", 64)
    if x.dtype not in _DTYPES:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"gated_linear: dtype {x.dtype} (need fp16 or bf16)")
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        return GatedLinearFn.apply(x, w_gate, w_up, activation)
    return _forward(x, w_gate, w_up, activation, False)[0]


def gated_linear_e4m3(x: torch.Tensor, x_scale: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor,
                      w_up: torch.Tensor, up_scale: torch.Tensor, activation: str = "silu",
                      out_dtype: torch.dtype = torch.bfloat16):
    """``gated_linear`` on ``torch.float8_e4m3fn`` operands with fp32 scales, for serving.

    ``x`` [..., H] and ``x_scale`` [...] as ``add_rms_norm_e4m3`` returns them; each weight
    [F, H] with one scale per row [F], laid out once when the weights are loaded::

        scale = w.float().abs().amax(1).clamp(min=1e-12) / 448
        w8 = (w.float() / scale[:, None]).to(torch.float8_e4m3fn)

    H a multiple of 128, F of 64. Products accumulate in fp32, are scaled there, and the
    result is rounded once to ``out_dtype`` (fp16 or bf16). No backward: the scales must not
    require a gradient."""
    who = "gated_linear_e4m3"
    _check(x, w_gate, w_up, activation, who, 128)
    if x.dtype != torch.float8_e4m3fn:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: dtype {x.dtype} (need float8_e4m3fn)")
    if out_dtype not in _DTYPES:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: out_dtype {out_dtype} (need fp16 or bf16)")
    f, h = w_gate.shape
    for name, t, shape in (("x_scale", x_scale, x.shape[:-1]), ("gate_scale", gate_scale, (f,)),
                           ("up_scale", up_scale, (f,))):
        if t.dtype != torch.float32 or t.shape != shape or t.device != x.device:
            raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT,
                                 f"{who}: {name} must be fp32 {tuple(shape)} on the device of x")
        if t.requires_grad and torch.is_grad_enabled():
            raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who} has no backward: call it under torch.no_grad()")
    xc, wg, wu = _rows(x), _rows(w_gate), _rows(w_up)
    sx, sg, su = _rows(x_scale), _rows(gate_scale), _rows(up_scale)
    n = xc.numel() // h
    out = xc.new_empty((*x.shape[:-1], f), dtype=out_dtype)
    if n > 0:
        _lib.launch(x.device, "lmce_gated_linear_e4m3", xc.data_ptr(), sx.data_ptr(), wg.data_ptr(), sg.data_ptr(),
                    wu.data_ptr(), su.data_ptr(), n, h, f, _DTYPES[out_dtype], ACTIVATIONS[activation],
                    out.data_ptr())
        if _debug_sync():
            _raise_device_error()
    return out
