"""Residual addition with its RMSNorm, and the same with an e4m3 output for 8-bit products.

What a decoder block runs in front of its attention and its feed-forward projections; the
reference fuses the pair in ``rms_norm_fwd`` (``solution/kernels.py:124-164``) with the
backward ``rms_norm_bwd`` (``kernels.py:167-190``, no weight gradient). ``rms_norm_pack``
(``packing.py``) is the final norm in front of the head; these stand in front of every
block. CUDA tensors only: there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import _DTYPES, _ptr


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and on a 16-byte boundary (a copy where it is not)."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def no_second_order(who: str) -> None:
    """In a backward: autograd runs it in grad mode only to differentiate it again."""
    if torch.is_grad_enabled():
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: no second derivative (create_graph=True)")


def _check(x, residual, weight, who: str) -> None:
    dt, dev, shape = x.dtype, x.device, x.shape
    if (dt in _DTYPES and dev.type == "cuda" and weight.dtype == dt and weight.device == dev and weight.dim() == 1
            and shape and shape[-1] == weight.shape[0] and shape[-1] % 8 == 0 and 0 < shape[-1] <= 16384
            and (residual is None or (residual.dtype == dt and residual.device == dev and residual.shape == shape))):
        return
    if not x.is_cuda or not weight.is_cuda or (residual is not None and not residual.is_cuda):
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who} runs on CUDA tensors only (no CPU path)")
    if dt not in _DTYPES:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: dtype {dt} (need fp16 or bf16)")
    if not shape or weight.dim() != 1 or weight.shape[0] != shape[-1]:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: weight must be [H] with H = x.shape[-1]")
    if weight.dtype != dt or (residual is not None and residual.dtype != dt):
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED, f"{who}: x, residual and weight must have the same dtype")
    if residual is not None and residual.shape != shape:
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: residual must have the shape of x")
    if weight.device != dev or (residual is not None and residual.device != dev):
        raise _lib.LmceError(_lib.LMCE_ERR_INVALID_ARGUMENT, f"{who}: all tensors must be on the same device")
    raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                         f"{who}: hidden size {shape[-1]} (need a multiple of 8, at most 16384)")


def _forward(x, residual, weight, eps, keep_rstd: bool):
    h = x.shape[-1]
    xc, w = _rows(x), _rows(weight)
    rc = None if residual is None else _rows(residual)
    n = xc.numel() // h
    y = torch.empty_like(xc)
    s = xc if rc is None else torch.empty_like(xc)
    rstd = xc.new_empty(n, dtype=torch.float32) if keep_rstd else None
    if n > 0:
        _lib.launch(x.device, "lmce_add_rmsnorm", xc.data_ptr(), _ptr(rc), w.data_ptr(), eps, n, h, _DTYPES[x.dtype],
                    s.data_ptr(), y.data_ptr(), _ptr(rstd))
    return y, s, w, rstd


class AddRMSNormFn(torch.autograd.Function):
    """(y, s) of ``add_rms_norm`` (y alone without a residual)."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, s, w, rstd = _forward(x, residual, weight, eps, True)
        ctx.save_for_backward(s, w, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, s)

    @staticmethod
    def backward(ctx, dy, ds=None):
        no_second_order("add_rms_norm")
        s, w, rstd = ctx.saved_tensors
        want_x, want_r, want_w = ctx.needs_input_grad[:3]
        if dy is None and ds is None:
            return None, None, None, None
        n, h = rstd.numel(), s.shape[-1]
        dev = s.device
        dx = torch.empty_like(s) if want_x or want_r else None
        dw = torch.zeros_like(w) if want_w and (dy is None or n == 0) else torch.empty_like(w) if want_w else None
        want_dw = want_w and dy is not None
        if n > 0 and (dx is not None or want_dw):
            g = None if dy is None else _rows(dy)
            gs = None if ds is None else _rows(ds)
            ws, ws_bytes = None, 0
            if want_dw:
                ws_bytes = int(_lib.load().lmce_add_rmsnorm_bwd_workspace_bytes(n, h))
                ws = s.new_empty(ws_bytes, dtype=torch.uint8)
            _lib.launch(dev, "lmce_add_rmsnorm_backward", _ptr(g), _ptr(gs), s.data_ptr(), w.data_ptr(),
                        rstd.data_ptr(), n, h, _DTYPES[s.dtype], _ptr(dx), dw.data_ptr() if want_dw else None,
                        _ptr(ws), ws_bytes)
        return dx if want_x else None, dx if want_r else None, dw, None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6):
    """The residual stream ``s = x + residual`` and its RMSNorm ``y``: returns ``(y, s)``.

    ``x`` and ``residual`` [..., H] fp16 or bf16 of one shape (``residual=None``: the first
    block, ``s`` is ``x``), ``weight`` [H] in the same dtype, H a multiple of 8. ``s`` is
    rounded to the inputs' dtype and ``y = s / sqrt(mean(s^2) + eps) * weight`` is computed
    from that ``s`` in fp32 and rounded once. Differentiable in all three tensors; the
    gradient of ``x`` and of ``residual`` is the same tensor. A row that holds an infinity or
    a NaN affects no other row of the outputs (it does reach the weight's gradient)."""
    _check(x, residual, weight, "add_rms_norm")
    needs = x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)
    if torch.is_grad_enabled() and needs:
        out = AddRMSNormFn.apply(x, residual, weight, eps)
        return (out, x) if residual is None else out
    y, s, _, _ = _forward(x, residual, weight, eps, False)
    return y, (x if residual is None else s)


def add_rms_norm_e4m3(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6):
    """``add_rms_norm`` with the norm's output in 8 bits: returns ``(q, scale, s)``.

    ``q`` [..., H] ``torch.float8_e4m3fn`` and ``scale`` [...] fp32 stand for ``q * scale``:
    each row's scale maps its largest magnitude to e4m3's largest value, 448 (scale 1 for a
    row of zeros). They are the operand ``gated_linear_e4m3`` takes. Serving only: a call
    that autograd would have to record is refused."""
    _check(x, residual, weight, "add_rms_norm_e4m3")
    needs = x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)
    if torch.is_grad_enabled() and needs:
        raise _lib.LmceError(_lib.LMCE_ERR_UNSUPPORTED,
                             "add_rms_norm_e4m3 has no backward: call it under torch.no_grad()")
    h = x.shape[-1]
    xc, w = _rows(x), _rows(weight)
    rc = None if residual is None else _rows(residual)
    n = xc.numel() // h
    q = torch.empty_like(xc, dtype=torch.float8_e4m3fn)
    scale = xc.new_empty(x.shape[:-1], dtype=torch.float32)
    s = xc if rc is None else torch.empty_like(xc)
    if n > 0:
        _lib.launch(x.device, "lmce_add_rmsnorm_e4m3", xc.data_ptr(), _ptr(rc), w.data_ptr(), eps, n, h,
                    _DTYPES[x.dtype], s.data_ptr(), q.data_ptr(), scale.data_ptr())
    return q, scale, (x if residual is None else s)
