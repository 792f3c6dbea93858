"""CPU: what the operators around the head refuse (residual norm, gated projection, gradient
clipping), at the C entries, which check their arguments before they touch a device, and at the
Python functions for tensors that are not on one."""
from __future__ import annotations

import ctypes

import pytest
import torch

from rus_b200 import (_lib, add_rms_norm, add_rms_norm_e4m3, clip_grad_norm_, gated_linear, gated_linear_e4m3)

INVALID, UNSUPPORTED, WORKSPACE = _lib.LMCE_ERR_INVALID_ARGUMENT, _lib.LMCE_ERR_UNSUPPORTED, _lib.LMCE_ERR_WORKSPACE
P = 4096  # an aligned address that no refused call reads


def _refused(name, args, code):
    assert getattr(_lib.load(), name)(*args) == code, (name, args)
    assert _lib.load().lmce_last_error()


@pytest.mark.parametrize("name", ["lmce_add_rmsnorm", "lmce_add_rmsnorm_e4m3"])
def test_add_rmsnorm_entries(name):
    #        x  residual w  eps   n  h   dt s  y/q rstd/scale stream
    good = [P, P, P, 1e-6, 4, 64, 0, P, P, P, None]

    def bad(code, **changes):
        args = list(good)
        for i, v in changes.items():
            args[int(i[1:])] = v
        _refused(name, args, code)

    for i in (0, 2, 8):
        bad(INVALID, **{f"_{i}": None})
    bad(INVALID, _7=None)  # a residual without room for the sum
    for n in (0, -1, (1 << 30) + 1):
        bad(INVALID, _4=n)
    for h in (0, -8, 4, 60, 16392):
        bad(UNSUPPORTED, _5=h)
    for dt in (2, -1, 7):
        bad(UNSUPPORTED, _6=dt)
    for i in (0, 1, 2, 7, 8):
        bad(INVALID, **{f"_{i}": P + 2})


def test_add_rmsnorm_backward_entry():
    #        dy ds s  w  rstd n  h   dt dx dw ws bytes stream
    good = [P, P, P, P, P, 4, 64, 0, P, P, P, 1 << 20, None]
    for i, v, code in ((2, None, INVALID), (3, None, INVALID), (4, None, INVALID), (5, 0, INVALID),
                       (6, 20, UNSUPPORTED), (7, 3, UNSUPPORTED), (8, P + 8, INVALID), (10, None, WORKSPACE),
                       (11, 4 * 64 * 4 - 1, WORKSPACE)):
        _refused("lmce_add_rmsnorm_backward", good[:i] + [v] + good[i + 1:], code)
    _refused("lmce_add_rmsnorm_backward", good[:8] + [None, None] + good[10:], INVALID)  # no output at all


def test_gated_entries():
    #        x  wg wu n  h   f   dt act h  saved stream
    good = [P, P, P, 4, 64, 128, 1, 0, P, P, None]
    for i, v, code in ((0, None, INVALID), (1, None, INVALID), (2, None, INVALID), (8, None, INVALID),
                       (3, 0, INVALID), (3, (1 << 26) + 1, INVALID), (4, 0, UNSUPPORTED), (4, 72, UNSUPPORTED),
                       (5, 96, UNSUPPORTED), (5, -64, UNSUPPORTED), (6, 2, UNSUPPORTED), (7, 2, UNSUPPORTED),
                       (0, P + 2, INVALID), (1, P + 8, INVALID), (9, P + 4, INVALID)):
        _refused("lmce_gated_linear", good[:i] + [v] + good[i + 1:], code)
    #        x  xs wg gs wu us n  h    f   dt act h  stream
    good = [P, P, P, P, P, P, 4, 128, 128, 1, 0, P, None]
    for i, v, code in ((1, None, INVALID), (3, None, INVALID), (5, None, INVALID), (7, 64, UNSUPPORTED),
                       (8, 32, UNSUPPORTED), (9, 5, UNSUPPORTED), (10, -1, UNSUPPORTED), (3, P + 4, INVALID),
                       (1, P + 2, INVALID), (11, None, INVALID)):
        _refused("lmce_gated_linear_e4m3", good[:i] + [v] + good[i + 1:], code)
    #        dh saved x wg wu n  h   f   dt act dx dg du ws bytes stream
    good = [P, P, P, P, P, 4, 64, 128, 0, 0, P, P, P, P, 1 << 30, None]
    for i, v, code in ((0, None, INVALID), (1, None, INVALID), (13, None, INVALID), (5, 0, INVALID),
                       (6, 32, UNSUPPORTED), (8, 9, UNSUPPORTED), (9, 3, UNSUPPORTED), (12, P + 2, INVALID),
                       (13, P + 16, INVALID), (14, 100, WORKSPACE)):
        _refused("lmce_gated_backward", good[:i] + [v] + good[i + 1:], code)
    _refused("lmce_gated_backward", good[:10] + [None] * 3 + good[13:], INVALID)


def _clip(ptrs, numels, dtypes, max_norm=1.0, total=P, ws=P, ws_bytes=1 << 20):
    n = len(ptrs)
    return [(ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numels), (ctypes.c_int32 * n)(*dtypes), n, max_norm,
            total, ws, ws_bytes, None]


def test_clip_entry():
    f32, f16 = _lib.LMCE_DTYPE_F32, _lib.LMCE_DTYPE_F16
    refuse = lambda args, code: _refused("lmce_clip_grad_norm", args, code)  # noqa: E731
    refuse(_clip([P, P + 396], [100, 5], [f32, f32]), INVALID)              # one element shared
    refuse(_clip([P + 4096, P], [100, 3000], [f16, f16]), INVALID)          # in any order
    refuse(_clip([P, P], [100, 100], [f32, f32]), INVALID)                  # listed twice
    refuse(_clip([P + 2], [4], [f32]), INVALID)
    refuse(_clip([P + 1], [4], [f16]), INVALID)
    refuse(_clip([0], [4], [f16]), INVALID)
    refuse(_clip([P], [-1], [f16]), INVALID)
    refuse(_clip([P], [4], [3]), UNSUPPORTED)
    for bad in (-1.0, float("nan")):
        refuse(_clip([P], [4], [f32], max_norm=bad), INVALID)
    refuse(_clip([P], [4], [f32], total=None), INVALID)
    refuse(_clip([P], [4], [f32], ws_bytes=16), WORKSPACE)
    refuse(_clip([P], [4], [f32], ws=P + 4), WORKSPACE)
    refuse([None] * 3 + [1, 1.0, P, P, 1 << 20, None], INVALID)
    args = _clip([P], [4], [f32])
    args[3] = 0
    refuse(args, INVALID)


def test_workspaces():
    lib = _lib.load()
    assert lib.lmce_gated_saved_bytes(33, 64) == 64 * 64 * 6  # tokens in blocks of 32
    assert lib.lmce_gated_saved_bytes(0, 64) == 0 and lib.lmce_clip_grad_workspace_bytes(0) == 0
    assert lib.lmce_add_rmsnorm_bwd_workspace_bytes(5, 64) == 5 * 64 * 4
    # the partial rows of the norm's weight gradient do not grow with the tokens
    assert lib.lmce_add_rmsnorm_bwd_workspace_bytes(1 << 20, 64) == lib.lmce_add_rmsnorm_bwd_workspace_bytes(1000, 64)
    # many tokens: dg and du, no partial sums of dx
    n, h, f = 8192, 4096, 14336
    assert lib.lmce_gated_bwd_workspace_bytes(n, h, f, 1, 2) == 2 * n * f * 2
    # few tokens: fp32 partials of dx as well, at most 16
    small = lib.lmce_gated_bwd_workspace_bytes(1, 1536, 8960, 1, 2)
    assert small <= 2 * (8960 * 2 + 256) + 16 * 256 * 1536 * 4 + 256
    assert lib.lmce_gated_bwd_workspace_bytes(1, 1536, 8960, 0, 2) < 1 << 16


def test_host_side_loads_and_takes_cuda_tensors_only():
    host = _lib.host()
    assert host is _lib.host() and host.torch_version == torch.__version__.split("+")[0]
    x, w = torch.randn(4, 128).half(), torch.ones(128).half()
    wg = torch.randn(64, 128).half()
    q, s4, s64 = x.to(torch.float8_e4m3fn), torch.ones(4), torch.ones(64)
    assert host.add_rms_norm(x, x, w, 1e-6) is None and host.add_rms_norm_e4m3(x, None, w, 1e-6) is None
    assert host.gated_linear(x, wg, wg, 0) is None
    q8 = wg.to(torch.float8_e4m3fn)
    assert host.gated_linear_e4m3(q, s4, q8, s64, q8, s64, 0, torch.float16) is None
    p = torch.zeros(4, requires_grad=True)
    assert host.clip_grad_norm([], 1.0, True) is None and host.clip_grad_norm([p], 1.0, True) is None
    p.grad = torch.ones(4)
    assert host.clip_grad_norm([p], 1.0, True) is None and host.clip_grad_norm([p.grad, 3], 1.0, False) is None
    with pytest.raises(TypeError):
        host.add_rms_norm(x, x, None, 1e-6)


def test_tensors_on_the_cpu():
    x, w = torch.randn(4, 128).half(), torch.ones(128).half()
    wg = torch.randn(64, 128).half()
    q, sx, sw = x.to(torch.float8_e4m3fn), torch.ones(4), torch.ones(64)
    q8 = wg.to(torch.float8_e4m3fn)
    for call in (lambda: add_rms_norm(x, x, w), lambda: add_rms_norm_e4m3(x, None, w),
                 lambda: gated_linear(x, wg, wg), lambda: gated_linear_e4m3(q, sx, q8, sw, q8, sw)):
        with pytest.raises(_lib.LmceError, match="CUDA"):
            call()
    p = torch.zeros(4, requires_grad=True)
    assert clip_grad_norm_([p], 1.0).item() == 0.0 and clip_grad_norm_([], 1.0).item() == 0.0  # no gradient yet
    p.grad = torch.ones(4)
    with pytest.raises(_lib.LmceError, match="CUDA"):
        clip_grad_norm_([p], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(_lib.LmceError, match="max_norm"):
            clip_grad_norm_([p], bad)
    with pytest.raises(_lib.LmceError, match="activation"):
        gated_linear(x, wg, wg, "relu")
