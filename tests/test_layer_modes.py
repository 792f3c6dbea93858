"""CPU: the operators around the head under torch's modes. Their host side looks at these before it
looks at a device, so the refusals are the same for tensors that are not on one."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from rus_b200 import _lib


def _calls():
    """Per operator: its host function's arguments and which of them are floating-point tensors."""
    x, w = torch.randn(4, 128).half(), torch.ones(128).half()
    wg, wu = torch.randn(64, 128).half(), torch.randn(64, 128).half()
    q, q8, u8 = (t.to(torch.float8_e4m3fn) for t in (x, wg, wu))
    s4, s64 = torch.ones(4), torch.ones(64)
    return {
        "add_rms_norm": ([x, x.clone(), w, 1e-6], (0, 1, 2)),
        "add_rms_norm_e4m3": ([x, x.clone(), w, 1e-6], (0, 1, 2)),
        "gated_linear": ([x, wg, wu, 0], (0, 1, 2)),
        "gated_linear_e4m3": ([q, s4, q8, s64, u8, s64.clone(), 0, torch.float16], (1, 3, 5)),
        "clip_grad_norm": ([[s4, s64], 1.0, False], ()),
    }


@pytest.mark.parametrize("name", list(_calls()))
def test_tangents_are_refused(name):
    """A dual tensor does not require a gradient: the derivative must not be dropped in silence."""
    args, tensors = _calls()[name]
    call = getattr(_lib.host(), name)
    with fwd.dual_level():
        if name == "clip_grad_norm":
            cases = [[[fwd.make_dual(args[0][0], torch.ones(4)), args[0][1]], 1.0, False]]
        else:
            cases = [args[:i] + [fwd.make_dual(args[i], torch.ones_like(args[i]))] + args[i + 1:] for i in tensors]
        for bad in cases:
            with pytest.raises(_lib.LmceError, match="forward-mode") as e:
                call(*bad)
            assert e.value.code == _lib.LMCE_ERR_UNSUPPORTED
            with fwd._set_fwd_grad_enabled(False):  # tangents are not asked for
                assert call(*bad) is None
        assert call(*args) is None  # no tangent among the arguments: what is wrong here is the device


def _refused_as_traced(call, *args):
    with pytest.raises(_lib.LmceError, match="traced") as e:
        call(*args)
    assert e.value.code == _lib.LMCE_ERR_UNSUPPORTED


@pytest.mark.parametrize("name", list(_calls()))
def test_traces_are_refused(name):
    """A trace holds the outputs' allocation and not the kernel: it would return memory as found."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    args, _ = _calls()[name]
    call = getattr(_lib.host(), name)
    seen = []

    def f(a):
        _refused_as_traced(call, *args)
        seen.append(1)
        return a + 1

    a = torch.ones(3)
    torch.jit.trace(f, (a,), check_trace=False)
    make_fx(f)(a)
    make_fx(f, pre_dispatch=True)(a)
    make_fx(f, tracing_mode="fake")(a)
    with FakeTensorMode():
        f(torch.ones(3))
    assert len(seen) == 5
    with FlopCounterMode(display=False):  # a mode that watches what runs
        assert call(*args) is None
    assert call(*args) is None


@pytest.mark.parametrize("name", ["lmce_add_rmsnorm", "lmce_add_rmsnorm_e4m3"])
def test_the_sum_is_not_looked_at_without_a_residual(name):
    """The entries refuse a misaligned s_out only where they would write it: here they go on to the
    device, or to the next argument that is wrong."""
    p = 4096  # an aligned address that no refused call reads
    #       x  residual w  eps   n  h   dt s      y/q    rstd/scale stream
    args = [p, None, p, 1e-6, 4, 64, 0, p + 2, p + 2, p, None]  # y misaligned
    entry, lib = getattr(_lib.load(), name), _lib.load()
    assert entry(*args) == _lib.LMCE_ERR_INVALID_ARGUMENT and b"misaligned" in lib.lmce_last_error()
    args[1], args[8] = p, p
    assert entry(*args) == _lib.LMCE_ERR_INVALID_ARGUMENT and b"misaligned" in lib.lmce_last_error()
    if not torch.cuda.is_available():
        args[1] = None
        assert entry(*args) == _lib.LMCE_ERR_CUDA
