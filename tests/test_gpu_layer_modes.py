"""GPU: the operators around the head under torch's modes, hooks and unusual calls."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from rus_b200 import (_lib, add_rms_norm, add_rms_norm_e4m3, clip_grad_norm_, gated_linear, gated_linear_e4m3)

pytestmark = pytest.mark.gpu


def _e4m3(t):
    scale = t.float().abs().amax(1) / 448
    return (t.float() / scale[:, None]).to(torch.float8_e4m3fn), scale


def _inputs(dev, n=4, h=128, f=64):
    g = torch.Generator(device=dev).manual_seed(11)
    x, r = (torch.randn(n, h, device=dev, generator=g).half() for _ in range(2))
    w = (1 + 0.1 * torch.randn(h, device=dev, generator=g)).half()
    wg, wu = ((torch.randn(f, h, device=dev, generator=g) * h ** -0.5).half() for _ in range(2))
    return x, r, w, wg, wu


def test_tangents_are_refused(cuda_device):
    x, r, w, wg, wu = _inputs(cuda_device)
    q, sx = _e4m3(x)
    (g8, sg), (u8, su) = _e4m3(wg), _e4m3(wu)
    p = torch.zeros(4, device=cuda_device, requires_grad=True)
    with fwd.dual_level():
        d = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        p.grad = d(torch.full((4,), 3.0, device=cuda_device))
        for call in (lambda: add_rms_norm(d(x), r, w), lambda: add_rms_norm(x, d(r), w),
                     lambda: add_rms_norm(x, None, d(w)), lambda: add_rms_norm_e4m3(d(x), None, w),
                     lambda: add_rms_norm(d(x), r, w.clone().requires_grad_(True)),
                     lambda: gated_linear(d(x), wg, wu), lambda: gated_linear(x, wg, d(wu)),
                     lambda: gated_linear_e4m3(q, d(sx), g8, sg, u8, su), lambda: clip_grad_norm_([p], 1.0)):
            with pytest.raises(_lib.LmceError, match="forward-mode"):
                call()
    assert (p.grad == 3.0).all()


def test_a_backward_raises_the_packages_error(cuda_device):
    x, r, w, wg, wu = _inputs(cuda_device)
    x.requires_grad_(True)
    for out in (add_rms_norm(x, r, w)[0], gated_linear(x, wg, wu)):
        with pytest.raises(_lib.LmceError, match="second derivative") as e:
            torch.autograd.grad(out.sum(), x, create_graph=True)
        assert e.value.code == _lib.LMCE_ERR_UNSUPPORTED
        loss = out.float().square().sum()
        with pytest.raises(_lib.LmceError):
            loss.backward(create_graph=True)
        assert x.grad is None


def test_traces_are_refused(cuda_device):
    from torch.fx.experimental.proxy_tensor import make_fx

    x, r, w, wg, wu = _inputs(cuda_device)
    q, sx = _e4m3(x)
    (g8, sg), (u8, su) = _e4m3(wg), _e4m3(wu)

    def clip(a):
        p = torch.zeros_like(a, requires_grad=True)
        p.grad = a
        return clip_grad_norm_([p], 1.0)

    for f in (lambda a: add_rms_norm(a, r, w), lambda a: add_rms_norm_e4m3(a, None, w),
              lambda a: gated_linear(a, wg, wu), lambda a: gated_linear_e4m3(q, sx, g8, sg, u8, su),
              clip):
        for trace in (lambda: torch.jit.trace(f, (x,), check_trace=False), lambda: make_fx(f)(x),
                      lambda: make_fx(f, tracing_mode="fake")(x)):
            with pytest.raises(_lib.LmceError, match="traced"):
                trace()
    # the backward alone
    a = x.clone().requires_grad_(True)
    for out in (add_rms_norm(a, r, w)[0], gated_linear(a, wg, wu)):
        with pytest.raises(_lib.LmceError, match="traced"):
            make_fx(lambda d: torch.autograd.grad(out, a, d))(torch.ones_like(out))
    # torch.compile leaves these calls to run as they are
    f = torch.compile(lambda a: add_rms_norm(a * 2, r, w)[0], backend="eager")
    assert torch.equal(f(x), add_rms_norm(x * 2, r, w)[0])


def test_modes_that_watch_see_the_same_results(cuda_device):
    from torch.utils.flop_counter import FlopCounterMode

    x, r, w, wg, wu = _inputs(cuda_device)
    a = x.clone().requires_grad_(True)

    def step():
        y, s = add_rms_norm(a, r, w)
        h = gated_linear(y, wg, wu)
        return (h.detach(), *torch.autograd.grad(h.float().sum() + s.float().sum(), a))

    want = step()
    with FlopCounterMode(display=False):
        got = step()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_tensors_without_memory_are_refused(cuda_device):
    """Their null pointer must not read as an argument that was left out."""
    x, r, w, wg, wu = _inputs(cuda_device)
    zeros = torch._efficientzerotensor(x.shape, device=cuda_device, dtype=x.dtype)
    inside = torch.func.functionalize
    for call in (lambda: add_rms_norm(x, zeros, w), lambda: add_rms_norm_e4m3(x, zeros, w),
                 lambda: gated_linear(zeros, wg, wu), lambda: inside(lambda t: add_rms_norm(x, t, w)[1])(r),
                 lambda: inside(lambda t: gated_linear(t, wg, wu))(x)):
        with pytest.raises(_lib.LmceError, match="no memory") as e:
            call()
        assert e.value.code == _lib.LMCE_ERR_UNSUPPORTED
    for n in (0, 4):  # an empty tensor has a null pointer too
        assert add_rms_norm(x[:n], x[:n], w)[1].shape == (n, 128)


def test_clipping_is_an_in_place_change(cuda_device):
    """Of every gradient, through either path, as torch's own; measuring alone is none."""
    def param(n, strided=False):
        p = torch.zeros(n, n, device=cuda_device, requires_grad=True)
        g = torch.ones(n, n, device=cuda_device)
        p.grad = g.t().contiguous().t() if strided else g
        return p

    for strided in (False, True):
        params = [param(3), param(5, strided)]
        versions = lambda: [p.grad._version for p in params]  # noqa: E731
        before = versions()
        clip_grad_norm_(params, float("inf"))
        assert versions() == before
        leaf = torch.ones(5, 5, device=cuda_device, requires_grad=True)
        kept = (leaf * params[1].grad).sum()  # its backward needs the gradient as it was
        clip_grad_norm_(params, 1.0)
        assert all(a > b for a, b in zip(versions(), before))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
    with torch.inference_mode():
        p = param(4)
        clip_grad_norm_([p], 1.0)
        assert abs(p.grad.norm().item() - 1.0) < 1e-5


def _strided(t):
    if t.dim() >= 2:
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)
    return t.repeat_interleave(2)[::2] if t.dim() == 1 else t


def _unaligned(t):
    out = torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)[1:].view(t.shape)
    return out.copy_(t)


@pytest.mark.parametrize("residual", [True, False])
def test_hooks_of_saved_tensors(cuda_device, residual):
    """A hook may give back other strides; another device, type or size is refused before any launch."""
    x, r, w, wg, wu = (t.requires_grad_(True) for t in _inputs(cuda_device, n=40, h=256, f=192))
    g = torch.Generator(device=cuda_device).manual_seed(12)
    dh = torch.randn(2, 20, 192, device=cuda_device, generator=g).half()
    leaves = (x, w, wg, wu) + ((r,) if residual else ())

    def graph():
        y, s = add_rms_norm(x.view(2, 20, 256), r.view(2, 20, 256) if residual else None, w)
        return (gated_linear(y, wg, wu).float() * dh).sum() + s.float().sum()

    want = torch.autograd.grad(graph(), leaves)
    hooks = torch.autograd.graph.saved_tensors_hooks
    for unpack in (_strided, _unaligned, lambda t: t.clone()):
        with hooks(lambda t: t, unpack):
            loss = graph()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))

    def only(op):  # the operator's own saved tensors
        for unpack in (lambda t: t.cpu(), lambda t: t.to(torch.float64), lambda t: t[:1], lambda t: t.flatten()[:-1]):
            with hooks(lambda t: t, unpack):
                out = op()
            with pytest.raises(_lib.LmceError, match="came back") as e:
                torch.autograd.grad(out, x, torch.ones_like(out))
            assert e.value.code == _lib.LMCE_ERR_INVALID_ARGUMENT

    only(lambda: add_rms_norm(x, r if residual else None, w)[0])
    only(lambda: gated_linear(x, wg, wu))


def test_inputs_of_any_alignment_without_a_residual(cuda_device):
    x, r, w, wg, wu = _inputs(cuda_device, n=24, h=520)
    wide = torch.zeros(24, 600, device=cuda_device, dtype=x.dtype)
    wide[:, 3:523] = x
    others = (_unaligned(x), wide[:, 3:523], _strided(x))
    assert others[0].data_ptr() % 16 == 2
    for res, other in ((None, None), (r, _unaligned(r))):
        want, want8 = add_rms_norm(x, res, w), add_rms_norm_e4m3(x, res, w)
        for t in others:
            for got, ref in ((add_rms_norm(t, other, _unaligned(w)), want),
                             (add_rms_norm_e4m3(t, other, _unaligned(w)), want8)):
                assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, ref))


def test_e4m3_operands_that_require_a_gradient(cuda_device):
    x, r, w, wg, wu = _inputs(cuda_device)
    args = [*_e4m3(x), *_e4m3(wg), *_e4m3(wu)]
    want = gated_linear_e4m3(*args)
    for i in range(6):
        wanting = args[:i] + [torch.nn.Parameter(args[i])] + args[i + 1:]
        assert wanting[i].requires_grad
        with pytest.raises(_lib.LmceError, match="no backward") as e:
            gated_linear_e4m3(*wanting)
        assert e.value.code == _lib.LMCE_ERR_UNSUPPORTED
        with torch.no_grad():
            assert torch.equal(gated_linear_e4m3(*wanting), want)
    frozen = [torch.nn.Parameter(t, requires_grad=False) for t in args]
    assert torch.equal(gated_linear_e4m3(*frozen), want)


def test_clipping_says_what_the_library_refuses(cuda_device):
    empty = torch.zeros(0, device=cuda_device)
    params = [torch.zeros(0, device=cuda_device, requires_grad=True) for _ in range(2 ** 20 + 1)]
    for p in params:
        p.grad = empty
    with pytest.raises(_lib.LmceError, match=r"1048577 gradients \(need 1 to 2\^20\)"):
        clip_grad_norm_(params, 1.0)
    assert clip_grad_norm_(params[:-1], 1.0).item() == 0.0
    p = torch.zeros(4, device=cuda_device, requires_grad=True)
    p.grad = torch._efficientzerotensor((4,), device=cuda_device)
    with pytest.raises(_lib.LmceError, match="null"):
        clip_grad_norm_([p], 1.0)
    flat = torch.ones(100, device=cuda_device)
    a, b = (torch.zeros(60, device=cuda_device, requires_grad=True) for _ in range(2))
    a.grad, b.grad = flat[:60], flat[40:]
    for check in (False, True):
        with pytest.raises(_lib.LmceError, match="overlap"):
            clip_grad_norm_([a, b], 0.1, error_if_nonfinite=check)
    assert (flat == 1).all()


def test_debug_mode_waits_and_raises_what_a_kernel_recorded(cuda_device, monkeypatch):
    """With LMCE_DEBUG the call that runs behind the failing kernel raises, on any stream. The kernel here
    is a bounded wait that nothing satisfies."""
    x, r, w, wg, wu = _inputs(cuda_device)
    x.requires_grad_(True)
    e4m3 = [*_e4m3(x.detach()), *_e4m3(wg), *_e4m3(wu)]
    dh = torch.ones(4, 64, device=cuda_device, dtype=x.dtype)
    monkeypatch.setenv("LMCE_DEBUG", "1")
    _lib.device_error(reset=True)
    out = gated_linear(x, wg, wu)
    torch.autograd.grad(out, x, dh, retain_graph=True)
    gated_linear_e4m3(*e4m3)  # all kernels are loaded now
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        for call in (lambda: gated_linear(x, wg, wu), lambda: gated_linear_e4m3(*e4m3)):
            with torch.cuda.stream(stream):
                _lib.call("lmce_selftest_wait_timeout", 200_000_000, stream.cuda_stream)
                with pytest.raises(_lib.LmceError, match="reported by a kernel") as e:
                    call()
                assert e.value.code == _lib.LMCE_ERR_TIMEOUT
            torch.cuda.synchronize()
            assert _lib.device_error() == 0  # raised once
    _lib.call("lmce_selftest_wait_timeout", 200_000_000, torch.cuda.current_stream().cuda_stream)
    with pytest.raises(_lib.LmceError, match="reported by a kernel") as e:
        torch.autograd.grad(out, x, dh, retain_graph=True)
    assert e.value.code == _lib.LMCE_ERR_TIMEOUT
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.no_grad(), torch.cuda.graph(graph):
        captured = gated_linear(x, wg, wu)
    graph.replay()
    assert torch.equal(captured, out)
    for off in ("0", ""):
        monkeypatch.setenv("LMCE_DEBUG", off)
        _lib.call("lmce_selftest_wait_timeout", 1_000_000, torch.cuda.current_stream().cuda_stream)
        torch.autograd.grad(gated_linear(x, wg, wu), x, dh)
        torch.cuda.synchronize()
        assert _lib.device_error(reset=True) == _lib.LMCE_ERR_TIMEOUT


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_another_device_is_current():
    """Tensors of one device while another is current: forward, backward and clipping run where the
    tensors are, on that device's current stream."""
    def run(dev):
        x, r, w, wg, wu = (t.requires_grad_(True) for t in _inputs(dev, n=300, h=256, f=192))
        y, s = add_rms_norm(x, r, w)
        h = gated_linear(y, wg, wu)
        (h.float().square().sum() + s.float().sum()).backward()
        total = clip_grad_norm_([x, r, w, wg, wu], 1.0)
        with torch.no_grad():
            q, scale, _ = add_rms_norm_e4m3(x, r, w)
            h8 = gated_linear_e4m3(q, scale, *_e4m3(wg), *_e4m3(wu))
        return [t.detach().float().cpu() for t in (y, s, h, x.grad, wg.grad, total, q, scale, h8)]

    with torch.cuda.device(0):
        want = run(torch.device("cuda", 0))
        got = run(torch.device("cuda", 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
