"""GPU: the gated projection and its backward (rus_b200.gated) against the formula in 64 bits.

Tolerances, fixed before the first run. Per element of h: half a step of the type (eps / 2) of
the value, and the fp32 products: a K-long fp32 accumulation is off by at most about
K * 2^-24 * sum |x w| in the worst case and a small multiple of sqrt(K) * 2^-24 * |x| |w| on
such inputs; 2^-18 * |x| |w| (norms) is taken for K <= 4096, for g and u each, and 2^-18 of the
values for the activation. Gradients contract dg and du rounded to the type, independent
roundings: an element of dx is off by the norm of the terms' errors times some standard
deviations; 6 norms are allowed, next to the result's own half step. e4m3 operands are exact
inputs: the tolerance is the same as for h."""
from __future__ import annotations

import pytest
import torch

from rus_b200 import _lib, gated_linear, gated_linear_e4m3

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
# tokens around the tiles' borders (32, 128, 256), one and two to three K stages, feature blocks
# that end inside a tile
SHAPES = [(1, 64, 64), (1, 1536, 512), (2, 128, 192), (31, 192, 320), (33, 896, 64), (64, 256, 1024),
          (127, 320, 448), (128, 128, 128), (129, 64, 64), (200, 448, 576), (256, 256, 256), (257, 1024, 832),
          (513, 64, 2048), (700, 1536, 640), (1000, 512, 4864), (2049, 192, 128)]


def _eps(dtype):
    return torch.finfo(dtype).eps / 2


def _act(g, kind):
    v = g if kind == "silu" else 2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)
    dv = 1.0 if kind == "silu" else 2 * (2 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * g ** 2)
    s = torch.sigmoid(v)
    return g * s, s + g * s * torch.sigmoid(-v) * dv


def _inputs(dev, n, h, f, dtype, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(n, h, device=dev, generator=gen).to(dtype)
    wg = (torch.randn(f, h, device=dev, generator=gen) * 1.5 * h ** -0.5).to(dtype)
    wu = (torch.randn(f, h, device=dev, generator=gen) * h ** -0.5).to(dtype)
    dh = torch.randn(n, f, device=dev, generator=gen).to(dtype)
    return x, wg, wu, dh


def _assert_within(got, want, tol):
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"worst ratio {(err / tol).max().item():.3g}"


def _check_h(got, x, wg, wu, kind, dtype):
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, kind)
    want = a * u
    eg = x.norm(dim=1)[:, None] * wg.norm(dim=1) * 2 ** -18
    eu = x.norm(dim=1)[:, None] * wu.norm(dim=1) * 2 ** -18
    floor = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    # |act'| <= 1.13 for both activations
    _assert_within(got, want, want.abs() * (_eps(dtype) + 2 ** -18) + 1.13 * eg * u.abs() + eu * a.abs() + 2 * eg * eu
                   + floor)
    return g, u, a, da


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("n,h,f", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward(cuda_device, n, h, f, dtype, kind):
    x, wg, wu, _ = _inputs(cuda_device, n, h, f, dtype)
    got = gated_linear(x, wg, wu, kind)
    assert got.dtype == dtype and got.shape == (n, f)
    _check_h(got, x, wg, wu, kind, dtype)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("n,h,f", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(cuda_device, n, h, f, dtype, kind):
    x, wg, wu, dh = _inputs(cuda_device, n, h, f, dtype, seed=1)
    for t in (x, wg, wu):
        t.requires_grad_(True)
    out = gated_linear(x, wg, wu, kind)
    dx, dwg, dwu = torch.autograd.grad(out, (x, wg, wu), dh)
    assert _lib.device_error() == 0
    x, wg, wu = x.detach(), wg.detach(), wu.detach()
    g, u, a, da = _check_h(out.detach(), x, wg, wu, kind, dtype)
    d = dh.double()
    dg, du = d * u * da, d * a
    xd, gd, ud = x.double(), wg.double(), wu.double()
    # What dg and du may be off by before they are contracted: their rounding (half a step of the
    # value, or of the type's smallest), the fp32 errors eg and eu of g and u (as in h) through
    # |act''| <= 0.8 and |act'| <= 1.13, and 2^-18 for the terms sig and g sig (1 - sig) v', each
    # at most 1.2, of act'. Where act' is near its zero (g = -1.28 for silu, -0.75 for gelu) the last
    # three are larger than eps / 2 of the small value.
    # That 24 bits of g and u are kept adds 2^-15 of them at most, an eighth of fp16's eps / 2: it has
    # no term of its own, the six norms below are taken without it.
    eg = xd.norm(dim=1)[:, None] * gd.norm(dim=1) * 2 ** -18
    eu = xd.norm(dim=1)[:, None] * ud.norm(dim=1) * 2 ** -18
    floor = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off_g = dg.abs() * _eps(dtype) + floor / 2 + d.abs() * (u.abs() * (0.8 * eg + 2.4 * 2 ** -18) + 1.13 * eu)
    off_u = du.abs() * _eps(dtype) + floor / 2 + d.abs() * (1.13 * eg + a.abs() * 2 ** -18)
    # the result's own half step, six norms of what the terms are off by, 2^-18 of the terms' norm
    # for the fp32 sums
    for got, want, off, terms in (
            (dx, dg @ gd + du @ ud, off_g.square() @ gd.square() + off_u.square() @ ud.square(),
             dg.square() @ gd.square() + du.square() @ ud.square()),
            (dwg, dg.T @ xd, off_g.square().T @ xd.square(), dg.square().T @ xd.square()),
            (dwu, du.T @ xd, off_u.square().T @ xd.square(), du.square().T @ xd.square())):
        assert got.dtype == dtype
        _assert_within(got, want, want.abs() * _eps(dtype) * 1.01 + 6 * off.sqrt() + 2 ** -18 * terms.sqrt() + floor)


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
def test_gradient_against_differences(cuda_device, kind):
    """Directional derivatives of sum(h * dh) by central differences in 64 bits."""
    x, wg, wu, dh = _inputs(cuda_device, 40, 128, 192, torch.float16, seed=2)
    for t in (x, wg, wu):
        t.requires_grad_(True)
    grads = torch.autograd.grad(gated_linear(x, wg, wu, kind), (x, wg, wu), dh)
    base = [t.detach().double() for t in (x, wg, wu)]

    def value(x, wg, wu):
        return (_act(x @ wg.T, kind)[0] * (x @ wu.T) * dh.double()).sum()

    gen = torch.Generator(device=cuda_device).manual_seed(3)
    for i in range(3):
        d = torch.randn(base[i].shape, device=cuda_device, generator=gen, dtype=torch.float64)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        diff = (value(*up) - value(*down)) / 2e-5
        got = grads[i].double()
        # two roundings per gradient term (its own and dg's), independent over its elements
        assert abs((got * d).sum() - diff) <= 12 * _eps(torch.float16) * (got * d).norm() + 1e-3


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("n,h,f", [(5, 128, 192), (300, 320, 704), (1500, 256, 128)])
def test_only_the_wanted_gradients(cuda_device, n, h, f, wanted):
    x, wg, wu, dh = _inputs(cuda_device, n, h, f, torch.bfloat16, seed=4)
    every = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    full = torch.autograd.grad(gated_linear(*every), every, dh)
    some = [t.clone().requires_grad_(bool(w)) for t, w in zip((x, wg, wu), wanted)]
    leaves = [t for t in some if t.requires_grad]
    got = iter(torch.autograd.grad(gated_linear(*some), leaves, dh))
    for i, w in enumerate(wanted):
        if w:
            # dx may be summed in another number of parts: two roundings of nearly equal sums
            a, b = next(got).double(), full[i].double()
            assert ((a - b).abs() <= b.abs() * 2 * _eps(torch.bfloat16) * 2 + b.abs().max() * 2 ** -14).all()


E4M3_SHAPES = [(1, 128, 64), (3, 256, 192), (64, 3584, 320), (127, 384, 448), (128, 896, 128), (129, 128, 64),
               (300, 640, 832), (700, 1536, 640)]


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("n,h,f", E4M3_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_e4m3(cuda_device, n, h, f, dtype, kind):
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    ops = []
    for rows, size in ((n, 1.0), (f, 1.5 * h ** -0.5), (f, h ** -0.5)):
        t = torch.randn(rows, h, device=cuda_device, generator=gen) * size
        scale = t.abs().amax(1) / 448
        ops += [(t / scale[:, None]).to(torch.float8_e4m3fn), scale]
    got = gated_linear_e4m3(*ops, kind, dtype)
    assert got.dtype == dtype and got.shape == (n, f)
    x, wg, wu = (ops[i].double() * ops[i + 1].double()[:, None] for i in (0, 2, 4))
    _check_h(got, x, wg, wu, kind, dtype)
    assert _lib.device_error() == 0


def test_bad_values_stay_in_their_row(cuda_device):
    for n in (6, 300):
        x, wg, wu, dh = _inputs(cuda_device, n, 256, 320, torch.float16, seed=6)
        x.requires_grad_(True)
        clean = gated_linear(x, wg, wu)
        (dclean,) = torch.autograd.grad(clean, x, dh)
        keep = torch.arange(n, device=cuda_device) != 3
        for bad in (float("nan"), float("inf")):
            y = x.detach().clone()
            y[3, 17] = bad
            y.requires_grad_(True)
            got = gated_linear(y, wg, wu)
            (d,) = torch.autograd.grad(got, y, dh)
            assert torch.equal(got[keep], clean[keep]) and torch.equal(d[keep], dclean[keep])
            assert not torch.isfinite(got[3]).all()


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
def test_far_arguments(cuda_device, kind):
    """|g| up to 40000: the activation is 0 or g there, its derivative 0 or 1, nothing is NaN."""
    h, f = 64, 64
    x = torch.zeros(9, h, device=cuda_device, dtype=torch.bfloat16)
    x[:, 0] = torch.tensor([-40000.0, -1000.0, -95.0, -20.0, 0.0, 20.0, 95.0, 1000.0, 40000.0], device=cuda_device)
    x[:, 1] = 1.0
    wg, wu = (torch.zeros(f, h, device=cuda_device, dtype=torch.bfloat16) for _ in range(2))
    wg[:, 0], wu[:, 1] = 1.0, 0.5
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    out = gated_linear(*leaves, kind)
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    g = x.detach()[:, :1].double()
    a, da = _act(g, kind)
    want = (a * 0.5).expand(-1, f)
    assert torch.isfinite(out).all() and all(torch.isfinite(t).all() for t in grads)
    _assert_within(out.detach(), want, want.abs() * (_eps(torch.bfloat16) + 2 ** -18) + 1e-8)
    dx0 = (0.5 * da * f)[:, 0]
    _assert_within(grads[0][:, 0], dx0, dx0.abs() * 2.1 * _eps(torch.bfloat16) + 1e-6)


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
def test_arguments_whose_squares_overflow(cuda_device, kind):
    x = torch.zeros(4, 64, device=cuda_device, dtype=torch.bfloat16)
    x[:, 0] = torch.tensor([-1e30, -1e20, 1e20, 1e30], device=cuda_device)
    x[:, 1] = 1.0
    wg, wu = (torch.zeros(64, 64, device=cuda_device, dtype=torch.bfloat16) for _ in range(2))
    wg[:, 0], wu[:, 1] = 1.0, 0.5
    x.requires_grad_(True)
    out = gated_linear(x, wg, wu, kind)
    (dx,) = torch.autograd.grad(out, x, torch.ones_like(out))
    want = (x.detach()[:, :1].double().clamp(min=0) * 0.5).expand(-1, 64)
    _assert_within(out.detach(), want, want * _eps(torch.bfloat16) * 1.01)
    assert torch.equal(dx[:, 0].float(), torch.tensor([0.0, 0.0, 32.0, 32.0], device=cuda_device))


def test_strides_alignment_and_leading_dimensions(cuda_device):
    x, wg, wu, dh = _inputs(cuda_device, 150, 192, 320, torch.bfloat16, seed=7)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    want = gated_linear(*leaves)
    dwant = torch.autograd.grad(want, leaves, dh)
    buf = torch.zeros(320 * 192 + 1, device=cuda_device, dtype=torch.bfloat16)
    buf[1:] = wu.flatten()
    odd = buf[1:].view(320, 192)
    assert odd.data_ptr() % 16 == 2
    other = [x.view(3, 50, 192).clone(), wg.t().contiguous().t(), odd]
    for t in other:
        t.requires_grad_(True)
    got = gated_linear(*other)
    d = torch.autograd.grad(got, other, dh.t().contiguous().t().view(3, 50, 320))
    assert got.shape == (3, 50, 320) and torch.equal(got.view(150, 320), want)
    for a, b in zip(d, dwant):
        assert torch.equal(a.reshape(b.shape), b)


def test_empty(cuda_device):
    x = torch.zeros(2, 0, 64, device=cuda_device, dtype=torch.float16, requires_grad=True)
    wg, wu = (torch.ones(128, 64, device=cuda_device, dtype=torch.float16, requires_grad=True) for _ in range(2))
    out = gated_linear(x, wg, wu)
    assert out.shape == (2, 0, 128)
    out.sum().backward()
    assert x.grad.shape == x.shape and not wg.grad.any() and not wu.grad.any()


def test_same_bits_on_streams_and_in_graphs(cuda_device):
    """Two captured graphs with a backward each, replayed in turn, and a side stream, give the
    eager call's bits (no counters, no shared workspace, fixed orders of sums)."""
    x, wg, wu, dh = _inputs(cuda_device, 693, 512, 960, torch.float16, seed=8)

    def step(x, dh):
        leaves = [x.detach().requires_grad_(True), wg.detach().requires_grad_(True), wu.detach().requires_grad_(True)]
        out = gated_linear(*leaves)
        return (out.detach(), *torch.autograd.grad(out, leaves, dh))

    want = [t.clone() for t in step(x, dh)]
    x2, dh2 = x.flip(0).contiguous(), dh.flip(0).contiguous()
    want2 = [t.clone() for t in step(x2, dh2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dh)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, ds = x.clone(), dh.clone()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(step(xs, ds))
        graphs.append(graph)
    for graph, out, (a, b), ref in zip(graphs * 2, outs * 2, [(x, dh), (x2, dh2)] * 2, [want, want2] * 2):
        xs.copy_(a)
        ds.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ref))
    assert _lib.device_error() == 0


def test_two_streams_at_once(cuda_device):
    x, wg, wu, dh = _inputs(cuda_device, 1200, 512, 1024, torch.bfloat16, seed=9)
    for t in (x, wg, wu):
        t.requires_grad_(True)

    def step():
        return torch.autograd.grad(gated_linear(x, wg, wu), (x, wg, wu), dh)

    want = [t.clone() for t in step()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    assert _lib.device_error() == 0
