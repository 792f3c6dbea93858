"""GPU: residual addition with RMSNorm (rus_b200.norm) against the formula in 64 bits.

Tolerances, fixed before the first run: a rounding to the inputs' type is off by at most half
a step (eps / 2 relative); the fp32 arithmetic before it by a few units of 2^-24 of the terms
that are added, taken as 2^-20 of the sum of their magnitudes. fp16 values under 2^-14 have a
fixed step of 2^-24. s is exact: an fp32 sum of two 16-bit values rounded again to 16 bits
equals the sum rounded once (24 >= 2 * 11 + 2 significand bits)."""
from __future__ import annotations

import pytest
import torch

from rus_b200 import add_rms_norm, add_rms_norm_e4m3

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
SHAPES = [(1, 8), (1, 896), (1, 4096), (3, 264), (7, 32), (33, 1000), (64, 3584), (593, 1536), (700, 248),
          (1025, 2056), (2500, 4096), (5, 8200), (3, 16384), (700, 16384)]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def _inputs(dev, n, h, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(n, h, device=dev, generator=g).to(dtype)
    r = (torch.randn(n, h, device=dev, generator=g) * 4).to(dtype)
    w = (1 + 0.2 * torch.randn(h, device=dev, generator=g)).to(dtype)
    dy = torch.randn(n, h, device=dev, generator=g).to(dtype)
    ds = torch.randn(n, h, device=dev, generator=g).to(dtype)
    return x, r, w, dy, ds


def _reference(s, w, dy, ds, eps):
    """(y, dx, dw) in 64 bits from the held s, and the magnitudes that their errors scale with."""
    s, w, dy, ds = s.double(), w.double(), dy.double(), ds.double()
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    nrm = s * rstd
    p = dy * w
    mean = (p * nrm).mean(-1, keepdim=True)
    dx = ds + rstd * (p - nrm * mean)
    dx_mag = ds.abs() + rstd * (p.abs() + nrm.abs() * (p * nrm).abs().mean(-1, keepdim=True))
    return nrm * w, dx, dx_mag, (dy * nrm).sum(0), (dy * nrm).abs().sum(0)


def _close(got, want, tol):
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"worst excess {(err - tol).max().item():.3g}"


@pytest.mark.parametrize("n,h", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_and_gradients(cuda_device, n, h, dtype):
    x, r, w, dy, ds = _inputs(cuda_device, n, h, dtype)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = add_rms_norm(x, r, w, 1e-5)
    dx, dr, dw = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    assert y.dtype == dx.dtype == dw.dtype == dtype and torch.equal(dx, dr)
    y_ref, dx_ref, dx_mag, dw_ref, dw_mag = _reference(s.detach(), w.detach(), dy, ds, 1e-5)
    _close(y, y_ref, y_ref.abs() * (_half(dtype) + 2 ** -20) + _floor(dtype))
    _close(dx, dx_ref, dx_ref.abs() * _half(dtype) + dx_mag * 2 ** -20 + _floor(dtype))
    # a block adds up to n / 592 rows one after another before the tree of partial sums
    _close(dw, dw_ref, dw_ref.abs() * _half(dtype) + dw_mag * (n / 592 + 32) * 2 ** -24 + _floor(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_against_differences(cuda_device, dtype):
    """Directional derivatives of sum(y * dy + s * ds) by central differences in 64 bits."""
    x, r, w, dy, ds = _inputs(cuda_device, 5, 264, dtype, seed=2)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = add_rms_norm(x, r, w, 1e-6)
    dx, dw = torch.autograd.grad((y, s), (x, w), (dy, ds))
    s0, w0, dy, ds = s.detach().double(), w.detach().double(), dy.double(), ds.double()

    def f(s_, w_):
        rstd = (s_.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        return ((s_ * rstd * w_) * dy + s_ * ds).sum()

    g = torch.Generator(device=cuda_device).manual_seed(5)
    u = torch.randn(s0.shape, device=cuda_device, generator=g, dtype=torch.float64)
    v = torch.randn(w0.shape, device=cuda_device, generator=g, dtype=torch.float64)
    e = 1e-5
    for got, direction, diff in ((dx, u, (f(s0 + e * u, w0) - f(s0 - e * u, w0)) / (2 * e)),
                                 (dw, v, (f(s0, w0 + e * v) - f(s0, w0 - e * v)) / (2 * e))):
        tol = (got.double() * direction).abs().sum() * _half(dtype) + 1e-4
        assert abs((got.double() * direction).sum() - diff) <= tol


@pytest.mark.parametrize("n,h", [(1, 64), (3, 896), (300, 3584)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_without_residual_and_without_some_gradients(cuda_device, n, h, dtype):
    x, _, w, dy, ds = _inputs(cuda_device, n, h, dtype, seed=3)
    x.requires_grad_(True)
    y, s = add_rms_norm(x, None, w)  # frozen weight
    assert s is x
    (dx,) = torch.autograd.grad(y, x, dy)
    y_ref, dx_ref, mag, _, _ = _reference(x.detach(), w, dy, torch.zeros_like(dy), 1e-6)
    _close(y, y_ref, y_ref.abs() * (_half(dtype) + 2 ** -20) + _floor(dtype))
    _close(dx, dx_ref, dx_ref.abs() * _half(dtype) + mag * 2 ** -20 + _floor(dtype))
    # only s is used: the gradient passes through, the weight gets zeros
    r = x.detach().clone().requires_grad_(True)
    w.requires_grad_(True)
    _, s = add_rms_norm(x, r, w)
    dx, dr, dw = torch.autograd.grad(s, (x, r, w), ds)
    assert torch.equal(dx, ds) and torch.equal(dr, ds) and not dw.any()
    # only the weight wants a gradient
    y, _ = add_rms_norm(x.detach(), r.detach(), w)
    (dw,) = torch.autograd.grad(y, w, dy)
    held = (x.detach().float() + r.detach().float()).to(dtype)
    *_, dw_ref, dw_mag = _reference(held, w.detach(), dy, ds, 1e-6)
    _close(dw, dw_ref, dw_ref.abs() * _half(dtype) + dw_mag * 2 ** -19 + _floor(dtype))


@pytest.mark.parametrize("n,h", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_e4m3(cuda_device, n, h, dtype):
    x, r, w, dy, ds = _inputs(cuda_device, n, h, dtype, seed=4)
    r[n // 2] = -x[n // 2]  # a row whose sum is zero
    q, scale, s = add_rms_norm_e4m3(x, r, w, 1e-5)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (n,) and torch.equal(s, (x.float() + r.float()).to(dtype))
    y_ref = _reference(s, w, dy, ds, 1e-5)[0]
    top = y_ref.abs().amax(-1) / 448
    top[top == 0] = 1.0
    assert scale[n // 2] == 1 and not q[n // 2].float().any()
    _close(scale, top, top * 2 ** -20)
    # e4m3: half a step is 2^-4 relative, 2^-10 under its smallest normal value 2^-6
    _close(q.double() * scale.double()[:, None], y_ref,
           y_ref.abs() * (2 ** -4 + 2 ** -18) + top[:, None] * 2 ** -10)
    live = torch.arange(n, device=cuda_device) != n // 2
    assert (q.float().abs().amax(-1)[live] == 448).all()


@pytest.mark.parametrize("size", [1e-38, 1e-34, 1e-31, 1e-25, 1e15])
def test_e4m3_of_rows_of_any_size(cuda_device, size):
    x, r, w, dy, ds = _inputs(cuda_device, 4, 520, torch.bfloat16, seed=9)
    r = (r.float() * size).bfloat16()
    q, scale, s = add_rms_norm_e4m3(r, None, w, 1e-6)
    y_ref = _reference(s, w, dy, ds, 1e-6)[0]
    top = y_ref.abs().amax(-1) / 448
    # values of 1e-38 are under the smallest normal fp32, 2^-126, in parts: steps of 2^-149
    _close(scale, top, top * 2 ** -20 + 2.0 ** -146 * 1e3 / 448)
    _close(q.double() * scale.double()[:, None], y_ref,
           y_ref.abs() * (2 ** -4 + 2 ** -18) + top[:, None] * 2 ** -10 + 2.0 ** -145 * 1e3)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_bad_values_stay_in_their_row(cuda_device, value):
    x, r, w, dy, ds = _inputs(cuda_device, 9, 896, torch.bfloat16, seed=6)
    clean = add_rms_norm(x, r, w)
    clean8 = add_rms_norm_e4m3(x, r, w)
    r[4, 100] = value
    keep = torch.arange(9, device=cuda_device) != 4
    for got, want in zip(add_rms_norm(x, r, w) + add_rms_norm_e4m3(x, r, w), clean + clean8):
        assert torch.equal(got.float()[keep], want.float()[keep])
    y, s = add_rms_norm(x, r, w)
    assert torch.isnan(y[4, 100]) and not torch.isfinite(s[4, 100])
    q, scale, _ = add_rms_norm_e4m3(x, r, w)
    assert torch.isnan(q[4, 100].float() * scale[4])


def test_strides_alignment_and_shapes(cuda_device):
    """Transposed, sliced, expanded and 2-byte-aligned inputs give what contiguous ones give."""
    x, r, w, dy, ds = _inputs(cuda_device, 24, 520, torch.float16, seed=7)
    want = add_rms_norm(x, r, w)
    xt = x.t().contiguous().t()
    wide = torch.zeros(24, 600, device=cuda_device, dtype=torch.float16)
    wide[:, 3:523] = r
    buf = torch.zeros(521, device=cuda_device, dtype=torch.float16)
    buf[1:] = w
    assert buf[1:].data_ptr() % 16 == 2
    for got in (add_rms_norm(xt, wide[:, 3:523], buf[1:]),
                add_rms_norm(x.view(2, 3, 4, 520), r.view(2, 3, 4, 520), w)):
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(24, 520), b)
    xg = x.clone().requires_grad_(True)
    y, s = add_rms_norm(xg, r, w)
    (a,) = torch.autograd.grad((y, s), xg, (dy.t().contiguous().t(), ds[:1].expand(24, -1)), retain_graph=True)
    (b,) = torch.autograd.grad((y, s), xg, (dy, ds[:1].repeat(24, 1)))
    assert torch.equal(a, b)
    row = torch.randn(1, 520, device=cuda_device).half().requires_grad_(True)  # one row for many tokens
    y, s = add_rms_norm(x, row.expand(24, -1), w)
    (d,) = torch.autograd.grad((y, s), row, (dy, ds))
    held = (x.float() + row.detach().float()).half()
    dx_ref = _reference(held, w, dy, ds, 1e-6)[1]
    # each row's gradient is rounded, then torch adds the 24 rows in fp32 and rounds once more
    assert (d.double() - dx_ref.sum(0)).abs().max() <= dx_ref.abs().sum(0).max() * 3 * _half(torch.float16)


def test_empty(cuda_device):
    x = torch.zeros(0, 64, device=cuda_device, dtype=torch.float16, requires_grad=True)
    w = torch.ones(64, device=cuda_device, dtype=torch.float16, requires_grad=True)
    y, s = add_rms_norm(x, x.detach(), w)
    y.sum().backward()
    assert y.shape == s.shape == (0, 64) and x.grad.shape == (0, 64) and not w.grad.any()
    q, scale, s = add_rms_norm_e4m3(x.detach(), None, w.detach())
    assert q.shape == (0, 64) and scale.shape == (0,)


def test_deterministic_on_streams_and_in_a_graph(cuda_device):
    x, r, w, dy, ds = _inputs(cuda_device, 1500, 1536, torch.bfloat16, seed=8)
    for t in (x, r, w):
        t.requires_grad_(True)

    def step():
        y, s = add_rms_norm(x, r, w)
        return (y, s, *torch.autograd.grad((y, s), (x, r, w), (dy, ds)))

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = [t.detach().clone() for t in step()]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, rs, ws = x.detach().clone(), r.detach().clone(), w.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        add_rms_norm(xs, rs, ws)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y, s = add_rms_norm(xs, rs, ws)
            q, scale, _ = add_rms_norm_e4m3(xs, rs, ws)
        xs.copy_(r.detach())
        rs.copy_(x.detach())  # the sum commutes
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(s, want[1])
        q2, scale2, _ = add_rms_norm_e4m3(x.detach(), r.detach(), ws)
        assert torch.equal(q.float(), q2.float()) and torch.equal(scale, scale2)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("n,h", [(1, 8), (5, 64), (9, 896), (700, 1000), (300, 4096), (3, 16384)])
def test_e4m3_where_rows_times_weights_pass_fp32(cuda_device, n, h, residual):
    """bf16 rows and weights whose product is beyond fp32 (|s w| to 1e45) while s rstd w is not; every
    third row is an ordinary one. The sum of squares, 16384 * 2.5e31, stays within fp32."""
    x, r, w, dy, ds = _inputs(cuda_device, n, h, torch.bfloat16, seed=10)
    large = torch.arange(n, device=cuda_device) % 3 != 1
    x[large] = (x[large].float() * 1e15).bfloat16()
    r[large] = (r[large].float() * 1e15).bfloat16()
    w = (w.float() * torch.where(torch.arange(h, device=cuda_device) % 5 == 2, 1e28, 1e3)).bfloat16()
    q, scale, s = add_rms_norm_e4m3(x, r if residual else None, w, 1e-5)
    y_ref = _reference(s, w, dy, ds, 1e-5)[0]
    top = y_ref.abs().amax(-1) / 448
    assert (s.double().abs().amax() * w.double().abs().amax()) > 2.0 ** 128
    _close(scale, top, top * 2 ** -20)
    _close(q.double() * scale.double()[:, None], y_ref, y_ref.abs() * (2 ** -4 + 2 ** -18) + top[:, None] * 2 ** -10)
    assert (q.float().abs().amax(-1) == 448).all()
    y, _ = add_rms_norm(x, r if residual else None, w, 1e-5)
    _close(y, y_ref, y_ref.abs() * (_half(torch.bfloat16) + 2 ** -20))
