"""GPU: clipping by the global gradient norm (rus_b200.clip) against 64-bit arithmetic.

Tolerances, fixed before the first run: the norm is a sum of squares that are added in fp32 by
eights and in fp64 beyond, then rounded to fp32: 2^-20 relative. A scaled gradient is off by half
a step of its type and the factor's own few units of 2^-24 (2^-20); below the type's smallest
normal value a step is smallest_normal * eps whatever the value, so half of that is added (a bf16
gradient of 1e-30 clipped to 1e-30 / 1e-6 of itself is under its smallest step, 2^-133, and
becomes zero), and the fp32 product's own, 2^-150."""
from __future__ import annotations

import math

import pytest
import torch

from rus_b200 import _lib, clip_grad_norm_

pytestmark = pytest.mark.gpu

ALL = [torch.float16, torch.bfloat16, torch.float32]


def _params(dev, sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        p = torch.zeros(n, device=dev, dtype=dtypes[i % len(dtypes)], requires_grad=True)
        p.grad = (torch.randn(p.shape, device=dev, generator=g) * scale).to(p.dtype)
        out.append(p)
    return out


def _check(params, max_norm):
    before = [p.grad.double() for p in params]
    want = math.sqrt(math.fsum(float(b.square().sum()) for b in before))
    total = clip_grad_norm_(params, max_norm)
    assert total.dtype == torch.float32 and total.shape == ()
    assert abs(total.item() - want) <= want * 2 ** -20
    k = min(1.0, max_norm / (want + 1e-6))
    for p, b in zip(params, before):
        tol = (b * k).abs() * (torch.finfo(p.dtype).eps / 2 + 2 ** -20)
        tol += torch.finfo(p.dtype).smallest_normal * torch.finfo(p.dtype).eps / 2 + 2.0 ** -150
        assert ((p.grad.double() - b * k).abs() <= tol).all()
        if k == 1.0:
            assert torch.equal(p.grad.double(), b)


@pytest.mark.parametrize("dtypes", [[d] for d in ALL] + [ALL])
@pytest.mark.parametrize("sizes", [[1], [7], [0, 5], [2047, 2048, 2049, 3], [16383, 16384, 16385, 1, 0, 40000],
                                   [3000001, 17], list(range(1, 66))])
def test_norm_and_scaling(cuda_device, sizes, dtypes):
    for max_norm in (0.25, 1e6):
        _check(_params(cuda_device, sizes, dtypes, seed=len(sizes)), max_norm)


@pytest.mark.parametrize("count", [63, 64, 65, 1023, 1024, 1025, 2500])
def test_many_tensors(cuda_device, count):
    params = _params(cuda_device, [(i * 37) % 501 for i in range(count)], ALL, seed=1)
    _check(params, 3.0)


@pytest.mark.parametrize("dtype", ALL)
def test_views_at_every_alignment_leave_their_neighbours(cuda_device, dtype):
    """Gradients packed back to back at every element offset; what lies between stays."""
    size = torch.finfo(dtype).bits // 8
    for start in range(16 // size):
        flat = torch.full((9000,), 7.0, device=cuda_device, dtype=dtype)
        params, pos = [], start
        for n in (1, 2, 3, 5, 8, 13, 4099, 31):
            p = torch.zeros(n, device=cuda_device, dtype=dtype, requires_grad=True)
            p.grad = flat[pos:pos + n]
            p.grad.normal_()
            params.append(p)
            pos += n + 1  # one element between two gradients
        inside = torch.zeros(9000, dtype=torch.bool, device=cuda_device)
        pos = start
        for p in params:
            inside[pos:pos + p.numel()] = True
            pos += p.numel() + 1
        _check(params, 0.5)
        assert (flat[~inside] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e-30, 1e-22, 3e18, 1e25])
def test_squares_beyond_fp32(cuda_device, dtype, size):
    params = _params(cuda_device, [1000, 77], [dtype], scale=size)
    _check(params, size)


def test_zero_gradients_and_zero_limit(cuda_device):
    params = _params(cuda_device, [100, 3], ALL, scale=0.0)
    assert clip_grad_norm_(params, 1.0).item() == 0.0
    params = _params(cuda_device, [100, 3, 9], ALL)
    assert clip_grad_norm_(params, 0.0).item() > 0
    assert all(not p.grad.any() for p in params)


@pytest.mark.parametrize("dtype", ALL)
def test_not_finite(cuda_device, dtype):
    for bad in (float("nan"), float("inf"), float("-inf")):
        params = _params(cuda_device, [5000, 3], [dtype], seed=4)
        params[0].grad[4321] = bad
        before = [p.grad.clone() for p in params]
        with pytest.raises(RuntimeError, match="norm is"):
            clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
        assert torch.isnan(clip_grad_norm_(params, float("inf"))) == math.isnan(bad)
        for p, b in zip(params, before):
            assert torch.equal(p.grad.nan_to_num(7.0), b.nan_to_num(7.0))
        total = clip_grad_norm_(params, 1.0)
        if math.isnan(bad):
            assert torch.isnan(total) and all(torch.isnan(p.grad).all() for p in params)
        else:
            assert total.item() == math.inf and torch.isnan(params[0].grad[4321])
            assert not params[1].grad.any() and params[0].grad.isnan().sum() == 1


def test_repeated_missing_and_strided(cuda_device):
    params = _params(cuda_device, [50, 60], ALL, seed=5)
    none = torch.zeros(4, device=cuda_device, requires_grad=True)
    ref = [p.grad.double() for p in params]
    want = math.sqrt(sum(float(r.square().sum()) for r in ref))
    total = clip_grad_norm_([params[0], none, params[1], params[0]], 1.0)  # one listed twice
    assert abs(total.item() - want) <= want * 2 ** -20
    assert (params[0].grad.double() - ref[0] / (want + 1e-6)).abs().max() <= ref[0].abs().max() / want * 2 ** -10
    p = torch.zeros(40, 30, device=cuda_device, requires_grad=True)
    wide = torch.randn(30, 80, device=cuda_device)
    p.grad = wide[:, ::2].t()  # neither contiguous nor dense
    left = wide[:, 1::2].clone()
    _check([p], 2.0)
    assert torch.equal(wide[:, 1::2], left)
    assert clip_grad_norm_([none], 1.0).item() == 0.0
    before = p.grad.double().norm().item()  # the strided one listed twice, and with an empty one
    empty = torch.zeros(0, device=cuda_device, requires_grad=True)
    empty.grad = torch.zeros_like(empty)
    total = clip_grad_norm_([p, empty, p, empty], 0.5, error_if_nonfinite=True)
    assert abs(total.item() - before) <= before * 2 ** -20
    assert abs(p.grad.double().norm().item() - 0.5) <= 0.5 * 2 ** -10
    other = torch.zeros(40, 30, device=cuda_device, requires_grad=True)
    other.grad = p.grad
    with pytest.raises(_lib.LmceError, match="overlap"):
        clip_grad_norm_([p, other], 0.1)
    total = clip_grad_norm_(params[1], 1e9)  # a single tensor
    assert total.item() > 0


def test_overlapping_gradients_are_refused(cuda_device):
    flat = torch.randn(100, device=cuda_device)
    a, b = (torch.zeros(60, device=cuda_device, requires_grad=True) for _ in range(2))
    a.grad, b.grad = flat[:60], flat[40:]
    before = flat.clone()
    with pytest.raises(_lib.LmceError, match="overlap"):
        clip_grad_norm_([a, b], 0.1)
    assert torch.equal(flat, before)


def test_same_bits_on_a_stream_and_in_a_graph(cuda_device):
    def fresh():
        return _params(cuda_device, [100003, 4, 65537, 0, 12], ALL, seed=6)

    want = fresh()
    norm = clip_grad_norm_(want, 1.5)
    got = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n2 = clip_grad_norm_(got, 1.5)
    side.synchronize()
    assert torch.equal(norm, n2) and all(torch.equal(a.grad, b.grad) for a, b in zip(got, want))
    held = fresh()
    graphs, outs = [], []
    for limit in (1.5, 0.5):  # two graphs over the same gradients, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(clip_grad_norm_(held, limit))
        graphs.append(graph)
    for p, f in zip(held, fresh()):
        p.grad.copy_(f.grad)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], norm) and all(torch.equal(a.grad, b.grad) for a, b in zip(held, want))
    graphs[1].replay()
    torch.cuda.synchronize()
    assert abs(outs[1].item() - 1.5) <= 1.5 * 2 ** -7  # what the first left: 1.5 up to the gradients' rounding
