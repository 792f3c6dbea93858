"""GPU: the operators around the head together, as a program uses them: a training step (residual
norms, gated projection, final norm with packing, head, backward, clipping) against autograd in 64
bits, the serving chain on e4m3, the refusals that need tensors on a device, and sizes whose
offsets pass 32 bits."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from rus_b200 import (_lib, add_rms_norm, add_rms_norm_e4m3, chunked_lm_head, clip_grad_norm_, gated_linear,
                      gated_linear_e4m3)
from rus_b200.packing import rms_norm_pack, shift_and_pack
from rus_b200.tied import TiedGradSlot, tied_embedding

pytestmark = pytest.mark.gpu

B, S, H, FF, V, LAYERS = 2, 150, 256, 704, 5000, 2


def _model(dev, dtype):
    g = torch.Generator(device=dev).manual_seed(21)
    r = lambda *s, scale: (torch.randn(*s, device=dev, generator=g) * scale).to(dtype)  # noqa: E731
    p = {"emb": r(V, H, scale=0.5)}
    for i in range(LAYERS):
        p[f"norm{i}"] = (1 + 0.1 * torch.randn(H, device=dev, generator=g)).to(dtype)
        p[f"gate{i}"], p[f"up{i}"] = r(FF, H, scale=1.5 * H ** -0.5), r(FF, H, scale=H ** -0.5)
        p[f"down{i}"] = r(H, FF, scale=FF ** -0.5)
    p["final"] = (1 + 0.1 * torch.randn(H, device=dev, generator=g)).to(dtype)
    ids = torch.randint(0, V, (B, S), device=dev, generator=g)
    labels = ids.clone()
    labels[:, :20] = -100
    mask = torch.ones(B, S, dtype=torch.long, device=dev)
    mask[1, 100:] = 0
    labels[1, 100:] = -100
    return p, ids, labels, mask


def _ours(p, ids, labels, mask):
    packed = shift_and_pack(labels, mask)
    slot = TiedGradSlot()
    x, s = tied_embedding(ids, p["emb"], slot), None
    for i in range(LAYERS):
        y, s = add_rms_norm(x, s, p[f"norm{i}"])
        x = F.linear(gated_linear(y, p[f"gate{i}"], p[f"up{i}"]), p[f"down{i}"])
    hidden = rms_norm_pack(x + s, p["final"], packed)
    return chunked_lm_head(hidden, packed.shift_labels, p["emb"], None, None, slot)[0]


def _reference(p, ids, labels, mask):
    norm = lambda v, w: v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
    s = p["emb"][ids]
    for i in range(LAYERS):
        y = norm(s, p[f"norm{i}"])
        s = s + (F.silu(y @ p[f"gate{i}"].T) * (y @ p[f"up{i}"].T)) @ p[f"down{i}"].T
    logits = norm(s, p["final"])[:, :-1].reshape(-1, H) @ p["emb"].T
    target = labels[:, 1:].reshape(-1)
    return F.cross_entropy(logits, target, ignore_index=-100, reduction="sum") / (target != -100).sum()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_training_step(cuda_device, dtype):
    p, ids, labels, mask = _model(cuda_device, dtype)
    trained = [k for k in p if k != "final"]  # rms_norm_pack takes a frozen weight
    for k in trained:
        p[k].requires_grad_(True)
    loss = _ours(p, ids, labels, mask)
    scale = 2.0 ** 10 if dtype == torch.float16 else 1.0  # loss scaling, as fp16 training has it
    (loss * scale).backward()
    ref = {k: v.detach().double().requires_grad_(k in trained) for k, v in p.items()}
    want = _reference(ref, ids, labels, mask)
    (want * scale).backward()
    # About 12 roundings of activations and gradients to the type lie between the embedding and
    # the loss and as many on the way back, independent ones of eps / 2 at most (rms eps / 3.5):
    # sqrt(24) * eps / 3.5 = 1.4 eps of a gradient; 4 eps is allowed.
    eps = torch.finfo(dtype).eps
    assert abs(loss.item() - want.item()) <= 4 * eps * want.item()
    for k in trained:
        err = (p[k].grad.double() - ref[k].grad).norm() / ref[k].grad.norm()
        assert err <= 4 * eps, f"{k}: {err:.3g}"
    params = [p[k] for k in trained]
    before = [q.grad.double() for q in params]
    norm = sum(float(b.square().sum()) for b in before) ** 0.5
    total = clip_grad_norm_(params, 0.1 * norm)
    assert abs(total.item() - norm) <= norm * 2 ** -20
    for q, b in zip(params, before):
        # fp16 gradients below 2^-14 keep a step of 2^-24
        assert ((q.grad.double() - 0.1 * b).abs() <= 0.1 * b.abs() * (eps / 2 + 2 ** -16) + 2.0 ** -25).all()
    assert _lib.device_error() == 0


def test_checkpointed_block_gives_the_same_gradients(cuda_device):
    from torch.utils.checkpoint import checkpoint

    p, ids, *_ = _model(cuda_device, torch.bfloat16)
    s0 = p["emb"][ids].detach()
    leaves = [p[k] for k in ("norm0", "gate0", "up0")]

    def block(s):
        y, s = add_rms_norm(s, s, leaves[0])
        return gated_linear(y, *leaves[1:]), s

    grads = []
    for wrap in (lambda s: block(s), lambda s: checkpoint(block, s, use_reentrant=False)):
        s = s0.clone().requires_grad_(True)
        for t in leaves:
            t.grad = None
            t.requires_grad_(True)
        h, t = wrap(s)
        (h.sum() + t.sum()).backward()
        grads.append([s.grad] + [t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_autograd_modes(cuda_device):
    """Anomaly detection, offloaded saved tensors, inference mode, a retained graph, memory that is
    given back, and an output changed in place before the backward."""
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x, r = (torch.randn(300, 256, device=cuda_device, generator=g).half().requires_grad_(True) for _ in range(2))
    w = torch.ones(256, device=cuda_device).half().requires_grad_(True)
    wg, wu = ((torch.randn(128, 256, device=cuda_device, generator=g) / 16).half().requires_grad_(True)
              for _ in range(2))
    leaves = (x, r, w, wg, wu)

    def loss():
        y, s = add_rms_norm(x, r, w)
        return gated_linear(y, wg, wu).float().sum() + s.float().sum()

    want = torch.autograd.grad(loss(), leaves)
    with torch.autograd.detect_anomaly(check_nan=True):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss(), leaves), want))
    with torch.autograd.graph.save_on_cpu():
        value = loss()
    for retain in (True, False):
        got = torch.autograd.grad(value, leaves, retain_graph=retain)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        y, s = add_rms_norm(x, r, w)
        assert y.is_inference() and gated_linear(y, wg, wu).is_inference()
    del value, got, y, s
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        torch.autograd.grad(loss(), leaves)
        loss()  # a graph that is dropped without a backward
    assert torch.cuda.memory_allocated() <= before
    y, s = add_rms_norm(x, r, w)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("n", [1, 5, 64, 300])
def test_serving_chain_on_e4m3(cuda_device, n):
    """Residual norm into e4m3, gated projection on e4m3 weights: exactly the product of the
    values that q and scale stand for, and near the unquantised block."""
    g = torch.Generator(device=cuda_device).manual_seed(n)
    x, r = (torch.randn(n, 896, device=cuda_device, generator=g).bfloat16() for _ in range(2))
    w = (1 + 0.1 * torch.randn(896, device=cuda_device, generator=g)).bfloat16()
    weights = []
    for size in (1.5, 1.0):
        t = torch.randn(448, 896, device=cuda_device, generator=g) * size * 896 ** -0.5
        scale = t.abs().amax(1) / 448
        weights += [(t / scale[:, None]).to(torch.float8_e4m3fn), scale]
    with torch.no_grad():
        q, scale, s = add_rms_norm_e4m3(x, r, w)
        h = gated_linear_e4m3(q, scale, *weights)
        y, s2 = add_rms_norm(x, r, w)
    assert torch.equal(s, s2)
    v = q.double() * scale.double()[:, None]
    wg, wu = (weights[i].double() * weights[i + 1].double()[:, None] for i in (0, 2))
    exact = F.silu(v @ wg.T) * (v @ wu.T)
    assert (h.double() - exact).norm() <= exact.norm() * 2 ** -9 * 1.01  # one bf16 rounding
    full = F.silu(y.double() @ wg.T) * (y.double() @ wu.T)
    # e4m3 rounds by at most 2^-4, 2^-4 / sqrt(3) rms at the worst place of a binade
    assert (h.double() - full).norm() <= full.norm() * 2 ** -4


def _all_operators(dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x, r = (torch.randn(400, 256, device=dev, generator=g).bfloat16().requires_grad_(True) for _ in range(2))
    w = torch.ones(256, device=dev).bfloat16().requires_grad_(True)
    wg, wu = ((torch.randn(320, 256, device=dev, generator=g) / 16).bfloat16().requires_grad_(True) for _ in range(2))
    y, s = add_rms_norm(x, r, w)
    h = gated_linear(y, wg, wu)
    (h.float().square().sum() + s.float().sum()).backward()
    total = clip_grad_norm_([x, r, w, wg, wu], 1.0)
    with torch.no_grad():
        q, scale, _ = add_rms_norm_e4m3(x, r, w)
    return [t.detach().float() for t in (y, s, h, x.grad, r.grad, w.grad, wg.grad, wu.grad, total, q, scale)]


def test_threads_on_streams_of_their_own(cuda_device):
    from concurrent.futures import ThreadPoolExecutor

    want = [_all_operators(cuda_device, i) for i in range(4)]
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            out = [_all_operators(cuda_device, i) for _ in range(3)]
        stream.synchronize()
        return out

    with ThreadPoolExecutor(4) as pool:
        for i, runs in enumerate(pool.map(work, range(4))):
            for got in runs:
                assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
    assert _lib.device_error() == 0


def test_refusals_on_the_device(cuda_device):
    dev = cuda_device
    x, w = torch.randn(4, 128, device=dev).half(), torch.ones(128, device=dev).half()
    wg = torch.randn(64, 128, device=dev).half()
    f8 = lambda t: t.to(torch.float8_e4m3fn)  # noqa: E731
    sx, sw = torch.ones(4, device=dev), torch.ones(64, device=dev)
    calls = [
        lambda: add_rms_norm(x, x[:2], w), lambda: add_rms_norm(x, x.bfloat16(), w), lambda: add_rms_norm(x, x, w[:64]),
        lambda: add_rms_norm(x, x, w.float()), lambda: add_rms_norm(x.float(), None, w.float()),
        lambda: add_rms_norm(x[:, :100], None, w[:100]), lambda: add_rms_norm(x, x.cpu(), w),
        lambda: add_rms_norm(x, x[:1], w), lambda: add_rms_norm(x, None, w[None]),
        lambda: add_rms_norm_e4m3(x.clone().requires_grad_(True), None, w),
        lambda: gated_linear(x, wg, wg[:32]), lambda: gated_linear(x, wg, wg.bfloat16()),
        lambda: gated_linear(x, wg.cpu(), wg.cpu()), lambda: gated_linear(x[:, :64], wg, wg),
        lambda: gated_linear(x[:, :96], wg[:, :96], wg[:, :96]), lambda: gated_linear(x, wg[:32], wg[:32]),
        lambda: gated_linear(x.float(), wg.float(), wg.float()), lambda: gated_linear(x, wg, wg, "tanh"),
        lambda: gated_linear_e4m3(x, sx, wg, sw, wg, sw),
        lambda: gated_linear_e4m3(f8(x), sx[:2], f8(wg), sw, f8(wg), sw),
        lambda: gated_linear_e4m3(f8(x), sx, f8(wg), sw[:8], f8(wg), sw),
        lambda: gated_linear_e4m3(f8(x), sx.half(), f8(wg), sw, f8(wg), sw),
        lambda: gated_linear_e4m3(f8(x[:, :64]), sx, f8(wg[:, :64]), sw, f8(wg[:, :64]), sw),
        lambda: gated_linear_e4m3(f8(x), sx, f8(wg), sw, f8(wg), sw, "silu", torch.float32),
        lambda: gated_linear_e4m3(f8(x), sx.clone().requires_grad_(True), f8(wg), sw, f8(wg), sw),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(_lib.LmceError):
            call()
            pytest.fail(f"call {i} went through")
    # refused by the library itself, past the host side's checks
    wide = torch.zeros(64, (1 << 20) + 64, device=dev, dtype=torch.float16)
    with pytest.raises(_lib.LmceError, match="at most 2") as e:
        gated_linear(wide[:1], wide, wide)
    assert e.value.code == _lib.LMCE_ERR_UNSUPPORTED
    a = x.clone().requires_grad_(True)
    for out in (gated_linear(a, wg, wg), add_rms_norm(a, x, w)[0]):
        (d,) = torch.autograd.grad(out.sum(), a, retain_graph=True)
        with pytest.raises(RuntimeError, match="LMCE_ERR_UNSUPPORTED.*second"):
            torch.autograd.grad(out.sum(), a, create_graph=True)
        assert torch.equal(torch.autograd.grad(out.sum(), a)[0], d)
    p = torch.zeros(4, device=dev, requires_grad=True)
    p.grad = torch.ones(1, device=dev).expand(4)
    with pytest.raises(_lib.LmceError, match="expanded"):
        clip_grad_norm_([p], 1.0)
    p = torch.zeros(4, device=dev, dtype=torch.float64, requires_grad=True)
    p.grad = torch.ones_like(p)
    with pytest.raises(_lib.LmceError, match="float64"):
        clip_grad_norm_([p], 1.0)
    p = torch.zeros(4, 4, device=dev, requires_grad=True)
    p.grad = torch.eye(4, device=dev).to_sparse()
    with pytest.raises(_lib.LmceError, match="dense"):
        clip_grad_norm_([p], 1.0)


def test_offsets_beyond_32_bits(cuda_device):
    """Over 2^31 elements per tensor: the last rows are those of a small call on them alone."""
    n, h = 2 ** 31 // 4096 + 77, 4096
    x = torch.randn(n, h, device=cuda_device, dtype=torch.bfloat16)
    w = torch.ones(h, device=cuda_device, dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    y, s = add_rms_norm(x, x, w)
    tail = slice(n - 700, n)
    ty, ts = add_rms_norm(x[tail].clone(), x[tail].clone(), w)
    assert torch.equal(y[tail], ty) and torch.equal(s[tail], ts)
    del y, s
    q, scale, _ = add_rms_norm_e4m3(x, None, w)
    tq, tscale, _ = add_rms_norm_e4m3(x[tail].clone(), None, w)
    assert torch.equal(q[tail].float(), tq.float()) and torch.equal(scale[tail], tscale)
    del q
    p = x.requires_grad_(True)
    p.grad = torch.full_like(x, 2.0)
    total = clip_grad_norm_([p], 1.0)
    assert abs(total.item() - 2.0 * p.numel() ** 0.5) <= total.item() * 2 ** -20
    want = torch.tensor(2.0 / (2.0 * p.numel() ** 0.5), dtype=torch.bfloat16)
    assert (p.grad[tail] == want.item()).all() and (p.grad[:700] == want.item()).all()
    del p, x
    torch.cuda.empty_cache()
    n, h, f = 150_100, 64, 14400  # h and both of dg and du over 2^31 elements, 13 GB of kept products
    x = torch.randn(n, h, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    wg, wu = (torch.randn(f, h, device=cuda_device, dtype=torch.bfloat16) * h ** -0.5 for _ in range(2))
    out = gated_linear(x, wg, wu)
    assert out.numel() > 2 ** 31
    (dx,) = torch.autograd.grad(out, x, out.detach())
    first = n // 256 * 256 - 512  # a border of 256-token tiles, so that a tail call has the same tiles
    xt = x.detach()[first:].clone().requires_grad_(True)
    small = gated_linear(xt, wg, wu)
    assert torch.equal(out[first:], small)
    (dt,) = torch.autograd.grad(small, xt, small.detach())
    # the tail's dx is summed in other parts: both are one rounding away from nearly equal sums
    assert (dx[first:].double() - dt.double()).norm() <= dt.double().norm() * 2 ** -8
    assert _lib.device_error() == 0
