"""Distillation from a teacher's top logits (``ops.distill``) against the formulas in 64 bits.

Tolerances.  log-sum-exp: a thread adds up to 200 terms one after another, then 29 joins, each 2^-24, and
ex2 is good to 2^-22: below 1.5e-5 in the sum, so in its logarithm (LSE).  A probability: that, and 2^-22
for each unit of its exponent.  The loss: LSE and 2e-6 of the sizes of the terms p (|log p| + |log q| + 1).
A gradient: one rounding (``finfo.eps / 2``), the probabilities' errors with their factors, four roundings of
2^-24 of the factors themselves; where a gradient formed with the loss meets an incoming factor, a second
rounding of the type."""
import math

import pytest
import torch

from my_muon_fsdp2_b200.ops.distill import distillation_loss, fused_linear_distillation

LSE = 1.5e-5
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(N, V, K, dtype=torch.float32, device="cpu", seed=0, teacher_dtype=torch.float32, id_dtype=torch.int64, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(N, V, generator=g) * scale
    ids = torch.randint(0, V, (N, K), generator=g)  # ids may come up twice
    a = torch.randn(N, K, generator=g) * 2 + 3
    z.scatter_(1, ids, a)
    a = a + torch.randn(N, K, generator=g)
    y = torch.randint(0, V, (N,), generator=g)
    for n in range(N):
        if n % 5 == 1:
            ids[n, (K + 1) // 2:] = -1  # fewer slots
        if n % 5 == 2:
            ids[n] = -1  # none, by id
        if n % 7 == 3:
            a[n] = -math.inf  # none, by value
        if n % 4 == 3:
            y[n] = -100
        if n % 6 == 0:
            y[n] = max(0, int(ids[n, 0]))  # the target is a slot too
        if n % 11 == 4:
            a[n, 0] = -math.inf
            free = [v for v in range(min(V, 3 * K + 9)) if v not in ids[n].tolist() and v != int(y[n])]
            z[n, free[:2]] = -math.inf  # words that the student rules out
    return z.to(device, dtype), ids.to(device, id_dtype), a.to(device, teacher_dtype), y.to(device)


def _formula(z, ids, a, y, tau, alpha, mean, up=1.0):
    """(loss, its tolerance, gradient, its error but for the last rounding), 64 bits."""
    z, a, ids = z.detach().double(), a.double(), ids.long()
    N, V = z.shape
    slot = (ids >= 0) & (a != -math.inf)
    has = slot.any(1)
    hard = torch.zeros_like(has) if y is None else y != -100
    wk = alpha / max(1, int(has.sum())) if mean else alpha
    wc = (1 - alpha) / max(1, int(hard.sum())) if mean else 1 - alpha
    p = torch.zeros_like(a)
    p[has] = torch.softmax((a[has] / tau).masked_fill(~slot[has], -math.inf), 1)
    dense = torch.zeros_like(z)
    live = (has & (alpha > 0)) | (hard & (alpha < 1))
    zs = torch.where(live[:, None], z, 0.0)
    lq, l1 = torch.log_softmax(zs / tau, 1), torch.log_softmax(zs, 1)
    gather = lq.gather(1, ids.clamp_min(0))
    terms = torch.where(p > 0, p * (p.clamp_min(1e-300).log() - gather), 0.0)
    sizes = torch.where(p > 0, p * (p.clamp_min(1e-300).log().abs() + gather.abs() + 1), 0.0)
    kd, kd_tol = tau**2 * terms.sum(1), tau**2 * (LSE + 2e-6 * sizes.sum(1))
    yt = torch.zeros(N, dtype=torch.long, device=z.device) if y is None else y.clamp_min(0)
    lh = l1.gather(1, yt[:, None])[:, 0]
    ce, ce_tol = torch.where(hard, -lh, 0.0), torch.where(hard, LSE + 2e-6 * lh.abs(), 0.0)
    if alpha == 0:
        kd, kd_tol = kd * 0, kd_tol * 0
    rows, tol = wk * torch.where(has, kd, 0.0) + wc * ce, wk * kd_tol + wc * ce_tol
    if mean:
        rows, tol = rows.sum(), tol.sum()
    upr = up[:, None].double() if isinstance(up, torch.Tensor) and up.dim() else up
    k, c = upr * wk * tau * has[:, None].double(), upr * wc * hard[:, None].double()
    q, q1 = lq.exp(), l1.exp()
    grad = k * q + c * q1
    err = (abs(k) * q * (LSE + 2e-6 * lq.abs().clamp_max(200)) + abs(c) * q1 * (LSE + 2e-6 * l1.abs().clamp_max(200)))
    grad.scatter_add_(1, ids.clamp_min(0), -k * p)
    err.scatter_add_(1, ids.clamp_min(0), abs(k) * p * 2e-6)
    grad.scatter_add_(1, yt[:, None], -c)
    # the target's own -c: (1 - alpha) * fl(1 / count) * up and the subtraction are four roundings of 2^-24
    err.scatter_add_(1, yt[:, None], abs(c) * 4 * 2**-24)
    return rows, tol, torch.where(live[:, None], grad, dense), torch.where(live[:, None], err, 0.0) + 1e-37


def _check(z, ids, a, y, tau, alpha, reduction, factor=1.0):
    z = z.detach().requires_grad_()
    mean = reduction == "mean"
    loss = distillation_loss(z, ids, a, y, temperature=tau, alpha=alpha, reduction=reduction)
    up = torch.tensor(factor, device=z.device) if mean else (torch.rand(z.shape[0], device=z.device) + 0.5) * factor
    (g,) = torch.autograd.grad(loss, z, up)
    assert loss.dtype == torch.float32 and g.dtype == z.dtype and g.shape == z.shape
    with torch.no_grad():
        alone = distillation_loss(z, ids, a, y, temperature=tau, alpha=alpha, reduction=reduction)
    assert torch.equal(alone, loss.detach())
    want, tol, wg, eg = _formula(z, ids, a, y, tau, alpha, mean, factor if mean else up)
    same = (loss.double() == want) | ((loss.double() - want).abs() <= tol + 2**-24 * want.abs())
    assert bool(same.all()), f"loss off by {((loss.double() - want).abs() / tol).max().item():.3g} tolerances"
    f = torch.finfo(z.dtype)
    # formed with the loss (not for fp16), then multiplied by the factor: a second rounding of the type
    steps = 2 if mean and z.dtype != torch.float16 and factor != 1.0 else 1
    off = (g.double() - wg).abs()
    tol = eg + steps * f.eps / 2 * (1 + f.eps) * wg.abs() + f.smallest_normal * f.eps * (1 + abs(factor) * (steps - 1))
    worst = (off / tol).max().item()
    assert worst <= 1, f"gradient off by {worst:.3g} tolerances"


# ---------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.5), (0.7, 0.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_cpu_against_formula_and_differences(tau, alpha, reduction):
    z, ids, a, y = _inputs(12, 9, 3)
    _check(z, ids, a, y, tau, alpha, reduction, factor=2.0)
    z = torch.randn(5, 7, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).requires_grad_()
    assert torch.autograd.gradcheck(
        lambda v: distillation_loss(v, ids[:5] % 7 * (ids[:5] >= 0) - (ids[:5] < 0).long(), a[:5].double(),
                                    y[:5].clamp_max(6), temperature=tau, alpha=alpha, reduction=reduction), (z,))


def test_alpha_zero_is_cross_entropy_and_same_teacher_gives_zero():
    z, ids, a, y = _inputs(6, 11, 4)
    ce = torch.nn.functional.cross_entropy(z, y, ignore_index=-100)
    assert torch.allclose(distillation_loss(z, ids, a, y, alpha=0.0), ce, atol=1e-6)
    every = torch.arange(11).expand(6, 11)
    zero = distillation_loss(z, every, z, temperature=3.0)
    assert abs(zero.item()) < 1e-5


def test_masked_rows_take_no_part_on_cpu():
    z, ids, a, y = _inputs(8, 10, 3)
    ids[4], y[4], z[4] = -1, -100, math.nan
    a[5, 1], ids[5, 1] = math.nan, -1  # what an empty slot holds does not matter
    z.requires_grad_()
    loss = distillation_loss(z, ids, a, y, alpha=0.5)
    (g,) = torch.autograd.grad(loss, z)
    assert torch.isfinite(loss) and torch.isfinite(g).all() and not g[4].any()
    none = torch.full_like(ids, -1)
    assert distillation_loss(z, none, a, reduction="mean").item() == 0.0


def test_fused_linear_on_cpu_is_the_composition():
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(2, 6, 5, generator=g, dtype=torch.float64), torch.randn(11, 5, generator=g, dtype=torch.float64)
    _, ids, a, y = _inputs(12, 11, 3)
    args = (ids.view(2, 6, 3), a.view(2, 6, 3), y.view(2, 6))
    got = fused_linear_distillation(x, w, *args, temperature=2.0, alpha=0.3)
    assert torch.allclose(got, distillation_loss(x @ w.t(), *args, temperature=2.0, alpha=0.3))


def test_refusals():
    z, ids, a, y = _inputs(4, 9, 3)
    f = distillation_loss
    for bad in (lambda: f(z, ids[:3], a), lambda: f(z, ids, a[:, :2]), lambda: f(z, ids, a, y[:3]), lambda: f(z, ids, a, alpha=0.5),
                lambda: f(z, ids, a, temperature=0.0), lambda: f(z, ids, a, temperature=math.nan), lambda: f(z, ids, a, temperature=1e4), lambda: f(z, ids, a, y, alpha=1.5),
                lambda: f(z, ids, a, y, alpha=math.nan), lambda: f(z, ids, a, reduction="sum"), lambda: f(z, ids[:, :0], a[:, :0]),
                lambda: f(z, ids.repeat(1, 400), a.repeat(1, 400)), lambda: f(z[:, :0], ids, a), lambda: f(z, ids + 9, a),
                lambda: f(z, ids, a, y.clamp_min(0) + 9, alpha=0.5), lambda: f(z, ids, a.clone().requires_grad_()),
                lambda: f(z.view(2, 2, 9), ids, a), lambda: f(z.sum(), ids, a)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(z.long(), ids, a), lambda: f(z, ids.float(), a), lambda: f(z, ids, a.long()), lambda: f(z, ids, a, y.int(), alpha=0.5)):
        with pytest.raises(TypeError):
            bad()
    x, w = torch.zeros(4, 5), torch.zeros(9, 5)
    for bad in (lambda: fused_linear_distillation(x, w[:, :4], ids, a), lambda: fused_linear_distillation(x, w.half(), ids, a),
                lambda: fused_linear_distillation(x, w, ids[:2], a[:2]), lambda: fused_linear_distillation(x, w, ids, a, chunk=0)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------------- GPU
SETTINGS = [(1.0, 1.0, "mean"), (1.0, 0.5, "none"), (2.0, 0.5, "mean"), (1.7, 0.25, "none"), (0.5, 1.0, "mean"), (3.0, 0.0, "none")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (3, 5, 2), (13, 17, 7), (9, 1000, 64), (25, 1003, 300), (300, 2049, 8), (6, 50257, 16),
                                   (40, 32001, 33), (5, 128256, 64), (3, 200001, 1024)], ids=str)
def test_gpu_against_formula(N, V, K, dtype):
    for n, (tau, alpha, reduction) in enumerate(SETTINGS):
        z, ids, a, y = _inputs(N, V, K, dtype, "cuda", seed=n)
        factor = 1024.0 if dtype == torch.float16 else (1.0 if n % 2 else 3.0)  # a loss scale for fp16
        _check(z, ids, a, y if alpha < 1 else None, tau, alpha, reduction, factor)


@pytest.mark.gpu
def test_gpu_types_of_the_teacher_and_extremes():
    for td in DTYPES:
        for it in (torch.int32, torch.int64):
            _check(*_inputs(9, 777, 12, torch.bfloat16, "cuda", teacher_dtype=td, id_dtype=it), 2.0, 0.5, "mean")
    # far apart, shifted by a constant, and the type's lowest value as a mask
    z, ids, a, y = _inputs(8, 4000, 6, torch.float32, "cuda", scale=30.0)
    _check(z, ids, a, y, 1.0, 0.5, "none")
    z[:, 100:] = torch.where(torch.rand(8, 3900, device="cuda") < 0.5, torch.finfo(torch.float32).min, z[:, 100:])
    keep = z.gather(1, ids.clamp_min(0)) > -1e30
    ids = torch.where(keep, ids, -1)
    y = torch.where((y >= 0) & (z.gather(1, y.clamp_min(0)[:, None])[:, 0] > -1e30), y, -100)
    _check(z, ids, a, y, 2.0, 0.5, "none")


@pytest.mark.gpu
def test_gpu_infinities_and_masked_rows():
    z, ids, a, y = _inputs(8, 3000, 4, torch.bfloat16, "cuda")
    ids[4], y[4], z[4] = -1, -100, math.nan
    ids[5], z[5, 7] = torch.tensor([7, -1, -1, -1], device="cuda"), -math.inf
    a[6, 1], ids[6, 1] = math.nan, -1
    z[0] = -math.inf
    z.requires_grad_()
    rows = distillation_loss(z, ids, a, y, alpha=0.5, reduction="none")
    (g,) = torch.autograd.grad(rows, z, torch.ones_like(rows))
    assert rows[4] == 0 and not g[4].any()
    assert rows[5] == math.inf and torch.isfinite(g[5]).all()
    assert rows[0].isnan() and torch.isfinite(rows[[1, 2, 3, 6, 7]]).all() and torch.isfinite(g[[1, 2, 3, 6, 7]]).all()
    none = distillation_loss(z, torch.full_like(ids, -1), a, torch.full_like(y, -100), alpha=0.5)
    assert none.item() == 0.0 and not torch.autograd.grad(none, z)[0].any()
    empty = distillation_loss(z[:0], ids[:0], a[:0], y[:0], alpha=0.5)
    assert empty.item() == 0.0 and torch.autograd.grad(empty, z)[0].shape == z.shape


@pytest.mark.gpu
def test_gpu_layouts():
    """Columns of wider rows, any offset, more dimensions, columns that are not contiguous."""
    for reduction in ("mean", "none"):
        for off, pad in ((0, 0), (1, 0), (3, 5), (8, 8), (5, 3)):
            z, ids, a, y = _inputs(10, 1009, 5, torch.bfloat16, "cuda")
            wide = torch.full((10 * (1009 + pad) + off,), math.nan, device="cuda", dtype=torch.bfloat16)
            view = wide[off:].view(10, 1009 + pad)[:, :1009]
            view.copy_(z)
            _check(view, ids, a, y, 2.0, 0.5, reduction)
            same = distillation_loss(z, ids, a, y, temperature=2.0, alpha=0.5, reduction=reduction)
            got = distillation_loss(view, ids, a, y, temperature=2.0, alpha=0.5, reduction=reduction)
            assert torch.allclose(same, got, rtol=1e-5)
        got = distillation_loss(z.view(2, 5, 1009), ids.view(2, 5, 5), a.view(2, 5, 5), y.view(2, 5), temperature=2.0, alpha=0.5,
                                reduction=reduction)
        assert torch.equal(got.reshape(same.shape), same)
        t = z.t().contiguous().t()
        assert torch.equal(distillation_loss(t, ids, a, y, temperature=2.0, alpha=0.5, reduction=reduction), same)


@pytest.mark.gpu
def test_gpu_bad_ids_and_targets_are_recorded():
    from my_muon_fsdp2_b200._ext import check_device_error

    check_device_error(0)
    z, ids, a, y = _inputs(6, 100, 3, torch.bfloat16, "cuda")
    want = distillation_loss(z, torch.where(torch.arange(3, device="cuda") == 1, -1, ids), a, y, alpha=0.5)
    bad = ids.clone()
    bad[:, 1] = 2**40
    got = distillation_loss(z, bad, a, y, alpha=0.5)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="rejected"):
        check_device_error(0)
    y2 = y.clone()
    y2[0] = 100
    distillation_loss(z, ids, a, y2, alpha=0.5)
    with pytest.raises(RuntimeError, match="rejected"):
        check_device_error(0)
    check_device_error(0)


@pytest.mark.gpu
def test_gpu_graphs_of_autograd():
    z, ids, a, y = _inputs(6, 300, 3, torch.float32, "cuda")
    z.requires_grad_()
    for reduction in ("mean", "none"):
        loss = distillation_loss(z, ids, a, y, alpha=0.5, reduction=reduction).sum()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(loss, z, create_graph=True)
    loss = distillation_loss(z, ids, a, y, alpha=0.5)
    (g,) = torch.autograd.grad(loss, z, retain_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, z)
    # two losses over the same logits, each with a factor of its own
    l1 = distillation_loss(z, ids, a, y, alpha=0.5)
    l2 = distillation_loss(z, ids, a, y, alpha=0.5)
    (h,) = torch.autograd.grad(0.25 * l1 + 0.75 * l2, z)
    assert torch.allclose(h, g, rtol=1e-6, atol=1e-12)


@pytest.mark.gpu
@pytest.mark.parametrize("reduction,dtype", [("mean", torch.bfloat16), ("none", torch.bfloat16), ("mean", torch.float16)], ids=str)
def test_gpu_same_bits_streams_and_graph(reduction, dtype):
    z, ids, a, y = _inputs(200, 5001, 9, dtype, "cuda")
    up = torch.tensor(4.0, device="cuda") if reduction == "mean" else torch.rand(200, device="cuda")

    def run():
        v = z.detach().requires_grad_()
        loss = distillation_loss(v, ids, a, y, temperature=2.0, alpha=0.5, reduction=reduction)
        return loss.detach(), torch.autograd.grad(loss, v, up)[0]

    first, again = run(), run()
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = run()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    del first, again, other
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    z.mul_(0.5)
    up.mul_(0.5)
    ids[::3] = -1
    for _ in range(2):  # a replay starts from the logits again, whatever the last one left
        g.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, run()))


@pytest.mark.gpu
def test_gpu_difference_quotient():
    z, ids, a, y = _inputs(7, 400, 5, torch.float32, "cuda")
    z[torch.isinf(z)] = -20.0
    v = torch.randn(7, 400, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    zc, args = z.double().cpu(), (ids.cpu(), a.double().cpu(), y.cpu())
    f = lambda s: float(distillation_loss(zc + s * v, *args, temperature=2.0, alpha=0.5))  # noqa: E731
    quotient = (f(1e-5) - f(-1e-5)) / 2e-5
    z.requires_grad_()
    (g,) = torch.autograd.grad(distillation_loss(z, ids, a, y, temperature=2.0, alpha=0.5), z)
    g = g.double().cpu()
    assert abs(float((g * v).sum()) - quotient) <= 2e-5 * float((g * v).abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("N,D,V,chunk", [(96, 128, 1000, 8192), (100, 128, 1003, 40), (257, 256, 5000, 64)], ids=str)
def test_gpu_fused_linear(N, D, V, chunk):
    """Against the 64-bit composition.  The logits are rounded to bf16 (half a step, 2^-9 of |z|, in each
    exponent), their gradient once more as the GEMMs' operand (2^-9), the results once; dW in one chunk
    too.  As norms: below 2^-9 (max|z| / tau + 2) of the dense part's, and 2^-8 in all for the rest."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(N, D, generator=g)).to("cuda", torch.bfloat16).requires_grad_()
    w = (torch.randn(V, D, generator=g) * 0.2).to("cuda", torch.bfloat16).requires_grad_()
    _, ids, a, y = _inputs(N, V, 8, device="cuda")
    loss = fused_linear_distillation(x, w, ids, a, y, temperature=2.0, alpha=0.5, chunk=chunk)
    gx, gw = torch.autograd.grad(loss * 2.0, (x, w), retain_graph=True)
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    z = xd @ wd.t()
    want, _, gz, _ = _formula(z, ids, a, y, 2.0, 0.5, True, 2.0)
    zmax = float(z.detach().abs().max())
    rel = 2**-9 * (zmax / 2 + 2) + 2**-8
    assert abs(loss.item() - want.item()) <= rel * abs(float(want))
    for got, ref in ((gx, gz @ wd.detach()), (gw, gz.t() @ xd.detach())):
        assert float((got.double() - ref).norm() / ref.norm()) < rel
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, x)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """More than 2^31 logits: the last rows are those of a call on them alone (but for how many blocks share
    a row there, which orders its sums)."""
    N, V = 17000, 128256
    z, ids, a, y = _inputs(5, V, 7, torch.bfloat16, "cuda")
    big = torch.zeros(N, V, device="cuda", dtype=torch.bfloat16)
    big[-5:] = z
    more = lambda t, fill: torch.cat([torch.full((N - 5,) + t.shape[1:], fill, device="cuda", dtype=t.dtype), t])  # noqa: E731
    args = (more(ids, -1), more(a, 0.0), more(y, -100))
    for reduction in ("none", "mean"):
        want = distillation_loss(z.requires_grad_(), ids, a, y, temperature=2.0, alpha=0.5, reduction=reduction)
        (wg,) = torch.autograd.grad(want.sum(), z)
        got = distillation_loss(big.requires_grad_(), *args, temperature=2.0, alpha=0.5, reduction=reduction)
        (g,) = torch.autograd.grad(got.sum(), big)
        assert torch.allclose(got[-5:] if reduction == "none" else got, want, rtol=1e-5)
        assert torch.allclose(g[-5:].float(), wg.float(), rtol=2**-7, atol=1e-12) and not g[:-5].any()
        del g


@pytest.mark.gpu
def test_gpu_refusals():
    """What the CPU form refuses before it looks at values the kernels' entry refuses in the same way."""
    z, ids, a, y = _inputs(4, 9, 3, torch.float32, "cuda")
    f = distillation_loss
    for bad in (lambda: f(z, ids[:3], a), lambda: f(z, ids, a[:, :2]), lambda: f(z, ids, a, y[:3]), lambda: f(z, ids, a, alpha=0.5),
                lambda: f(z, ids, a, temperature=0.0), lambda: f(z, ids, a, temperature=math.nan), lambda: f(z, ids, a, temperature=1e4),
                lambda: f(z, ids, a, y, alpha=1.5), lambda: f(z, ids, a, y, alpha=math.nan), lambda: f(z, ids, a, reduction="sum"),
                lambda: f(z, ids[:, :0], a[:, :0]), lambda: f(z, ids.repeat(1, 400), a.repeat(1, 400)), lambda: f(z[:, :0], ids, a),
                lambda: f(z, ids, a.clone().requires_grad_()), lambda: f(z.view(2, 2, 9), ids, a), lambda: f(z.sum(), ids, a),
                lambda: f(z, ids.cpu(), a), lambda: f(z, ids, a.cpu()), lambda: f(z, ids, a, y.cpu(), alpha=0.5)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(z.long(), ids, a), lambda: f(z.double(), ids, a), lambda: f(z, ids.float(), a), lambda: f(z, ids, a.long()),
                lambda: f(z, ids, a, y.int(), alpha=0.5)):
        with pytest.raises(TypeError):
            bad()


@pytest.mark.gpu
def test_gpu_one_word_and_more_dimensions():
    """A vocabulary of one word whose column stride means nothing, and leading dimensions that are views."""
    z = torch.randn(5, 4, device="cuda")[:, 1:2].as_strided((5, 1), (4, 3), 1)
    one = torch.zeros(5, 1, dtype=torch.long, device="cuda")
    # lse - z: R = fl(z / ln 2) and its product with ln 2 round by 2^-24 |z| each, besides the error of exp and log
    assert abs(distillation_loss(z, one, torch.zeros(5, 1, device="cuda")).item()) <= LSE + 2**-23 * z.abs().max().item()
    z, ids, a, y = _inputs(12, 300, 4, torch.float32, "cuda")
    flat = distillation_loss(z, ids, a, y, alpha=0.5, reduction="none")
    lead = lambda t: t.view(3, 4, *t.shape[1:])  # noqa: E731
    zl = lead(z).transpose(0, 1).requires_grad_()
    got = distillation_loss(zl, lead(ids).transpose(0, 1), lead(a).transpose(0, 1), lead(y).t(), alpha=0.5, reduction="none")
    assert got.shape == (4, 3) and torch.equal(got.t().reshape(12), flat)
    (g,) = torch.autograd.grad(got.sum(), zl)
    zf = z.detach().requires_grad_()
    (want,) = torch.autograd.grad(distillation_loss(zf, ids, a, y, alpha=0.5, reduction="none").sum(), zf)
    assert torch.equal(g.transpose(0, 1).reshape(12, 300), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,K", [(7, 40, 700), (4, 30001, 1000), (160, 50257, 130), (150, 20003, 257)], ids=str)
def test_gpu_many_slots_of_few_words(N, V, K, dtype):
    """Words that come up many times, in one block's slice and over several warps' slots; each number of
    blocks a row.  Equal calls give equal bits."""
    z, ids, a, y = _inputs(N, V, K, dtype, "cuda")
    some = torch.randint(0, V, (30,), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    ids = torch.where(ids >= 0, some[ids % 30], -1)
    y = torch.where(y >= 0, some[y % 30], y)
    for reduction in ("mean", "none"):
        _check(z, ids, a, y, 2.0, 0.5, reduction, 1024.0 if dtype == torch.float16 else 1.0)
        z.requires_grad_()
        runs = []
        for _ in range(3):
            loss = distillation_loss(z, ids, a, y, alpha=0.5, reduction=reduction)
            runs.append((loss.detach(), *torch.autograd.grad(loss.sum(), z)))
        z = z.detach()
        assert all(torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1]) for r in runs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tau", [1.0, 2.0, 1.7])
@pytest.mark.parametrize("value", [-1e10, 1e10, -math.inf, math.inf], ids=["-1e10", "1e10", "lowest", "highest"])
def test_gpu_rows_far_from_zero(value, tau, dtype):
    """Rows whose logits are all the same large value, the type's lowest (a mask over the whole row) or highest
    one among them, are uniform; rows beside them and the mean keep their values.  And rows of large logits
    that differ."""
    f = torch.finfo(dtype)
    value = max(f.min, min(f.max, value))
    for N, V in ((4, 301), (9, 50257)):
        z, ids, a, y = _inputs(N, V, 5, torch.float32, "cuda")
        z[torch.isinf(z)] = 0.0
        z = z.to(dtype)
        z[0::2] = value
        for reduction in ("none", "mean"):
            _check(z, ids, a, y, tau, 0.5, reduction)
            _check(z, ids, a, None, tau, 1.0, reduction)
        if abs(value) == 1e10:
            z[0::2, ::3] = value * (1 - 2**-6)
            _check(z, ids, a, y, tau, 0.5, "mean")


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [1.0, 2.0, 1.7])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_gpu_rows_around_a_large_value(sign, tau):
    """Logits a few units apart whose exponents are around 2^12 and 2^20, where the type has few steps left
    between them."""
    for N, V, size in ((5, 2003, 2**20), (9, 50257, 2**20), (5, 2003, 2**12)):
        z, ids, a, y = _inputs(N, V, 5, torch.float32, "cuda")
        z[torch.isinf(z)] = 0.0
        z = sign * size * math.log(2.0) * tau + z * torch.linspace(0.25, 4.0, N, device="cuda")[:, None]
        for reduction in ("none", "mean"):
            _check(z, ids, a, y, tau, 0.5, reduction)
            _check(z, ids, a, None, tau, 1.0, reduction)


def test_rows_far_from_zero_on_cpu():
    for value in (-1e10, torch.finfo(torch.float32).min, torch.finfo(torch.float32).max):
        z, ids, a, y = _inputs(5, 301, 4)
        z[torch.isinf(z)] = 0.0
        z[0::2] = value
        for tau in (1.0, 2.0, 1.7):
            _check(z, ids, a, y, tau, 0.5, "mean")


def _teacher_without_values(device):
    """A slot whose teacher logit is NaN or +inf makes its token's loss NaN, and no other's."""
    for bad in (math.nan, math.inf):
        for K in (4, 300):
            z, ids, a, y = _inputs(6, 1000, K, torch.float32, device)
            want = distillation_loss(z, ids, a, y, alpha=0.5, reduction="none")
            a[0, 1] = bad
            got = distillation_loss(z, ids, a, y, alpha=0.5, reduction="none")
            assert got[0].isnan() and torch.equal(got[1:], want[1:])
            assert distillation_loss(z, ids, a, y, alpha=0.5).isnan()


def test_teacher_without_values_on_cpu():
    _teacher_without_values("cpu")


@pytest.mark.gpu
def test_gpu_teacher_without_values():
    _teacher_without_values("cuda")


def _dual_logits(call, device):
    import torch.autograd.forward_ad as fw

    ids = torch.zeros(4, 2, dtype=torch.long, device=device)
    for dual in ("logits", "teacher"):
        with fw.dual_level():
            z, a = torch.ones(4, 16, device=device), torch.ones(4, 2, device=device)
            if dual == "logits":
                z = fw.make_dual(z, torch.ones_like(z))
            else:
                a = fw.make_dual(a, torch.ones_like(a))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="forward-mode|forward mode"):
                    call(z, ids, a)


def test_forward_mode_is_refused_by_the_entry():
    from my_muon_fsdp2_b200._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    _dual_logits(lambda z, ids, a: ext().distill(z, ids, a, None, 1.0, 1.0, -100, True), "cpu")


@pytest.mark.gpu
def test_gpu_forward_mode_is_refused():
    for reduction in ("mean", "none"):
        _dual_logits(lambda z, ids, a: distillation_loss(z, ids, a, reduction=reduction), "cuda")
    w = torch.ones(24, 16, device="cuda", dtype=torch.bfloat16)
    _dual_logits(lambda x, ids, a: fused_linear_distillation(x.bfloat16(), w, ids, a), "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [8192, 40])
def test_gpu_fused_linear_forms_what_is_wanted(chunk):
    """An evaluation, a frozen head and frozen inputs: the same loss, the gradients that are wanted with the same
    bits, and a GEMM launch and the memory of a gradient less for each that is not."""
    from my_muon_fsdp2_b200._ext import ext

    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(*s, generator=g).to("cuda", torch.bfloat16) for s in ((100, 128), (1003, 128)))
    _, ids, a, y = _inputs(100, 1003, 6, device="cuda")
    chunks = -(-100 // chunk)

    def run(want_x, want_w, mode=torch.enable_grad):
        xs, ws = x.clone().requires_grad_(want_x), w.clone().requires_grad_(want_w)
        with mode():
            before = ext().launch_count()
            loss = fused_linear_distillation(xs, ws, ids, a, y, temperature=2.0, alpha=0.5, chunk=chunk)
            launches = ext().launch_count() - before
        if loss.requires_grad:
            loss.backward()
        return loss.detach(), xs.grad, ws.grad, launches

    loss, dx, dw, most = run(True, True)
    for want_x, want_w, mode in ((True, False, torch.enable_grad), (False, True, torch.enable_grad), (False, False, torch.enable_grad),
                                 (True, True, torch.no_grad), (True, True, torch.inference_mode)):
        got = run(want_x, want_w, mode)
        assert torch.equal(got[0], loss)
        formed = 0 if mode is not torch.enable_grad else want_x + want_w
        assert most - got[3] == (2 - formed) * chunks
        for want, mine, full in ((want_x, got[1], dx), (want_w, got[2], dw)):
            assert torch.equal(mine, full) if want and mode is torch.enable_grad else mine is None


def _targets_without_weight(device):
    """alpha 1 gives targets no weight: what they hold (another padding than ignore_index, say) does not matter."""
    z, ids, a, y = _inputs(6, 96, 3, torch.float32, device)
    bad = torch.where(torch.arange(6, device=device) % 2 == 0, -1, 96)
    for reduction in ("mean", "none"):
        want = distillation_loss(z, ids, a, reduction=reduction)
        assert torch.equal(distillation_loss(z, ids, a, bad, reduction=reduction), want)
    x, w = torch.ones(6, 16, device=device, dtype=torch.bfloat16), torch.ones(96, 16, device=device, dtype=torch.bfloat16)
    assert torch.equal(fused_linear_distillation(x, w, ids, a, bad), fused_linear_distillation(x, w, ids, a))


def test_targets_without_weight_on_cpu():
    _targets_without_weight("cpu")


@pytest.mark.gpu
def test_gpu_targets_without_weight():
    from my_muon_fsdp2_b200._ext import check_device_error

    check_device_error(0)
    _targets_without_weight("cuda")
    check_device_error(0)  # nothing was recorded


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 819200), (torch.float16, 819193), (torch.float32, 409600)], ids=["bf16", "fp16", "fp32"])
def test_gpu_largest_vocabulary(dtype, V):
    """The largest rows with the most slots: eight blocks a row, each with all the shared memory that there is."""
    for n, (tau, reduction) in enumerate([(2.0, "mean"), (1.5, "none")]):
        _check(*_inputs(3, V, 1024, dtype, "cuda", seed=n), tau, 0.5, reduction, 1024.0 if dtype == torch.float16 else 1.0)
    z, ids, a, y = _inputs(1, V, 2, dtype, "cuda")
    with pytest.raises(RuntimeError, match="vocabulary"):
        distillation_loss(torch.cat([z, z], 1), ids, a, y, alpha=0.5)
