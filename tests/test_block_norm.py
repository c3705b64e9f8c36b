"""The norms around a block with its gate and residual scale (``ops.block_norm``), against the formulas
in 64 bits.

Tolerances, per value, come from what is rounded: each output once (``finfo.eps / 2`` of it), and the fp32
arithmetic: sums over a row and the products behind them, at most some 40 roundings of 2^-24 of the
terms' sizes (2.5e-6; 5e-6 is allowed; that of the normalised rows, ``delta``, is carried through the
formula of each gradient), sums over rows up to 160 (1e-5)."""
import pytest
import torch

from my_muon_fsdp2_b200.ops.block_norm import gated_residual_norm

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ROW, SUM = 5e-6, 1e-5


def _inputs(lead, D, dtype, layer, gate, post, pre, device="cpu", seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)

    def r(*s, scale=1.0, m=0.0):
        return (torch.randn(*s, generator=g) * scale + m).to(device=device, dtype=dtype)

    t = {"x": r(*lead, D, scale=2.0), "y": r(*lead, D, m=mean)}
    if post:
        t["post_weight"] = r(D, scale=0.2, m=1.0)
        if layer:
            t["post_bias"] = r(D, scale=0.2)
    shape = {None: None, "channel": (D,), "sequence": lead[:1] + (1,) * (len(lead) - 1) + (D,), "token": lead + (D,)}[gate]
    if shape:
        t["gate"] = r(*shape, m=0.5)
    if pre:
        t["pre_weight"] = r(D, scale=0.2, m=1.0)
        if layer:
            t["pre_bias"] = r(D, scale=0.2)
    t["dh"], t["dn"] = r(*lead, D), r(*lead, D)
    return t


NAMES = ("x", "y", "post_weight", "post_bias", "gate", "pre_weight", "pre_bias")


def _reference(t, layer, eps, rs, bs):
    """({name: value in 64 bits}, {name: tolerance}) of the outputs and all gradients."""
    f = {k: v.detach().double().requires_grad_(k in NAMES) for k, v in t.items()}
    half = torch.finfo(t["x"].dtype).eps / 2
    floor = torch.finfo(t["x"].dtype).smallest_normal * 2 * half

    def norm(v, w, b):
        m = v.mean(-1, keepdim=True) if layer else torch.zeros_like(v[..., :1])
        r = ((v - m).square().mean(-1, keepdim=True) + eps).rsqrt()
        u = (v - m) * r
        return (u * w if b is None else u * w + b), u, r, m

    one = torch.ones(())
    gate = f.get("gate", one.to(f["x"].device))
    p, uy, ry, my = f["y"], None, None, None
    if "post_weight" in f:
        p, uy, ry, my = norm(f["y"], f["post_weight"], f.get("post_bias"))
    h = rs * f["x"] + bs * gate * p
    val, err = {"h": h}, {}
    with torch.no_grad():
        size_p = p.abs() if uy is None else f["post_weight"].abs() * ry * (f["y"].abs() + my.abs()) + f.get("post_bias", one * 0).abs()
        size_h = abs(rs) * f["x"].abs() + abs(bs) * gate.abs() * size_p
        err["h"] = ROW * size_h
    n = None
    if "pre_weight" in f:
        n, uh, rh, mh = norm(h, f["pre_weight"], f.get("pre_bias"))
        val["n"] = n
        with torch.no_grad():
            err["n"] = ROW * (f["pre_weight"].abs() * rh * (size_h + mh.abs()) + f.get("pre_bias", one * 0).abs()) \
                + f["pre_weight"].abs() * (rh * err["h"].mean(-1, keepdim=True) * (1 + uh.abs()))
    loss = (h * f["dh"]).sum() + (0 if n is None else (n * f["dn"]).sum())
    names = [k for k in NAMES if k in f]
    for k, g in zip(names, torch.autograd.grad(loss, [f[k] for k in names])):
        val["d" + k] = g
    with torch.no_grad():
        mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
        dH = f["dh"].clone()
        e = ROW * f["dh"].abs()
        if n is not None:
            delta = ROW * rh * (size_h + mh.abs())  # of the normalised h
            a = f["dn"] * f["pre_weight"]
            c2 = mean(a * uh)
            dH += rh * (a - uh * c2 - (mean(a) if layer else 0))
            e = e + rh * (delta * c2.abs() + (uh.abs() + delta) * mean(a.abs() * delta)) \
                + ROW * rh * (a.abs() + uh.abs() * mean((a * uh).abs()) + mean(a.abs()))
            err["dpre_weight"] = (f["dn"].abs() * delta).flatten(0, -2).sum(0) + SUM * (f["dn"] * uh).abs().flatten(0, -2).sum(0)
            err["dpre_bias"] = SUM * f["dn"].abs().flatten(0, -2).sum(0)
        err["dx"] = abs(rs) * e
        dp, edp = bs * gate * dH, abs(bs) * gate.abs() * e
        if "gate" in f:
            eg = abs(bs) * (e * size_p + SUM * dH.abs() * size_p)
            shape = f["gate"].shape
            if len(shape) == 1:
                eg = eg.flatten(0, -2).sum(0)
            else:
                for i, m in enumerate(shape):
                    if m == 1:
                        eg = eg.sum(i, keepdim=True)
            err["dgate"] = eg
        if uy is not None:
            dy_hat = ROW * ry * (f["y"].abs() + my.abs())
            err["dpost_weight"] = (edp * uy.abs() + dp.abs() * dy_hat + SUM * (dp * uy).abs()).flatten(0, -2).sum(0)
            err["dpost_bias"] = (edp + SUM * dp.abs()).flatten(0, -2).sum(0)
            b, eb = dp * f["post_weight"], edp * f["post_weight"].abs()
            err["dy"] = ry * (eb + uy.abs() * mean(eb * uy.abs()) + mean(eb)) + ry * dy_hat * mean(b * uy).abs() \
                + ROW * ry * (b.abs() + uy.abs() * mean((b * uy).abs()) + mean(b.abs())) + ry * uy.abs() * mean(b.abs() * dy_hat)
        else:
            err["dy"] = edp + ROW * dp.abs()
    return {k: v.detach() for k, v in val.items()}, {k: err[k] + half * v.detach().abs() + floor for k, v in val.items()}


def _run(t, layer, eps, rs, bs):
    args = {k: t[k].detach().requires_grad_() for k in NAMES if k in t}
    out = gated_residual_norm(**args, norm="layer" if layer else "rms", eps=eps, residual_scale=rs, branch_scale=bs)
    outs, ups = (list(out), [t["dh"], t["dn"]]) if isinstance(out, tuple) else ([out], [t["dh"]])
    got = {"h": outs[0].detach()}
    if len(outs) > 1:
        got["n"] = outs[1].detach()
    for k, g in zip(args, torch.autograd.grad(outs, list(args.values()), ups)):
        assert g.shape == args[k].shape and g.dtype == args[k].dtype
        got["d" + k] = g
    return got


def _compare(t, layer, eps=1e-5, rs=0.9, bs=0.5):
    val, tol = _reference(t, layer, eps, rs, bs)
    got = _run(t, layer, eps, rs, bs)
    assert set(got) == set(val)
    for k in val:
        off = (got[k].double() - val[k]).abs()
        assert bool((off <= tol[k]).all()), f"{k}: off by {(off / tol[k]).max().item():.3g} tolerances"


# ---------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
def test_cpu_gradients_against_differences(layer, gate):
    t = _inputs((2, 3), 5, torch.float64, layer, gate, True, True)
    names = [k for k in NAMES if k in t]
    f = lambda *a: gated_residual_norm(**dict(zip(names, a)), norm="layer" if layer else "rms",  # noqa: E731
                                       residual_scale=0.7, branch_scale=1.3)
    assert torch.autograd.gradcheck(f, [t[k].requires_grad_() for k in names])


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
def test_cpu_against_formulas(dtype):
    for layer in (False, True):
        t = _inputs((2, 3), 9, dtype, layer, "channel", True, True)
        val, _ = _reference(t, layer, 1e-5, 1.0, 0.5)
        h, n = gated_residual_norm(**{k: t[k] for k in NAMES if k in t}, norm="layer" if layer else "rms", branch_scale=0.5)
        for got, want in ((h, val["h"]), (n, val["n"])):
            assert torch.allclose(got.double(), want, rtol=torch.finfo(dtype).eps, atol=1e-5)


def test_matches_the_separate_ops_on_cpu():
    from my_muon_fsdp2_b200.ops.model_ops import rms_norm

    t = _inputs((4, 6), 8, torch.float32, False, None, True, True)
    h, n = gated_residual_norm(t["x"], t["y"], t["post_weight"], pre_weight=t["pre_weight"])
    want = t["x"] + rms_norm(t["y"], t["post_weight"])
    assert torch.allclose(h, want, atol=1e-6) and torch.allclose(n, rms_norm(want, t["pre_weight"]), atol=1e-5)


def test_refusals():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    f = gated_residual_norm
    for bad in (lambda: f(x, x[:1]), lambda: f(x, x, w[:4]), lambda: f(x, x, gate=x[:, :2]), lambda: f(x, x, gate=torch.zeros(1, 3, 8)),
                lambda: f(x, x, gate=torch.zeros(2, 8)), lambda: f(x, x, gate=torch.zeros(2, 3, 1)), lambda: f(x, x, norm="group"),
                lambda: f(x, x, w, w), lambda: f(x, x, None, w, norm="layer"), lambda: f(x, x, pre_bias=w, norm="layer"),
                lambda: f(torch.zeros(2, 0), torch.zeros(2, 0)), lambda: f(torch.zeros(()), torch.zeros(())),
                lambda: f(torch.zeros(1, 8193), torch.zeros(1, 8193))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(x, x.bfloat16()), lambda: f(x, x, w.half()), lambda: f(x.long(), x.long()), lambda: f(x, x, gate=w.double())):
        with pytest.raises(TypeError):
            bad()


# ---------------------------------------------------------------------------------- GPU
# widths: one value, less than a warp, each access width and number of vectors a thread, the largest
WIDTHS = [1, 7, 64, 100, 203, 1024, 1032, 1280, 2050, 3001, 4096, 4104, 5000, 8191, 8192]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("D", WIDTHS)
def test_gpu_widths(D, layer, dtype):
    for n, (gate, lead) in enumerate([("channel", (5,)), ("token", (2, 3)), ("sequence", (3, 7)), (None, (1, 1))]):
        _compare(_inputs(lead, D, dtype, layer, gate, True, True, "cuda", seed=n), layer)


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
@pytest.mark.parametrize("lead", [(1,), (1, 1), (3, 701), (700, 3), (2, 2, 300)], ids=str)
def test_gpu_rows_and_parts(lead, gate, layer):
    """More rows than workers, more gates than workers, and each combination of the two norms."""
    for post in (False, True):
        for pre in (False, True):
            _compare(_inputs(lead, 136, torch.bfloat16, layer, gate, post, pre, "cuda"), layer, rs=1.0, bs=1.0)


@pytest.mark.gpu
def test_gpu_many_gates_in_one_launch_and_more():
    """A gate's group for each of more sequences than one launch's grid takes."""
    x = torch.ones(33000, 2, 8, device="cuda")
    y = torch.arange(33000, device="cuda", dtype=torch.float32)[:, None, None].expand(33000, 2, 8) % 97
    gate = torch.ones(33000, 1, 8, device="cuda", requires_grad=True)
    h = gated_residual_norm(x, y, gate=gate)
    (g,) = torch.autograd.grad(h, gate, torch.ones_like(h))
    assert torch.equal(g, 2 * y[:, :1])


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
def test_gpu_large_mean_and_extremes(layer):
    """A mean a thousand deviations off; rows of zeros; rows with infinities or NaN stay by themselves."""
    t = _inputs((64,), 1000, torch.float32, layer, "channel", True, True, "cuda", mean=1000.0)
    _compare(t, layer)
    t = _inputs((6,), 256, torch.bfloat16, layer, "channel", True, True, "cuda")
    clean = gated_residual_norm(**{k: t[k] for k in NAMES if k in t}, norm="layer" if layer else "rms")
    t["x"][1], t["y"][1] = 0, 0
    t["y"][3, 5], t["x"][4, 0] = float("inf"), float("nan")
    h, n = gated_residual_norm(**{k: t[k] for k in NAMES if k in t}, norm="layer" if layer else "rms")
    assert torch.isfinite(h[1]).all() and torch.isfinite(n[1]).all() and n[3].isnan().any() and n[4].isnan().all()
    for r in (0, 2, 5):
        assert torch.equal(h[r], clean[0][r]) and torch.equal(n[r], clean[1][r])


@pytest.mark.gpu
def test_gpu_difference_quotient():
    """The kernel's gradient along a direction against the difference quotient of the 64-bit formula."""
    t = _inputs((3, 5), 96, torch.float32, True, "sequence", True, True, "cuda")
    got = _run(t, True, 1e-5, 0.9, 0.5)
    names = [k for k in NAMES if k in t]
    g = torch.Generator().manual_seed(3)
    v = {k: torch.randn(t[k].shape, generator=g, dtype=torch.float64).cuda() for k in names}

    def loss(s):
        f = {k: t[k].double().cpu() + s * v[k].cpu() for k in names}
        h, n = gated_residual_norm(**f, norm="layer", residual_scale=0.9, branch_scale=0.5)
        return float((h * t["dh"].double().cpu()).sum() + (n * t["dn"].double().cpu()).sum())

    s = 1e-5
    quotient = (loss(s) - loss(-s)) / (2 * s)
    along = sum(float((got["d" + k].double() * v[k]).sum()) for k in names)
    size = sum(float((got["d" + k].double() * v[k]).abs().sum()) for k in names)
    assert abs(quotient - along) <= 1e-5 * size  # fp32 gradients; the quotient's own error is below 1e-8


@pytest.mark.gpu
def test_gpu_unused_outputs_empty_rows_and_layouts():
    t = _inputs((4, 6), 64, torch.bfloat16, False, "channel", True, True, "cuda")
    a = {k: t[k].requires_grad_() for k in NAMES if k in t}
    h, n = gated_residual_norm(**a)
    g = torch.autograd.grad(n, [a["x"], a["y"], a["pre_weight"]], t["dn"], retain_graph=True)
    z = torch.autograd.grad([h, n], [a["x"], a["y"], a["pre_weight"]], [torch.zeros_like(h), t["dn"]], retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(g, z))
    only_h = torch.autograd.grad(h, list(a.values()), t["dh"], allow_unused=True, retain_graph=True)
    assert only_h[list(a).index("pre_weight")] is None and torch.equal(only_h[0], t["dh"])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(n, a["x"], t["dn"], create_graph=True)
    # a gate for each sequence that takes no gradient itself: the others' are those with it
    t = _inputs((5, 9), 64, torch.bfloat16, True, "sequence", True, True, "cuda")
    full = _run(t, True, 1e-5, 0.9, 0.5)
    a = {k: t[k].detach().requires_grad_(k != "gate") for k in NAMES if k in t}
    out = gated_residual_norm(**a, norm="layer", residual_scale=0.9, branch_scale=0.5)
    rest = [k for k in a if k != "gate"]
    for k, g in zip(rest, torch.autograd.grad(out, [a[k] for k in rest], (t["dh"], t["dn"]))):
        assert torch.equal(g, full["d" + k])
    # rows with strides: a transposed view, and an offset that 16-byte accesses cannot take
    t = _inputs((4, 6), 64, torch.bfloat16, False, "channel", True, True, "cuda")
    h, n = gated_residual_norm(**{k: t[k] for k in NAMES if k in t})
    xt = t["x"].detach().transpose(0, 1).contiguous().transpose(0, 1)
    flat = torch.empty(1 + 24 * 64, device="cuda", dtype=torch.bfloat16)
    off = flat[1:].view(4, 6, 64).copy_(t["y"].detach())
    h2, n2 = gated_residual_norm(xt, off, *[t[k].detach() for k in ("post_weight",)], gate=t["gate"].detach(),
                                 pre_weight=t["pre_weight"].detach())
    assert torch.allclose(h2.float(), h.float(), rtol=2**-7) and torch.allclose(n2.float(), n.float(), rtol=2**-7, atol=1e-6)
    e = torch.zeros(0, 6, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    h, n = gated_residual_norm(e, e, w, gate=w, pre_weight=w)
    (gw,) = torch.autograd.grad(n.sum(), w)
    assert h.shape == (0, 6, 64) and torch.equal(gw, torch.zeros_like(w))


@pytest.mark.gpu
def test_gpu_same_bits_streams_and_graph():
    t = _inputs((9, 77), 1280, torch.float16, True, "sequence", True, True, "cuda")
    a, b = _run(t, True, 1e-5, 1.0, 1.0), _run(t, True, 1e-5, 1.0, 1.0)
    assert all(torch.equal(a[k], b[k]) for k in a)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        c = _run(t, True, 1e-5, 1.0, 1.0)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a[k], c[k]) for k in a)
    del a, b, c
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _run(t, True, 1e-5, 1.0, 1.0)
    t["y"].mul_(0.5)
    t["dn"].mul_(2)
    g.replay()
    want = _run(t, True, 1e-5, 1.0, 1.0)
    assert all(torch.equal(out[k], want[k]) for k in want)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """More than 2^31 values: the last rows are those of a call on them alone."""
    R, D = 530000, 4096
    x = torch.empty(R, D, device="cuda", dtype=torch.bfloat16)
    t = _inputs((3,), D, torch.bfloat16, False, None, True, True, "cuda")
    x[-3:] = t["x"]
    w = dict(post_weight=t["post_weight"], pre_weight=t["pre_weight"])
    want = gated_residual_norm(t["x"], t["x"], **w)
    got = gated_residual_norm(x, x, **w)
    assert torch.equal(got[0][-3:], want[0]) and torch.equal(got[1][-3:], want[1])
    del got
    small = t["x"].clone().requires_grad_()
    (wg,) = torch.autograd.grad(gated_residual_norm(small, small, **w), small, (t["dh"], t["dn"]))
    x[:-3] = 1
    x.requires_grad_()
    dh = torch.zeros_like(x)
    dh[-3:] = t["dh"]
    dn = torch.zeros_like(x)
    dn[-3:] = t["dn"]
    (g,) = torch.autograd.grad(gated_residual_norm(x, x, **w), x, (dh, dn))
    assert torch.equal(g[-3:], wg) and not g[:-3].any()


@pytest.mark.gpu
def test_gpu_refusals():
    """What the CPU form refuses the kernels' entry refuses in the same way."""
    z = lambda *s, dtype=torch.float32: torch.zeros(s, device="cuda", dtype=dtype)  # noqa: E731
    x, w, f = z(2, 3, 8), torch.ones(8, device="cuda"), gated_residual_norm
    for bad in (lambda: f(x, x[:1]), lambda: f(x, x.view(3, 2, 8)), lambda: f(x, x, w[:4]), lambda: f(x, x, w.view(1, 8)),
                lambda: f(x, x, gate=x[:, :2]), lambda: f(x, x, gate=z(1, 3, 8)), lambda: f(x, x, gate=z(2, 8)),
                lambda: f(x, x, gate=z(2, 3, 1)), lambda: f(x, x, gate=z(1, 2, 3, 8)), lambda: f(x, x, gate=z()),
                lambda: f(x, x, norm="group"), lambda: f(x, x, w, w), lambda: f(x, x, None, w, norm="layer"),
                lambda: f(x, x, pre_bias=w, norm="layer"), lambda: f(x, x, pre_weight=w, pre_bias=w),
                lambda: f(z(2, 0), z(2, 0)), lambda: f(z(), z()), lambda: f(z(), z(), gate=z()), lambda: f(z(1, 8193), z(1, 8193))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(x, x.bfloat16()), lambda: f(x, x, w.half()), lambda: f(x.long(), x.long()), lambda: f(x, x, gate=w.double()),
                lambda: f(x.double(), x.double()), lambda: f(x, x.cpu()), lambda: f(x, x, w.cpu())):
        with pytest.raises(TypeError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("D", [4098, 5000, 8192])
def test_gpu_wide_rows_in_many_turns(D, layer, dtype):
    """Rows shared by two blocks, more of them than go over the device at once, and each gate."""
    for n, (gate, lead) in enumerate([("channel", (2, 301)), ("token", (601,)), ("sequence", (3, 211)), ("sequence", (300, 2)), (None, (500,))]):
        args = _inputs(lead, D, dtype, layer, gate, True, True, "cuda", seed=n)
        _compare(args, layer)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [5120, 8192])
def test_gpu_wide_rows_same_bits_streams_and_graph(D):
    """Rows over several blocks: two calls at once, a captured one and its replay give the same bits."""
    t = _inputs((2, 331), D, torch.bfloat16, False, "token", True, True, "cuda")
    a = _run(t, False, 1e-5, 1.0, 1.0)
    streams, runs = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            runs.append(_run(t, False, 1e-5, 1.0, 1.0))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a[k], r[k]) for r in runs for k in a)
    del a, runs
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _run(t, False, 1e-5, 1.0, 1.0)
    t["y"].mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    got = {k: v.clone() for k, v in out.items()}
    del out, g
    want = _run(t, False, 1e-5, 1.0, 1.0)
    assert all(torch.equal(got[k], want[k]) for k in want)


def _duals(call, shapes, device):
    import torch.autograd.forward_ad as fw

    for name in shapes:
        with fw.dual_level():
            ts = {n: torch.ones(s, device=device) for n, s in shapes.items()}
            ts[name] = fw.make_dual(ts[name], torch.ones_like(ts[name]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(ts)


SHAPES = {"x": (2, 3, 8), "y": (2, 3, 8), "post_weight": (8,), "post_bias": (8,), "gate": (2, 1, 8), "pre_weight": (8,), "pre_bias": (8,)}


def test_forward_mode_is_refused_by_the_entry():
    """A tangent on any of the tensors; the extension refuses it before it looks at where they are."""
    from my_muon_fsdp2_b200._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    _duals(lambda t: ext().block_norm(*[t[n] for n in NAMES], True, 1e-5, 1.0, 1.0), SHAPES, "cpu")


@pytest.mark.gpu
def test_gpu_forward_mode_is_refused():
    _duals(lambda t: gated_residual_norm(**t, norm="layer"), SHAPES, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("D", [5122, 6001, 8191])
def test_gpu_rows_over_two_blocks_in_many_turns(D, layer, dtype):
    """Two blocks a row (widths above 5120; up to there it is four), unequal shares and narrow accesses: more
    rows than go over the device at once, so that the exchange's places and phases go round."""
    for n, (gate, lead) in enumerate([("channel", (2, 301)), ("token", (601,)), ("sequence", (3, 211)), ("sequence", (300, 2)), (None, (500,))]):
        _compare(_inputs(lead, D, dtype, layer, gate, True, True, "cuda", seed=n), layer)


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("D", [64, 1000, 4096, 5000, 8192])
def test_gpu_backward_of_rows_beside_bad_ones(D, layer):
    """Infinities and NaN in a row or its gradients stay in that row's dx and dy."""
    t = _inputs((601,), D, torch.bfloat16, layer, "channel", True, True, "cuda")
    clean = _run(t, layer, 1e-5, 1.0, 1.0)
    t["y"][3, 5], t["x"][4, 0], t["dn"][6, 1], t["dh"][300, 2] = float("inf"), float("nan"), float("nan"), float("inf")
    got = _run(t, layer, 1e-5, 1.0, 1.0)
    keep = [i for i in range(601) if i not in (3, 4, 6, 300)]
    for k in ("h", "n", "dx", "dy"):
        assert torch.equal(got[k][keep], clean[k][keep]), k
    assert not any(torch.isfinite(got["dx"][i]).all() for i in (3, 4, 6, 300))
