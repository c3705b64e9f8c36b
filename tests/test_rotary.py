"""Rotary positions (``ops.rotary``) against the formula in 64 bits.

Tolerance, per value: half a rounding step of the type (``finfo.eps / 2`` of the value, half of the
smallest subnormal), and for the fp32 arithmetic 1e-6 of ``m (|x1| + |x2|)``: the fraction of a half turn
is rounded once (2^-24, 1.9e-7 in the angle), sincospi and the factor m add 3 * 2^-24, the products and
the sum 3 * 2^-24 more."""
import math

import pytest
import torch

from my_muon_fsdp2_b200.ops.rotary import RopeScaling, RotaryEmbedding, apply_rotary

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _formula(x, pos, rot, inverse=False):
    """([..., T, H, D] in 64 bits, m (|x1| + |x2|) of each value); pos [..., T]."""
    R = rot.rotary_dim
    a = pos.double()[..., None, None] * torch.tensor(rot.frequencies, dtype=torch.float64, device=x.device)
    c, s = rot.magnitude * a.cos(), rot.magnitude * a.sin() * (-1 if inverse else 1)
    x = x.double()
    i = torch.arange(R // 2, device=x.device)
    i1, i2 = (2 * i, 2 * i + 1) if rot.interleaved else (i, i + R // 2)
    x1, x2 = x[..., i1], x[..., i2]
    out, size = x.clone(), torch.zeros_like(x)
    out[..., i1], out[..., i2] = x1 * c - x2 * s, x2 * c + x1 * s
    size[..., i1] = size[..., i2] = abs(rot.magnitude) * (x1.abs() + x2.abs())
    return out, size


def _close(got, want, size):
    f = torch.finfo(got.dtype)
    tol = f.eps / 2 * want.abs() + f.smallest_normal * f.eps / 2 + 1e-6 * size
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"off by {(off / tol).max().item():.3g} tolerances"


def _rand(shape, dtype, device="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(device=device, dtype=dtype)


SCALINGS = [None, RopeScaling("linear", 4.0), RopeScaling("ntk", 8.0), RopeScaling("llama3", 8.0), RopeScaling("yarn", 4.0, 4096)]


# ---------------------------------------------------------------------------------- CPU
def test_scaled_frequencies():
    """Each kind of scaling against its definition at the ends and in between."""
    base = RotaryEmbedding(64, 10000.0).frequencies
    assert base[0] == 1.0 and abs(base[31] - 10000.0 ** (-62 / 64)) < 1e-18
    lin = RotaryEmbedding(64, scaling=RopeScaling("linear", 4.0)).frequencies
    assert all(abs(a - b / 4) < 1e-18 for a, b in zip(lin, base))
    ntk = RotaryEmbedding(64, scaling=RopeScaling("ntk", 4.0)).frequencies
    assert ntk[0] == 1.0 and abs(ntk[31] / base[31] - 1 / 4) < 1e-12
    l3 = RotaryEmbedding(64, scaling=RopeScaling("llama3", 8.0, 1024)).frequencies
    for f, g in zip(base, l3):
        turns = 1024 * f / (2 * math.pi)
        if turns >= 4:
            assert g == f
        elif turns <= 1:
            assert abs(g - f / 8) < 1e-18
        else:
            w = (turns - 1) / 3
            assert f / 8 < g < f and abs(g - (w * f + (1 - w) * f / 8)) < 1e-15
    r = RotaryEmbedding(64, scaling=RopeScaling("yarn", 8.0, 4096))
    assert r.frequencies[0] == base[0] and abs(r.frequencies[31] - base[31] / 8) < 1e-18
    assert abs(r.magnitude - (0.1 * math.log(8.0) + 1)) < 1e-12
    assert RotaryEmbedding(64, scaling=RopeScaling("yarn", 8.0, magnitude=1.0)).magnitude == 1.0


def test_default_is_apply_rope_on_cpu():
    from my_muon_fsdp2_b200.ops.model_ops import _rope_torch

    x = _rand((2, 5, 3, 16), torch.float32)
    y = apply_rotary(x, None, RotaryEmbedding(16, 10000.0))
    assert torch.allclose(y, _rope_torch(x, 5, 10000.0), atol=1e-5)


@pytest.mark.parametrize("interleaved", [False, True])
def test_cpu_matches_formula_and_gradient(interleaved):
    rot = RotaryEmbedding(12, 100.0, rotary_dim=8, interleaved=interleaved, scaling=RopeScaling("yarn", 2.0, 64))
    q = _rand((2, 3, 4, 12), torch.float64).requires_grad_()
    k = _rand((2, 3, 2, 12), torch.float64, seed=1).requires_grad_()
    pos = torch.tensor([[0, 7, 100000], [3, 3, -5]])
    a, b = apply_rotary(q, k, rot, pos)
    assert torch.allclose(a, _formula(q.detach(), pos, rot)[0], atol=1e-12)
    assert torch.allclose(b, _formula(k.detach(), pos, rot)[0], atol=1e-12)
    assert torch.autograd.gradcheck(lambda x, y: apply_rotary(x, y, rot, pos), (q, k))
    x = q.detach().clone()
    assert apply_rotary(x, None, rot, pos, inplace=True) is x
    assert torch.equal(x, a.detach())


def test_fixed_point_turns_far_positions():
    """position * turns modulo 2^64, as the kernel forms it, is the angle's fraction of a turn."""
    rot = RotaryEmbedding(128, 500000.0, scaling=RopeScaling("llama3", 8.0))
    for p in (0, 1, 131071, 10**6, 2**31 - 1, -3):
        for f, t in zip(rot.frequencies, rot._turns.tolist()):
            frac = ((p * t) % 2**64) / 2**64
            want = math.fmod(p * f / (2 * math.pi), 1.0) % 1.0
            d = abs(frac - want)
            assert min(d, 1 - d) < 1e-9 * max(1, abs(p) / 2**20)


def test_refusals():
    rot = RotaryEmbedding(8)
    q, k = torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 1, 8)
    for bad in (dict(head_dim=7), dict(head_dim=0), dict(head_dim=512), dict(head_dim=8, rotary_dim=3),
                dict(head_dim=8, rotary_dim=10), dict(head_dim=8, theta=1.0), dict(head_dim=8, theta=math.inf),
                dict(head_dim=8, rotary_dim=2, scaling=RopeScaling("ntk", 2.0))):
        with pytest.raises(ValueError):
            RotaryEmbedding(**bad)
    for bad in (dict(kind="cubic"), dict(kind="linear", factor=0.0), dict(kind="linear", factor=math.nan),
                dict(kind="yarn", original_max_position=0), dict(kind="llama3", low_freq_factor=4.0),
                dict(kind="yarn", beta_slow=40.0), dict(kind="yarn", magnitude=math.inf)):
        with pytest.raises(ValueError):
            RopeScaling(**bad)
    with pytest.raises(TypeError):
        apply_rotary(q, k, None)
    with pytest.raises(ValueError):
        apply_rotary(q[0, 0], None, rot)
    with pytest.raises(ValueError):
        apply_rotary(q[..., :6], None, rot)
    with pytest.raises(TypeError):
        apply_rotary(q.long(), None, rot)
    with pytest.raises(ValueError):
        apply_rotary(q, k[:, :1], rot)
    with pytest.raises(ValueError):
        apply_rotary(q, k.bfloat16(), rot)
    with pytest.raises(TypeError):
        apply_rotary(q, k, rot, torch.zeros(2))
    with pytest.raises(ValueError):
        apply_rotary(q, k, rot, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError):
        apply_rotary(q, k, rot, torch.zeros(1, 1, 2, dtype=torch.long))
    with pytest.raises(RuntimeError):
        apply_rotary(q.clone().requires_grad_(), k, rot, inplace=True)
    with pytest.raises(ValueError):
        apply_rotary(k.expand(1, 2, 3, 8), None, rot, inplace=True)
    with pytest.raises(ValueError):
        apply_rotary(torch.zeros(1, 2, 8, 3).transpose(2, 3), None, rot, inplace=True)
    with pytest.raises(ValueError):
        apply_rotary(q, q, rot, inplace=True)


def test_messages_of_the_entry_hold_numbers():
    """A refusal that names a number comes back as an error (its text is formed in the extension)."""
    from my_muon_fsdp2_b200._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    q = torch.zeros(4, 2, 9)
    with pytest.raises(RuntimeError, match=r"heads, 8\]"):
        ext().rotary(q, None, None, q, 8, 8, False, 1.0, False)


# ---------------------------------------------------------------------------------- GPU
# (batch, seq, q heads, k heads, head_dim, rotary_dim): one token, odd lengths, heads that are no
# multiple of what a thread takes, parts whose width allows 16-, 4- and 2-byte accesses only
SHAPES = [(1, 1, 1, 0, 2, 2), (1, 1, 32, 8, 128, 128), (3, 17, 5, 1, 64, 32), (2, 33, 7, 3, 80, 20), (1, 129, 2, 2, 256, 256),
          (2, 5, 3, 1, 96, 6), (1, 700, 9, 9, 64, 64), (2, 9, 2, 1, 256, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "neighbours"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gpu_forward_backward(shape, interleaved, dtype):
    B, T, hq, hk, D, R = shape
    for n, scaling in enumerate(SCALINGS):
        if scaling is not None and scaling.kind == "ntk" and R < 4:
            continue
        rot = RotaryEmbedding(D, 10000.0, rotary_dim=R, interleaved=interleaved, scaling=scaling)
        q = _rand((B, T, hq, D), dtype, "cuda", n).requires_grad_()
        k = _rand((B, T, hk, D), dtype, "cuda", n + 50).requires_grad_() if hk else None
        pos = (torch.arange(T, device="cuda") + torch.randint(-9, 131072, (B, 1), device="cuda")) if n % 2 else None
        at = pos if pos is not None else torch.arange(T, device="cuda").expand(B, T)
        out = apply_rotary(q, k, rot, pos)
        outs, ins = ([out], [q]) if k is None else (list(out), [q, k])
        ups = [_rand(o.shape, dtype, "cuda", 7 + i) for i, o in enumerate(outs)]
        for x, o, u, g in zip(ins, outs, ups, torch.autograd.grad(outs, ins, ups)):
            assert o.is_contiguous() and o.dtype == dtype
            _close(o.detach(), *_formula(x.detach(), at, rot))
            _close(g, *_formula(u, at, rot, inverse=True))
            assert torch.equal(o[..., R:], x[..., R:])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "neighbours"])
def test_gpu_strides_alignment_and_positions(interleaved):
    """Views of a packed projection, odd storage offsets, transposed and expanded heads, [tokens, heads,
    head_dim], int32 and broadcast positions: all equal to the contiguous call, bit by bit."""
    rot = RotaryEmbedding(64, 10000.0, rotary_dim=32, interleaved=interleaved)
    for off in (0, 1, 2, 4):
        flat = _rand((off + 2 * 9 * 10 * 64,), torch.bfloat16, "cuda")
        qkv = flat[off:].view(2, 9, 10, 64)
        q, k = qkv[:, :, :6], qkv[:, :, 6:8]
        want = apply_rotary(q.contiguous().clone(), k.contiguous().clone(), rot)
        for a, b in zip(apply_rotary(q, k, rot), want):
            assert torch.equal(a, b)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(apply_rotary(qt, None, rot), want[0])
    odd = q.transpose(2, 3).contiguous().transpose(2, 3)  # the head's values are not contiguous
    assert torch.equal(apply_rotary(odd, None, rot), want[0])
    e = k[:, :, :1].expand(2, 9, 4, 64).requires_grad_(False)
    assert torch.equal(apply_rotary(e, None, rot)[:, :, 3], want[1][:, :, 0])
    flat3 = apply_rotary(q.reshape(18, 6, 64), None, rot, torch.arange(9, device="cuda").repeat(2))
    assert torch.equal(flat3.view(2, 9, 6, 64), want[0])
    for pos in (torch.arange(9, device="cuda", dtype=torch.int32), torch.arange(18, device="cuda")[::2] // 2,
                torch.arange(9, device="cuda")[None]):
        assert torch.equal(apply_rotary(q, None, rot, pos), want[0])
    one = apply_rotary(q, None, rot, torch.tensor([3], device="cuda"))
    assert torch.equal(one[:, 3], want[0][:, 3])
    assert torch.equal(apply_rotary(q[:, :0], None, rot), q[:, :0])
    # the gradient of an expanded (shared) head is the sum over its readers
    s = k[:, :, :1].detach().float().requires_grad_()
    up = _rand((2, 9, 4, 64), torch.float32, "cuda", 3)
    (g,) = torch.autograd.grad(apply_rotary(s.expand(2, 9, 4, 64), None, rot), s, up)
    want_g = _formula(up, torch.arange(9, device="cuda").expand(2, 9), rot, inverse=True)[0].sum(2, keepdim=True)
    assert torch.allclose(g.double(), want_g, atol=1e-5)


@pytest.mark.gpu
def test_gpu_in_place_leaves_the_rest():
    """In place, into rows of a cache: neighbours in memory keep their values."""
    rot = RotaryEmbedding(64, rotary_dim=16)
    cache = _rand((4, 12, 2, 80), torch.float16, "cuda")
    was = cache.clone()
    pos = torch.tensor([[5], [0], [70000], [9]], device="cuda")
    q, k = _rand((4, 1, 6, 64), torch.float16, "cuda", 1), cache[:, 7:8, :, :64]
    q0 = q.clone()
    want = apply_rotary(q, k, rot, pos)
    got = apply_rotary(q, k, rot, pos, inplace=True)
    assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and not torch.equal(q, q0)
    was[:, 7, :, :16] = cache[:, 7, :, :16]
    assert torch.equal(cache, was)


@pytest.mark.gpu
def test_gpu_streams_and_graph():
    """On another stream, and captured: a replay sees new positions and new values."""
    rot = RotaryEmbedding(128, 500000.0, scaling=RopeScaling("llama3", 8.0)).to("cuda")
    q, k = _rand((8, 1, 4, 128), torch.bfloat16, "cuda"), _rand((8, 1, 2, 128), torch.bfloat16, "cuda", 1)
    pos = torch.arange(8, device="cuda")[:, None] * 1000
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a = apply_rotary(q, k, rot, pos)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(x, y) for x, y in zip(a, apply_rotary(q, k, rot, pos)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = apply_rotary(q, k, rot, pos)
    pos += 17
    q.mul_(2)
    g.replay()
    assert all(torch.equal(x, y) for x, y in zip(out, apply_rotary(q, k, rot, pos)))


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """More than 2^31 values: the last tokens are those of a call on them alone."""
    rot = RotaryEmbedding(128, 500000.0)
    T = 270000
    q = torch.empty(1, T, 64, 128, device="cuda", dtype=torch.bfloat16)
    q[:, -3:] = _rand((1, 3, 64, 128), torch.bfloat16, "cuda")
    want = apply_rotary(q[:, -3:].clone(), None, rot, torch.arange(T - 3, T, device="cuda"))
    assert torch.equal(apply_rotary(q, None, rot)[:, -3:], want)


@pytest.mark.gpu
def test_gpu_refusals():
    rot = RotaryEmbedding(8, interleaved=True)
    flat = torch.zeros(1 + 2 * 3 * 8, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):  # neighbouring pairs that straddle an access, nowhere to copy them to
        apply_rotary(flat[1:].view(1, 2, 3, 8), None, rot, inplace=True)
    with pytest.raises(ValueError):
        apply_rotary(flat[:-1].view(1, 2, 3, 8), None, rot, torch.arange(2))
    x = torch.zeros(1, 2, 3, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(apply_rotary(x, None, rot).sum(), x, create_graph=True)


@pytest.mark.gpu
def test_gpu_refusals_of_arguments():
    """What the CPU form refuses the kernel's entry refuses in the same way."""
    rot = RotaryEmbedding(8)
    q, k = torch.zeros(1, 2, 3, 8, device="cuda"), torch.zeros(1, 2, 1, 8, device="cuda")
    pos = lambda *s: torch.zeros(s, dtype=torch.long, device="cuda")  # noqa: E731
    for bad in (lambda: apply_rotary(q, k, None), lambda: apply_rotary(q.long(), None, rot), lambda: apply_rotary(q.double(), None, rot),
                lambda: apply_rotary(q, k, rot, pos(2).float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: apply_rotary(q[0, 0], None, rot), lambda: apply_rotary(q[None], None, rot), lambda: apply_rotary(q[..., :6], None, rot),
                lambda: apply_rotary(q, k[:, :1], rot), lambda: apply_rotary(q, k.bfloat16(), rot), lambda: apply_rotary(q, k.cpu(), rot),
                lambda: apply_rotary(q, "k", rot),
                lambda: apply_rotary(q, k, rot, pos(3)), lambda: apply_rotary(q, k, rot, pos(1, 1, 2)), lambda: apply_rotary(q, k, rot, pos()),
                lambda: apply_rotary(k.expand(1, 2, 3, 8), None, rot, inplace=True), lambda: apply_rotary(q, q, rot, inplace=True),
                lambda: apply_rotary(torch.zeros(1, 2, 8, 3, device="cuda").transpose(2, 3), None, rot, inplace=True)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        apply_rotary(q.clone().requires_grad_(), k, rot, inplace=True)


@pytest.mark.gpu
def test_gpu_inplace_is_seen_by_autograd():
    """A product that kept q for its backward notices that q was rotated in place."""
    rot = RotaryEmbedding(8).to("cuda")
    for mode in ("q", "k"):
        q, k = torch.randn(1, 2, 3, 8, device="cuda"), torch.randn(1, 2, 1, 8, device="cuda")
        w = torch.randn(8, 4, device="cuda", requires_grad=True)
        out = ((q if mode == "q" else k) @ w).sum()
        apply_rotary(q, k, rot, inplace=True)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(out, w)
    with torch.inference_mode():
        q = torch.randn(1, 2, 3, 8, device="cuda")
        want = apply_rotary(q, None, rot)
        assert apply_rotary(q, None, rot, inplace=True) is q and torch.equal(q, want)


def _dual_is_refused(call, *shapes, device="cuda"):
    """call(tensors) raises when any one of them has a tangent, whether or not gradients are recorded."""
    import torch.autograd.forward_ad as fw

    for i in range(len(shapes)):
        with fw.dual_level():
            ts = [torch.ones(s, device=device) for s in shapes]
            ts[i] = fw.make_dual(ts[i], torch.ones_like(ts[i]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*ts)


def test_forward_mode_is_refused_by_the_entry():
    """The extension refuses tensors with a tangent before it looks at where they are."""
    from my_muon_fsdp2_b200._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    rot = RotaryEmbedding(8)
    for inplace in (False, True):
        _dual_is_refused(lambda q, k: ext().rotary(q, k, None, rot._turns, 8, 8, False, 1.0, inplace), (1, 2, 3, 8), (1, 2, 1, 8),
                         device="cpu")


@pytest.mark.gpu
def test_gpu_forward_mode_is_refused():
    rot = RotaryEmbedding(8)
    for inplace in (False, True):
        _dual_is_refused(lambda q, k: apply_rotary(q, k, rot, inplace=inplace), (1, 2, 3, 8), (1, 2, 1, 8))


def test_tables_made_in_inference_mode_are_ordinary_tensors():
    with torch.inference_mode():
        rot = RotaryEmbedding(8)
        table = rot._table(torch.device("cpu"))
    assert not rot._turns.is_inference() and not table.is_inference()


@pytest.mark.gpu
def test_gpu_evaluation_before_training():
    """The plan's first use, and its making, in inference mode; then a step with gradients."""
    from my_muon_fsdp2_b200.models.llama import Llama, LlamaConfig

    made = RotaryEmbedding(8)
    with torch.inference_mode():
        inside = RotaryEmbedding(8)
        for rot in (made, inside):
            apply_rotary(torch.ones(1, 2, 3, 8, device="cuda"), None, rot)
    q = _rand((1, 2, 3, 8), torch.float32, "cuda").requires_grad_()
    for rot in (made, inside):
        out = apply_rotary(q, None, rot)
        (g,) = torch.autograd.grad(out, q, torch.ones_like(out))
        _close(g, *_formula(torch.ones_like(q), torch.arange(2, device="cuda")[None], rot, inverse=True))
    torch.manual_seed(0)
    model = Llama(LlamaConfig.tiny(dim=128, n_heads=2, n_kv_heads=1, ffn_dim=256, n_layers=1, rope_scaling=SCALINGS[3]))
    model = model.to("cuda", torch.bfloat16)
    tokens = torch.randint(0, 512, (2, 17), device="cuda")
    with torch.inference_mode():
        model(tokens)
    model(tokens[:, :-1], tokens[:, 1:]).backward()
    assert all(p.grad is not None for p in model.parameters())


def test_plan_made_under_another_default_device():
    """A model is often built under the meta device before it is sharded: the plan's table has its values."""
    want = RotaryEmbedding(8)
    with torch.device("meta"):
        rot = RotaryEmbedding(8)
    assert torch.equal(rot._turns, want._turns)
    x = _rand((1, 2, 3, 8), torch.float32)
    assert torch.equal(apply_rotary(x, None, rot), apply_rotary(x, None, want))


@pytest.mark.gpu
def test_gpu_plan_made_under_another_default_device():
    x = _rand((1, 2, 3, 8), torch.float32, "cuda")
    want = apply_rotary(x, None, RotaryEmbedding(8))
    for device in ("meta", "cuda"):
        with torch.device(device):
            rot = RotaryEmbedding(8)
        assert torch.equal(apply_rotary(x, None, rot), want)


def test_refused_in_place_call_leaves_versions():
    """The extension refuses CPU tensors: their version counters stay."""
    from my_muon_fsdp2_b200._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    rot, q, k = RotaryEmbedding(8), torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError):
        ext().rotary(q, k, None, rot._turns, 8, 8, False, 1.0, True)
    assert q._version == 0 and k._version == 0


@pytest.mark.gpu
def test_gpu_refused_in_place_call_leaves_versions():
    rot = RotaryEmbedding(8).to("cuda")
    q, k = torch.randn(1, 2, 3, 8, device="cuda"), torch.randn(1, 2, 1, 8, device="cuda")
    w = torch.randn(8, 4, device="cuda", requires_grad=True)
    out = (q @ w).sum() + (k @ w).sum()
    for bad, error in ((dict(positions=torch.zeros(2, device="cuda")), TypeError), (dict(positions=torch.zeros(3, dtype=torch.long, device="cuda")), ValueError),
                       (dict(k=k.bfloat16()), ValueError), (dict(k=k[:, :1]), ValueError)):
        with pytest.raises(error):
            apply_rotary(q, bad.get("k", k), rot, bad.get("positions"), inplace=True)
    assert q._version == 0 and k._version == 0
    torch.autograd.grad(out, w)
    apply_rotary(q, k, rot, inplace=True)
    assert q._version == 1 and k._version == 1


def test_saved_plan_leaves_its_tables():
    """Tables of devices stay behind, whatever device the plan is loaded for."""
    import copy
    import io

    rot = RotaryEmbedding(8, interleaved=True)
    rot._on[torch.device("cuda", 0)] = torch.zeros(4, dtype=torch.int64)
    buf = io.BytesIO()
    torch.save(rot, buf)
    buf.seek(0)
    for other in (torch.load(buf, map_location="cpu", weights_only=False), copy.deepcopy(rot)):
        assert not other._on and torch.equal(other._turns, rot._turns) and other.interleaved
    assert rot._on


@pytest.mark.gpu
def test_gpu_saved_plan_on_another_device():
    import io

    x = _rand((1, 2, 3, 8), torch.float32, "cuda")
    rot = RotaryEmbedding(8)
    want, buf = apply_rotary(x, None, rot), io.BytesIO()
    torch.save(rot, buf)
    buf.seek(0)
    assert torch.equal(apply_rotary(x, None, torch.load(buf, map_location="cpu", weights_only=False)), want)
