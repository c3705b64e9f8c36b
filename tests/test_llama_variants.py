"""The Llama blocks with the options of ``ops.rotary``, ``ops.block_norm`` and ``ops.distill`` together, as a
student is trained: scaled partial rotary positions given for each token, norms on both sides of each
block with gates, distillation from a teacher's top logits."""
import math

import pytest
import torch
import torch.nn.functional as F

from my_muon_fsdp2_b200.models.llama import Llama, LlamaConfig
from my_muon_fsdp2_b200.ops.rotary import RopeScaling

VARIANT = dict(dim=256, n_heads=4, n_kv_heads=2, ffn_dim=512, vocab_size=1000, rope_scaling=RopeScaling("llama3", 8.0, 64),
               rotary_dim=32, rope_interleaved=True, post_norms=True, block_gates=True, residual_scale=0.9, branch_scale=0.7)


def _student(dtype, device, **kw):
    torch.manual_seed(0)
    model = Llama(LlamaConfig.tiny(**{**VARIANT, **kw}))
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(torch.randn_like(p) * (0.1 if p.dim() == 1 else 0.05) + (1.0 if p.dim() == 1 else 0.0))
            p.copy_(p.bfloat16())  # the same values in every dtype
    return model.to(device, dtype)


def _batch(device, B=2, T=48, K=6, vocab=1000):
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, vocab, (B, T + 1), generator=g)
    ids = torch.randint(0, vocab, (B, T, K), generator=g)
    ids[0, :5], ids[1, 7, 3:] = -1, -1
    logits = torch.randn(B, T, K, generator=g) * 2
    positions = torch.arange(T) + torch.tensor([[0], [1000]])
    targets = tokens[:, 1:].clone()
    targets[1, -4:] = -100
    return [t.to(device) for t in (tokens[:, :-1], targets, positions, ids, logits)]


def _loss(model, batch):
    tokens, targets, positions, ids, logits = batch
    return model(tokens, targets, positions=positions, teacher=(ids, logits), temperature=2.0, alpha=0.6)


def _by_hand(model, batch):
    """The same student written out from plain PyTorch ops, in the model's dtype (CPU)."""
    c, (tokens, targets, positions, ids, logits) = model.cfg, batch
    B, T = tokens.shape
    rms = lambda v, w: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + c.norm_eps) * w  # noqa: E731
    R, hd = c.rotary_dim, c.head_dim
    f = [c.rope_theta ** (-2.0 * i / R) for i in range(R // 2)]
    keep = [min(1.0, max(0.0, (64 * v / (2 * math.pi) - 1) / 3)) for v in f]
    f = torch.tensor([k * v + (1 - k) * v / 8 for v, k in zip(f, keep)], dtype=torch.float64)
    turn = torch.polar(torch.ones(()).double(), positions.double()[..., None, None] * f)

    def rope(x):
        r = torch.view_as_real(torch.view_as_complex(x[..., :R].unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        return torch.cat([r, x[..., R:]], -1)

    x = model.tok_embeddings.weight[tokens]
    for l in model.layers:
        n, a = rms(x, l.attention_norm.weight), l.attention
        q = rope(F.linear(n, a.wq.weight).view(B, T, c.n_heads, hd)).transpose(1, 2)
        k = rope(F.linear(n, a.wk.weight).view(B, T, c.n_kv_heads, hd)).transpose(1, 2).repeat_interleave(2, 1)
        v = F.linear(n, a.wv.weight).view(B, T, c.n_kv_heads, hd).transpose(1, 2).repeat_interleave(2, 1)
        s = (q @ k.transpose(2, 3)) / math.sqrt(hd) + torch.full((T, T), -math.inf, dtype=x.dtype).triu(1)
        y = F.linear((s.softmax(-1) @ v).transpose(1, 2).reshape(B, T, -1), a.wo.weight)
        x = c.residual_scale * x + c.branch_scale * l.attention_gate * rms(y, l.attention_post_norm.weight)
        n, m = rms(x, l.ffn_norm.weight), l.feed_forward
        y = F.linear(F.silu(F.linear(n, m.w1.weight)) * F.linear(n, m.w3.weight), m.w2.weight)
        x = c.residual_scale * x + c.branch_scale * l.ffn_gate * rms(y, l.ffn_post_norm.weight)
    z = F.linear(rms(x, model.norm.weight), model.output.weight)
    has = (ids >= 0).any(-1)
    p = torch.softmax((logits.to(z.dtype) / 2).masked_fill(ids < 0, -math.inf)[has], -1)
    logq = torch.log_softmax(z / 2, -1).gather(-1, ids.clamp_min(0))[has]
    kd = 4 * (torch.xlogy(p, p) - p * logq).sum() / has.sum()
    return 0.6 * kd + 0.4 * F.cross_entropy(z.flatten(0, 1), targets.flatten(), ignore_index=-100)


def test_student_is_the_written_out_composition():
    """In 64 bits, but for the plain norms (before the attention and at the end), which round their input and
    result to fp32 on the CPU: 2^-24 at five places, each into a loss of 16 terms or a gradient: 1e-6."""
    model, batch = _student(torch.float64, "cpu"), _batch("cpu")
    got, want = _loss(model, batch), _by_hand(model, batch)
    assert abs(got.item() - want.item()) < 1e-6 * abs(want.item())
    params = dict(model.named_parameters())
    assert {n.split(".", 2)[-1] for n in params if "gate" in n or "post_norm" in n} == {
        "attention_gate", "ffn_gate", "attention_post_norm.weight", "ffn_post_norm.weight"}
    for n, a, b in zip(params, torch.autograd.grad(got, list(params.values())), torch.autograd.grad(want, list(params.values()))):
        assert (a - b).norm() <= 1e-6 * b.norm(), n


def test_options_off_is_the_plain_block():
    """post_norms with unit weights and scales differ from the plain block; positions 0..T-1 do not."""
    torch.manual_seed(0)
    model = Llama(LlamaConfig.tiny()).double()
    tokens = torch.randint(0, 512, (2, 16))
    want = model(tokens)
    assert torch.allclose(model(tokens, positions=torch.arange(16)), want, atol=1e-5)
    assert not torch.allclose(model(tokens, positions=2 * torch.arange(16)), want, atol=1e-3)
    with pytest.raises(ValueError):
        LlamaConfig.tiny(block_gates=True)
    cfg = LlamaConfig.tiny(**VARIANT)
    assert cfg.num_params() == sum(p.numel() for p in Llama(cfg).parameters())
    m = Llama(cfg)
    m.init_weights()
    assert all(bool((p == 1).all()) for n, p in m.named_parameters() if n.endswith("_gate") or "norm" in n)
    assert not any("gate" in n or "norm" in n for n in m.muon_param_names())


def test_trainer_distils_on_cpu():
    from my_muon_fsdp2_b200.train import Trainer

    model = _student(torch.float32, "cpu", n_layers=1)
    batch = _batch("cpu")
    tokens = torch.cat([batch[0], batch[1].clamp_min(0)[:, -1:]], 1)
    host, teacher = tokens[None].repeat(2, 1, 1), (batch[3][None].repeat(2, 1, 1, 1), batch[4][None].repeat(2, 1, 1, 1))
    tr = Trainer(model, [torch.optim.SGD(model.parameters(), lr=0.0)], grad_accum=2, temperature=2.0, alpha=0.5)
    want = model(tokens[:, :-1], tokens[:, 1:], teacher=(batch[3], batch[4]), temperature=2.0, alpha=0.5)
    assert abs(tr.train_step(host, teacher) - want.item()) < 1e-5 * abs(want.item())
    assert abs(tr.train_step(host) - model(tokens[:, :-1], tokens[:, 1:]).item()) < 1e-5 * abs(want.item())


def test_gpt2_distils_on_cpu():
    from my_muon_fsdp2_b200.models.gpt2 import GPTConfig, GPTModel
    from my_muon_fsdp2_b200.ops.distill import distillation_loss

    torch.manual_seed(0)
    model = GPTModel(GPTConfig(vocab_size=101, n_positions=16, n_embd=32, n_layer=1, n_head=2))
    x, ids, a = torch.randint(0, 101, (2, 9)), torch.randint(0, 101, (2, 9, 4)), torch.randn(2, 9, 4)
    got = model(x, teacher=(ids, a), temperature=1.5)
    assert torch.allclose(got, distillation_loss(model(x), ids, a, temperature=1.5), atol=1e-6)


@pytest.mark.gpu
def test_gpu_student_and_its_gradients():
    """bf16 kernels against the fp64 composition.  Some 14 tensors a layer are rounded on the way forward and
    as many back, two layers and the head: about 60 roundings of 2^-9 that add up as sqrt(60) 2^-9 = 1.5 %
    of a gradient's norm; each enters with a factor of at most about 3 (norms, softmax): 5 %."""
    ref, batch = _student(torch.float64, "cpu"), _batch("cpu")
    want = _by_hand(ref, batch)
    names = [n for n, _ in ref.named_parameters()]
    wg = torch.autograd.grad(want, list(ref.parameters()))
    model, gb = _student(torch.bfloat16, "cuda"), _batch("cuda")
    loss = _loss(model, gb)
    assert abs(loss.item() - want.item()) < 0.01 * abs(want.item())
    for n, g, w in zip(names, torch.autograd.grad(loss, list(model.parameters())), wg):
        rel = ((g.double().cpu() - w).norm() / w.norm()).item()
        assert rel < 0.05, f"{n}: {rel:.3g}"


@pytest.mark.gpu
def test_gpu_positions_given_are_the_epilogue_rope():
    """Positions 0..T-1 through ops.rotary and the RoPE of the projections' epilogue: the same logits but for
    roundings (q and k are rounded once more in between: 2^-9 of them, in scores of size about 1)."""
    torch.manual_seed(0)
    model = Llama(LlamaConfig.tiny(dim=256, n_heads=4, n_kv_heads=2, ffn_dim=512)).to("cuda", torch.bfloat16)
    model.init_weights()
    tokens = torch.randint(0, 512, (2, 64), device="cuda")
    a, b = model(tokens), model(tokens, positions=torch.arange(64, device="cuda"))
    assert ((a - b).float().norm() / a.float().norm()).item() < 0.02


@pytest.mark.gpu
def test_gpu_training_step_in_a_graph():
    """Forward and backward of the student captured once and replayed on new tokens: the eager step's bits."""
    model, batch = _student(torch.bfloat16, "cuda"), _batch("cuda")
    params = list(model.parameters())

    def step():
        loss = _loss(model, batch)
        return (loss.detach(),) + torch.autograd.grad(loss, params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    batch[0].copy_(batch[0].flip(1))
    batch[2].add_(5)
    g.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_gpu_gpt2_distils_with_its_odd_vocabulary():
    from my_muon_fsdp2_b200.models.gpt2 import GPTConfig, GPTModel

    torch.manual_seed(0)
    cfg = GPTConfig(vocab_size=1003, n_positions=32, n_embd=128, n_layer=1, n_head=2)
    ref = GPTModel(cfg)
    with torch.no_grad():
        for p in ref.parameters():
            p.copy_(p.bfloat16())
    ref = ref.double()
    x, ids, a = torch.randint(0, 1003, (2, 24)), torch.randint(0, 1003, (2, 24, 4)), torch.randn(2, 24, 4)
    want = ref(x, x, teacher=(ids, a), temperature=2.0, alpha=0.5)
    wg = torch.autograd.grad(want, list(ref.parameters()))
    model = GPTModel(cfg).to("cuda", torch.bfloat16)
    model.load_state_dict(ref.state_dict())
    loss = model(x.cuda(), x.cuda(), teacher=(ids.cuda(), a.cuda()), temperature=2.0, alpha=0.5)
    assert abs(loss.item() - want.item()) < 0.01 * abs(want.item())
    for (n, _), g, w in zip(ref.named_parameters(), torch.autograd.grad(loss, list(model.parameters())), wg):
        if "c_attn.bias" in n:
            continue  # the key bias has no gradient but for roundings
        assert ((g.double().cpu() - w).norm() / w.norm()).item() < 0.05, n


class _Wrapper(torch.Tensor):
    """A tensor with a device and a shape, and no memory, as a DTensor is."""

    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        return cls(*args[0].shape, dtype=args[0].dtype)


def _wrappers_are_refused(device, rotary, norm, loss, fused):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, device=device, dtype=dtype)  # noqa: E731
    bf, ids = torch.bfloat16, torch.zeros(4, 2, dtype=torch.long, device=device)
    w = _Wrapper
    for call in (lambda: rotary(w(1, 2, 3, 8), z(1, 2, 1, 8), None), lambda: rotary(z(1, 2, 3, 8), w(1, 2, 1, 8), None),
                 lambda: rotary(z(1, 2, 3, 8), z(1, 2, 1, 8), w(2, dtype=torch.long)),
                 lambda: norm(w(4, 8), z(4, 8), z(8), z(8), z(8)), lambda: norm(z(4, 8), w(4, 8), z(8), z(8), z(8)),
                 lambda: norm(z(4, 8), z(4, 8), w(8), z(8), z(8)), lambda: norm(z(4, 8), z(4, 8), z(8), w(8), z(8)),
                 lambda: norm(z(4, 8), z(4, 8), z(8), z(8), w(8)), lambda: loss(w(4, 16), ids, z(4, 2)),
                 lambda: loss(z(4, 16), w(4, 2, dtype=torch.long), z(4, 2)), lambda: loss(z(4, 16), ids, w(4, 2)),
                 lambda: fused(w(4, 8, dtype=bf), w(16, 8, dtype=bf), ids, z(4, 2))):
        with pytest.raises(RuntimeError, match="memory of their own"):
            call()


def test_wrappers_without_memory_are_refused_by_the_entries():
    """Before anything is read or launched; the entries look at this first, wherever the tensors are."""
    from my_muon_fsdp2_b200._ext import available, ext
    from my_muon_fsdp2_b200.ops.distill import fused_linear_distillation
    from my_muon_fsdp2_b200.ops.rotary import RotaryEmbedding

    if not available():
        pytest.skip("the extension is not built")
    E, turns = ext(), RotaryEmbedding(8)._turns
    _wrappers_are_refused("cpu", lambda q, k, pos: E.rotary(q, k, pos, turns, 8, 8, False, 1.0, False),
                          lambda x, y, pw, gate, nw: E.block_norm(x, y, pw, None, gate, nw, None, False, 1e-5, 1.0, 1.0),
                          lambda z, ids, a: E.distill(z, ids, a, None, 1.0, 1.0, -100, True), fused_linear_distillation)


@pytest.mark.gpu
def test_gpu_wrappers_without_memory_are_refused():
    from my_muon_fsdp2_b200.ops.block_norm import gated_residual_norm
    from my_muon_fsdp2_b200.ops.distill import distillation_loss, fused_linear_distillation
    from my_muon_fsdp2_b200.ops.rotary import RotaryEmbedding, apply_rotary

    rot = RotaryEmbedding(8).to("cuda")
    x, w = torch.zeros(4, 8, device="cuda", dtype=torch.bfloat16), _Wrapper(16, 8, dtype=torch.bfloat16)
    _wrappers_are_refused("cuda", lambda q, k, pos: apply_rotary(q, k, rot, pos),
                          lambda x, y, pw, gate, nw: gated_residual_norm(x, y, pw, gate=gate, pre_weight=nw), distillation_loss,
                          fused_linear_distillation)
    with pytest.raises(RuntimeError, match="memory of their own"):
        fused_linear_distillation(x, w, torch.zeros(4, 2, dtype=torch.long, device="cuda"), torch.zeros(4, 2, device="cuda"))


@pytest.mark.gpu
def test_gpu_trainer_distils():
    """A Trainer's step from host batches: the loss and the gradients of its micro-batches, taken one by one."""
    from my_muon_fsdp2_b200.train import Trainer

    model, batch = _student(torch.bfloat16, "cuda"), _batch("cpu")
    tokens = torch.cat([batch[0], batch[1].clamp_min(0)[:, -1:]], 1)
    host = torch.stack([tokens, tokens.flip(0)])
    teacher = (torch.stack([batch[3], batch[3].flip(0)]), torch.stack([batch[4], batch[4].flip(0).half().float()]))
    want, grads = 0.0, [torch.zeros_like(p, dtype=torch.float64) for p in model.parameters()]
    for i in range(2):
        t = host[i].cuda()
        loss = model(t[:, :-1], t[:, 1:], teacher=tuple(x[i].cuda() for x in teacher), temperature=2.0, alpha=0.5)
        want += loss.item() / 2
        for s, g in zip(grads, torch.autograd.grad(loss, list(model.parameters()))):
            s += g.double() / 2
    tr = Trainer(model, [torch.optim.SGD(model.parameters(), lr=0.0)], grad_accum=2, temperature=2.0, alpha=0.5)
    kept = {}
    for n, p in model.named_parameters():
        p.register_post_accumulate_grad_hook(lambda p, n=n: kept.__setitem__(n, p.grad.clone()))
    got = tr.train_step(host, teacher)
    assert abs(got - want) < 1e-5 * abs(want)  # the sum of two fp32 losses
    for (n, p), g in zip(model.named_parameters(), grads):
        # halving is exact; the sum of two bf16 gradients is rounded once more
        assert (kept[n].double() - g).norm() <= 2**-8 * g.norm(), n


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [True, False], ids=["reentrant", "not_reentrant"])
def test_gpu_operators_in_a_checkpoint(reentrant):
    """Activations formed again in the backward, or kept on the host: the gradients of the plain call, bit by bit."""
    from torch.utils.checkpoint import checkpoint

    from my_muon_fsdp2_b200.ops.block_norm import gated_residual_norm
    from my_muon_fsdp2_b200.ops.distill import distillation_loss, fused_linear_distillation
    from my_muon_fsdp2_b200.ops.rotary import RotaryEmbedding, apply_rotary

    g = torch.Generator().manual_seed(0)
    rot = RotaryEmbedding(16)
    pos = torch.arange(6, device="cuda") + 3
    ids, a = torch.randint(0, 64, (4, 6, 3), generator=g).cuda(), torch.randn(4, 6, 3, generator=g).cuda()
    y = torch.randint(0, 64, (4, 6), generator=g).cuda()
    leaves = [torch.randn(s, generator=g).to("cuda", torch.bfloat16).requires_grad_() for s in ((4, 6, 16), (4, 6, 16), (16,), (64, 16))]

    def student(x, z, w, head):
        h, n = gated_residual_norm(x, z, w, gate=w, pre_weight=w)
        q = apply_rotary(n.view(4, 6, 1, 16), None, rot, pos).view(4, 6, 16) + h
        logits = q @ head.t()
        kd = dict(targets=y, temperature=2.0, alpha=0.5)
        return fused_linear_distillation(q, head, ids, a, **kd) + distillation_loss(logits, ids, a, **kd) \
            + distillation_loss(logits, ids, a, reduction="none", **kd).sum() + distillation_loss(logits.half(), ids, a, **kd)

    want = torch.autograd.grad(student(*leaves), leaves)
    got = [t.detach().clone().requires_grad_() for t in leaves]
    checkpoint(student, *got, use_reentrant=reentrant).backward()
    assert all(torch.equal(t.grad, w) for t, w in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        loss = student(*leaves)
    assert all(torch.equal(t, w) for t, w in zip(torch.autograd.grad(loss, leaves), want))
