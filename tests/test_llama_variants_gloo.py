"""A student Llama (scaled rotary positions, norms on both sides of the blocks with gates, distillation as the
loss) trained on 2 gloo ranks under FSDP2 and under the fused-FSDP linears, through the Trainer.  The trained
weights must match one process that trains on the union of the ranks' micro-batches."""
import pytest
import torch

from tests.conftest import rel_err
from tests.dist_util import run_ranks

pytestmark = pytest.mark.distributed

ACCUM, MB, SEQ, STEPS, TOP = 2, 2, 16, 2, 5


def _build():
    from my_muon_fsdp2_b200.models.llama import Llama, LlamaConfig
    from my_muon_fsdp2_b200.ops.rotary import RopeScaling

    torch.manual_seed(0)
    return Llama(LlamaConfig.tiny(dim=64, n_heads=4, n_kv_heads=2, ffn_dim=128, vocab_size=96, n_layers=2, rotary_dim=8,
                                  rope_scaling=RopeScaling("yarn", 4.0, 64), post_norms=True, block_gates=True,
                                  residual_scale=0.9, branch_scale=0.7))


def _batch(step, rank):
    """Every token has slots and a target, so that the mean over ranks is the mean over their union."""
    g = torch.Generator().manual_seed(1000 * step + rank)
    return (torch.randint(0, 96, (ACCUM, MB, SEQ + 1), generator=g),
            (torch.randint(0, 96, (ACCUM, MB, SEQ, TOP), generator=g), torch.randn(ACCUM, MB, SEQ, TOP, generator=g)))


def _trainer(model, **kw):
    from my_muon_fsdp2_b200 import FusedAdamW, MuonOptimizer
    from my_muon_fsdp2_b200.train import Trainer

    names = set(model.muon_param_names())
    opts = [MuonOptimizer([p for n, p in model.named_parameters() if n in names], lr=0.02, weight_decay=0.01),
            FusedAdamW([p for n, p in model.named_parameters() if n not in names], lr=1e-3)]
    return Trainer(model, opts, grad_accum=ACCUM, device="cpu", max_grad_norm=1.0, temperature=2.0, alpha=0.6, **kw)


def _ranked(rank, world, mode):
    from my_muon_fsdp2_b200.models.llama import apply_fsdp
    from my_muon_fsdp2_b200.parallel.symm_fsdp import apply_symm_fsdp

    model = _build()
    (apply_symm_fsdp if mode == "symm" else apply_fsdp)(model)
    trainer = _trainer(model, keep_gathered=True)
    losses = [trainer.train_step(*_batch(s, rank)) for s in range(STEPS)]
    full = lambda t: t.full_tensor() if hasattr(t, "full_tensor") else t  # noqa: E731
    return {"loss": losses[0], "params": {n: full(p.detach()).clone() for n, p in model.named_parameters()}}


@pytest.mark.parametrize("mode", ["fsdp2", "symm"])
def test_student_matches_single_process(mode):
    world = 2
    got = run_ranks(_ranked, world, mode)
    ref = _build()
    trainer = _trainer(ref)
    for s in range(STEPS):
        (t0, (i0, a0)), (t1, (i1, a1)) = _batch(s, 0), _batch(s, 1)
        trainer.train_step(torch.cat([t0, t1], 1), (torch.cat([i0, i1], 1), torch.cat([a0, a1], 1)))
    params = dict(ref.named_parameters())
    assert sum("gate" in n or "post_norm" in n for n in params) == 8 and set(params) == set(got["params"])
    for n, p in params.items():
        assert rel_err(got["params"][n], p.detach()) < 1e-4, n
