"""Distillation from a teacher's top logits, with its gradient, beside the hard-label loss of
``ops.model_ops.fused_linear_cross_entropy``.

For a token with student logits z and the teacher's top slots (id_j, a_j):

    p    = softmax over the slots of a_j / tau
    kd   = tau^2 sum_j p_j (log p_j - log softmax(z / tau)[id_j])
    ce   = -log softmax(z)[target]
    loss = alpha * kd + (1 - alpha) * ce

A slot with a negative id, or with a teacher logit of -inf, is empty; a token without a slot has no kd, one
whose target is ``ignore_index`` no ce, and a token with neither takes no part (its logits may hold
anything).  A mean is taken for each of the two over the tokens that have it.  CUDA tensors run
``csrc/distill.cu``; CPU tensors run the same mathematics in PyTorch.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .._ext import ext

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_TOP = 1024


def _check(rows, device, vocab, teacher_ids, teacher_logits, targets, temperature, alpha) -> None:
    if teacher_ids.dim() != 2 or teacher_ids.shape[0] != rows or not 1 <= teacher_ids.shape[1] <= MAX_TOP:
        raise ValueError(f"distillation: teacher_ids must be [tokens, top] with the logits' tokens and 1 to {MAX_TOP} "
                         f"slots, got {tuple(teacher_ids.shape)} for {rows} tokens")
    if teacher_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"distillation: teacher_ids must be int64 or int32, got {teacher_ids.dtype}")
    if teacher_logits.shape != teacher_ids.shape:
        raise ValueError("distillation: teacher_logits must have the shape of teacher_ids")
    if teacher_logits.dtype not in _DTYPES and not (teacher_logits.dtype == torch.float64 and device.type == "cpu"):
        raise TypeError(f"distillation: teacher_logits must be bf16, fp16 or fp32, got {teacher_logits.dtype}")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("distillation: the teacher takes no gradient; detach teacher_logits")
    if targets is not None:
        if targets.dtype != torch.int64:
            raise TypeError(f"distillation: targets must be int64, got {targets.dtype}")
        if targets.dim() != 1 or targets.shape[0] != rows:
            raise ValueError(f"distillation: targets must have one entry for each of {rows} tokens")
    for name, t in (("teacher_ids", teacher_ids), ("teacher_logits", teacher_logits), ("targets", targets)):
        if t is not None and t.device != device:
            raise ValueError(f"distillation: {name} must be on the logits' device")
    if vocab < 1:
        raise ValueError("distillation: the vocabulary is empty")
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError(f"distillation: temperature must be from 1e-3 to 1e3, got {temperature}")
    if not 0 <= alpha <= 1:
        raise ValueError(f"distillation: alpha must be from 0 to 1, got {alpha}")
    if targets is None and alpha != 1:
        raise ValueError("distillation: alpha below 1 needs targets")


def _loss_torch(z, ids, teacher, targets, tau, alpha, ignore_index, mean):
    """The definition in PyTorch ops, differentiable; z [N, V]."""
    ct = torch.promote_types(z.dtype, torch.float32)
    z, a = z.to(ct), teacher.to(ct)
    slot = (ids >= 0) & (a != -math.inf)
    if bool((ids >= z.shape[1]).any()):
        raise ValueError("distillation: a teacher id is outside the vocabulary")
    has = slot.any(1)
    soft = has if alpha > 0 else torch.zeros_like(has)
    hard = torch.zeros_like(has) if targets is None or alpha == 1 else targets != ignore_index
    if bool(hard.any()) and bool(((targets < 0) | (targets >= z.shape[1]))[hard].any()):
        raise ValueError("distillation: a target is outside the vocabulary")
    z = torch.where((soft | hard)[:, None], z, torch.zeros((), dtype=ct, device=z.device))  # the rest takes no part
    kd = torch.zeros(z.shape[0], dtype=ct, device=z.device)
    ce = torch.zeros_like(kd)
    if bool(soft.any()):
        s = slot[soft]
        logp = torch.log_softmax((a[soft] / tau).masked_fill(~s, -math.inf), dim=1)
        p = logp.exp()
        logq = torch.log_softmax(z[soft] / tau, dim=1).gather(1, ids[soft].clamp_min(0).long())
        live = p > 0
        terms = p * (logp.masked_fill(~live, 0.0) - logq.masked_fill(~live, 0.0))
        kd = kd.index_put((soft.nonzero()[:, 0],), tau * tau * terms.sum(1))
    if bool(hard.any()):
        ce = ce.index_put((hard.nonzero()[:, 0],), F.cross_entropy(z[hard], targets[hard], reduction="none"))
    if not mean:
        return alpha * kd + (1 - alpha) * ce
    n_ce = 0 if targets is None else int((targets != ignore_index).sum())
    return alpha * kd.sum() / max(1, int(has.sum())) + (1 - alpha) * ce.sum() / max(1, n_ce)


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                      targets: Optional[torch.Tensor] = None, *, temperature: float = 1.0, alpha: float = 1.0,
                      ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """The loss of the module's formulas for ``logits`` [..., vocab] (bf16, fp16, fp32; rows may be views
    of wider ones), ``teacher_ids`` / ``teacher_logits`` [..., top] and ``targets`` [...] (needed for
    ``alpha`` below 1).  fp32: a scalar, or with ``reduction="none"`` one value for each token.

    An id that comes up twice counts with both probabilities.  On CUDA an id or a target outside the
    vocabulary is left out and recorded (``check_device_error``); on the CPU it raises.  With
    ``reduction="mean"`` on bf16 and fp32 the gradient is formed together with the loss and kept for
    one backward pass.
    """
    if logits.is_cuda and reduction in ("mean", "none"):
        try:
            return ext().distill(logits, teacher_ids, teacher_logits, targets, temperature, alpha, ignore_index,
                                 reduction == "mean")
        except (RuntimeError, TypeError):
            _flat(logits, teacher_ids, teacher_logits, targets, temperature, alpha, reduction)  # names what was refused
            raise
    z, ids, a, y = _flat(logits, teacher_ids, teacher_logits, targets, temperature, alpha, reduction)
    loss = _loss_torch(z, ids, a, y, temperature, alpha, ignore_index, reduction == "mean")
    return loss.reshape(logits.shape[:-1]) if reduction == "none" else loss


def _flat(logits, teacher_ids, teacher_logits, targets, temperature, alpha, reduction):
    """The arguments, looked over, with one leading dimension."""
    if reduction not in ("mean", "none"):
        raise ValueError(f"distillation: reduction must be 'mean' or 'none', got {reduction!r}")
    if logits.dim() < 1:
        raise ValueError("distillation: logits must be [..., vocab]")
    if logits.dtype not in _DTYPES and not (logits.dtype == torch.float64 and not logits.is_cuda):
        raise TypeError(f"distillation: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    lead = logits.shape[:-1]
    if teacher_ids.shape[:-1] != lead or (targets is not None and targets.shape != lead):
        raise ValueError(f"distillation: teacher_ids {tuple(teacher_ids.shape)} and targets must have the logits' "
                         f"leading dimensions {tuple(lead)}")
    if teacher_logits.shape != teacher_ids.shape:
        raise ValueError("distillation: teacher_logits must have the shape of teacher_ids")
    V, rows = logits.shape[-1], lead.numel()
    z = logits.reshape(rows, V)
    ids = teacher_ids.reshape(rows, teacher_ids.shape[-1])
    a = teacher_logits.reshape(ids.shape)
    y = None if targets is None else targets.reshape(-1)
    _check(rows, z.device, V, ids, a, y, temperature, alpha)
    return z, ids, a, y


class _LinearDistillFn(torch.autograd.Function):
    """The loss of ``x @ weight.T`` with the logits formed chunk by chunk, like the fused cross entropy:
    per chunk the tcgen05 GEMM for the bf16 logits, the kernel that turns them into their gradient in
    place, and the GEMMs for dX and dW, of which those that are wanted.  The backward only multiplies by
    the incoming gradient."""

    @staticmethod
    def forward(ctx, x, w, ids, teacher, targets, tau, alpha, ignore_index, chunk, want_x, want_w):
        from .linear import EPI_STORE, gemm, mm_dw, mm_fwd

        N, D = x.shape
        V = w.shape[0]
        E = ext()
        # the GEMMs take rows of whole 16-byte vectors: an odd vocabulary gets words of weight zero, whose
        # logits (zero) the loss kernel neither reads nor writes
        pad = -V % 8
        w_dtype, w = w.dtype, F.pad(w, (0, 0, 0, pad)) if pad else w
        counts = E.distill_count(x, V, ids, teacher, targets, ignore_index, alpha)
        rows = torch.empty(N, dtype=torch.float32, device=x.device)
        dx = torch.empty_like(x) if want_x else None
        single = N <= chunk
        dw = None if not want_w else torch.empty(V + pad, D, dtype=w.dtype, device=x.device) if single else \
            torch.zeros(V + pad, D, dtype=torch.float32, device=x.device)
        for s in range(0, N, chunk):
            e = min(N, s + chunk)
            xs = x[s:e]
            (logits,) = mm_fwd(xs, [w])
            E.distill_rows_(logits[:, :V], ids[s:e], teacher[s:e], None if targets is None else targets[s:e], tau, alpha,
                            ignore_index, counts, rows[s:e], want_x or want_w)
            if want_x:
                gemm([logits], [w], False, True, [dx[s:e]], EPI_STORE)
            if want_w:
                mm_dw([logits], xs, [dw], accumulate=s > 0)
        ctx.kept = (dx, dw)
        ctx.vocab, ctx.w_dtype = V, w_dtype
        return E.distill_sum(rows)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if ctx.kept is None:
            raise RuntimeError("fused_linear_distillation: this loss keeps its gradients for one backward pass; its graph "
                               "cannot be gone through a second time")
        dx, dw = ctx.kept
        ctx.kept = None
        s = g.float().reshape(1)
        for d in (dx, dw):
            if d is not None:
                ext().distill_scale_(d, s)
        return (dx, None if dw is None else dw[:ctx.vocab].to(ctx.w_dtype)) + (None,) * 9


def fused_linear_distillation(x: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                              teacher_logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *,
                              temperature: float = 1.0, alpha: float = 1.0, ignore_index: int = -100,
                              chunk: int = 8192) -> torch.Tensor:
    """The mean ``distillation_loss`` of the logits ``x @ weight.T`` without holding them all: x [..., dim],
    weight [vocab, dim], the rest as there.  bf16 CUDA tensors (dim a multiple of 8, a contiguous weight) run this
    library's GEMMs around the in-place loss kernel, ``chunk`` tokens at a time, and form the gradients that are
    wanted (none in an evaluation); others form the logits in one product."""
    if chunk < 1:
        raise ValueError(f"distillation: chunk must be at least 1, got {chunk}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or x.dtype != weight.dtype or x.device != weight.device:
        raise ValueError("distillation: x must be [..., dim] and weight [vocab, dim], of one dtype and device")
    if x.is_cuda and any(t is not None and t.numel() and t.data_ptr() == 0 for t in (x, weight, teacher_ids, teacher_logits, targets)):
        raise RuntimeError("distillation: the kernels take tensors that have memory of their own (of a DTensor, its local tensor)")
    lead = x.shape[:-1]
    if teacher_ids.shape[:-1] != lead or (targets is not None and targets.shape != lead):
        raise ValueError(f"distillation: teacher_ids {tuple(teacher_ids.shape)} and targets must have x's leading "
                         f"dimensions {tuple(lead)}")
    x2 = x.reshape(-1, x.shape[-1])
    if not (x2.is_cuda and x2.dtype == torch.bfloat16 and x2.shape[0] > 0):
        logits = (x2 @ weight.t()).view(*lead, weight.shape[0])
        return distillation_loss(logits, teacher_ids, teacher_logits, targets, temperature=temperature, alpha=alpha,
                                 ignore_index=ignore_index)
    if teacher_logits.shape != teacher_ids.shape:
        raise ValueError("distillation: teacher_logits must have the shape of teacher_ids")
    ids = teacher_ids.reshape(x2.shape[0], teacher_ids.shape[-1])
    a = teacher_logits.reshape(ids.shape)
    y = None if targets is None else targets.reshape(-1)
    _check(x2.shape[0], x2.device, weight.shape[0], ids, a, y, temperature, alpha)
    grad = torch.is_grad_enabled()
    return _LinearDistillFn.apply(x2.contiguous(), weight, ids.contiguous(), a.contiguous(),
                                  None if y is None else y.contiguous(), temperature, alpha, ignore_index, chunk,
                                  grad and x2.requires_grad, grad and weight.requires_grad)
