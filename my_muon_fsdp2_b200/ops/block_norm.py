"""The norms before and after a block, fused with the block's gate and the residual's scale:

    h = residual_scale * x + branch_scale * gate * norm_post(y)
    n = norm_pre(h)

``x`` is the residual stream, ``y`` a block's output (attention or FFN), ``n`` what the next block
reads.  Forward and backward are one pass over the rows each (``csrc/block_norm.cu``,
``csrc/block_norm_bwd.cu``) for bf16, fp16 and fp32 CUDA tensors; CPU tensors run the same mathematics
in PyTorch.  Beside the plain norms of ``ops.model_ops``.
"""
from __future__ import annotations

from typing import Optional

import torch

from .._ext import ext

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_DIM = 8192


def _check_gate(gate: torch.Tensor, x: torch.Tensor) -> None:
    """The gate's leading dimensions are x's up to some dimension, and 1 (or missing altogether) from there on."""
    lead, own = x.shape[:-1], gate.shape[:-1]
    if gate.shape[-1:] == x.shape[-1:]:
        if not own:
            return
        if len(own) == len(lead):
            i = len(lead)
            while i > 0 and own[i - 1] == 1:
                i -= 1
            if own[:i] == lead[:i]:
                return
    raise ValueError(f"gated_residual_norm: gate {tuple(gate.shape)} must be [dim], or x's shape {tuple(x.shape)} with "
                     f"ones in the place of trailing leading dimensions (one gate for each sequence: [batch, 1, dim])")


def _check(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, norm) -> None:
    if norm not in ("rms", "layer"):
        raise ValueError(f"gated_residual_norm: norm must be 'rms' or 'layer', got {norm!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("gated_residual_norm: x must be [..., dim] with dim >= 1")
    if x.shape[-1] > MAX_DIM:
        raise ValueError(f"gated_residual_norm: dim up to {MAX_DIM} is supported, got {x.shape[-1]}")
    if x.dtype not in _DTYPES and not (x.dtype == torch.float64 and not x.is_cuda):
        raise TypeError(f"gated_residual_norm: x must be bf16, fp16 or fp32, got {x.dtype}")
    if y.shape != x.shape:
        raise ValueError(f"gated_residual_norm: y {tuple(y.shape)} must have x's shape {tuple(x.shape)}")
    dtype, device, dim = x.dtype, x.device, x.shape[-1:]
    for name, t in (("y", y), ("post_weight", post_weight), ("post_bias", post_bias), ("gate", gate),
                    ("pre_weight", pre_weight), ("pre_bias", pre_bias)):
        if t is None:
            continue
        if t.dtype != dtype or t.device != device:
            raise TypeError(f"gated_residual_norm: {name} must have x's dtype {dtype} and device {device}")
        if name not in ("y", "gate") and t.shape != dim:
            raise ValueError(f"gated_residual_norm: {name} must be [{dim[0]}], got {tuple(t.shape)}")
    for name, b, w in (("post_bias", post_bias, post_weight), ("pre_bias", pre_bias, pre_weight)):
        if b is not None and (w is None or norm != "layer"):
            raise ValueError(f"gated_residual_norm: {name} needs its weight and norm='layer'")
    if gate is not None:
        _check_gate(gate, x)


def _norm_torch(v, w, b, layer, eps):
    d = v - v.mean(-1, keepdim=True) if layer else v
    u = d * torch.rsqrt(d.square().mean(-1, keepdim=True) + eps) * w
    return u if b is None else u + b


def gated_residual_norm(x: torch.Tensor, y: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
                        post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None, *,
                        norm: str = "rms", eps: float = 1e-5, residual_scale: float = 1.0, branch_scale: float = 1.0):
    """``(h, n)``, or ``h`` alone without ``pre_weight``; see the module's formulas.

    x, y: [..., dim], all tensors of one dtype.  ``post_weight`` [dim] None: y is not normalised.
    ``gate``: [dim], [batch, 1, dim] (one for each sequence) or x's shape (one for each token).
    ``norm``: ``"rms"`` or ``"layer"``, with biases for the latter.  Statistics and sums are fp32, each
    output is rounded once, n is formed from h before its rounding.  Gradients flow to every tensor.
    """
    if x.is_cuda and norm in ("rms", "layer"):
        try:
            return ext().block_norm(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, norm == "layer", eps,
                                    residual_scale, branch_scale)
        except (RuntimeError, TypeError):
            _check(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, norm)  # names what was refused
            raise
    _check(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, norm)
    layer = norm == "layer"
    ct = torch.promote_types(x.dtype, torch.float32)
    up = lambda t: None if t is None else t.to(ct)  # noqa: E731
    p = up(y)
    if post_weight is not None:
        p = _norm_torch(p, up(post_weight), up(post_bias), layer, eps)
    if gate is not None:
        p = p * up(gate)
    h = residual_scale * up(x) + branch_scale * p
    if pre_weight is None:
        return h.to(x.dtype)
    return h.to(x.dtype), _norm_torch(h, up(pre_weight), up(pre_bias), layer, eps).to(x.dtype)

