"""Rotary positions beyond the fixed form of ``ops.model_ops.apply_rope``: both pair layouts, a part
of the head, frequencies scaled for long contexts, a position for each token, q and k in one launch.

A pair (x1, x2) of a head at position p becomes ``m (x1 cos a - x2 sin a, x2 cos a + x1 sin a)`` with
``a = p * frequency``; the backward pass is its transpose.  CUDA tensors in bf16, fp16 and fp32 run
``csrc/rotary.cu``; CPU tensors run the same mathematics in PyTorch.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Dict, Optional, Tuple

import torch

from .._ext import ext

_KINDS = ("linear", "ntk", "llama3", "yarn")
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_HEAD_DIM = 256


@dataclass(frozen=True)
class RopeScaling:
    """How the frequencies are changed for contexts longer than the trained one.

    * ``linear``: every frequency divided by ``factor``.
    * ``ntk``: the base becomes ``theta * factor ** (R / (R - 2))`` for ``R`` rotated values, so that
      the slowest pair is stretched by ``factor`` and the fastest not at all.
    * ``llama3``: pairs that turn less than ``low_freq_factor`` times within
      ``original_max_position`` are divided by ``factor``, those with more than
      ``high_freq_factor`` turns kept, the ones between blended linearly in their number of turns.
    * ``yarn``: the blend is a linear ramp over the pair's index, from the pair with ``beta_fast``
      turns (rounded down) to that with ``beta_slow`` (rounded up); cos and sin are multiplied by
      ``magnitude`` (default ``0.1 ln(factor) + 1``).
    """

    kind: str
    factor: float = 1.0
    original_max_position: int = 8192
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    magnitude: Optional[float] = None

    def __post_init__(self):
        if self.kind not in _KINDS:
            raise ValueError(f"RopeScaling: kind must be one of {_KINDS}, got {self.kind!r}")
        if not (math.isfinite(self.factor) and self.factor > 0):
            raise ValueError(f"RopeScaling: factor must be positive and finite, got {self.factor}")
        if self.original_max_position < 1:
            raise ValueError("RopeScaling: original_max_position must be at least 1")
        if not 0 < self.low_freq_factor < self.high_freq_factor:
            raise ValueError("RopeScaling: 0 < low_freq_factor < high_freq_factor is required")
        if not 0 < self.beta_slow < self.beta_fast:
            raise ValueError("RopeScaling: 0 < beta_slow < beta_fast is required")
        if self.magnitude is not None and not math.isfinite(self.magnitude):
            raise ValueError("RopeScaling: magnitude must be finite")


class RotaryEmbedding:
    """The plan of a rotary embedding: its frequencies, computed once in 64 bits.

    ``rotary_dim`` (even, default the whole head) values of each head are rotated, as pairs
    ``(i, i + rotary_dim / 2)`` or, with ``interleaved``, ``(2 i, 2 i + 1)``; the rest passes through.
    The table for a device is laid out at its first use there (``to(device)`` does it ahead of time,
    which a capture into a CUDA graph needs).
    """

    def __init__(self, head_dim: int, theta: float = 10000.0, *, rotary_dim: Optional[int] = None,
                 interleaved: bool = False, scaling: Optional[RopeScaling] = None):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim % 2 or head_dim > MAX_HEAD_DIM:
            raise ValueError(f"RotaryEmbedding: head_dim must be even, from 2 to {MAX_HEAD_DIM}, got {head_dim}")
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError(f"RotaryEmbedding: rotary_dim must be even, from 2 to head_dim {head_dim}, got {rotary_dim}")
        if not (math.isfinite(theta) and theta > 1):
            raise ValueError(f"RotaryEmbedding: theta must be above 1 and finite, got {theta}")
        if scaling is not None and scaling.kind == "ntk" and rotary_dim < 4:
            raise ValueError("RotaryEmbedding: ntk scaling needs a rotary_dim of 4 or more")
        self.head_dim, self.rotary_dim, self.theta = head_dim, rotary_dim, float(theta)
        self.interleaved, self.scaling = bool(interleaved), scaling
        self.frequencies, self.magnitude = self._frequencies()
        # turns per position as 64-bit fixed-point fractions of a turn (kept in int64 bit patterns)
        turns = [int(math.fmod(f / (2 * math.pi), 1.0) * 2**64) for f in self.frequencies]
        with torch.inference_mode(False):
            self._turns = torch.tensor([t - 2**64 if t >= 2**63 else t for t in turns], dtype=torch.int64, device="cpu")
        self._on: Dict[torch.device, torch.Tensor] = {}

    def _frequencies(self) -> Tuple[list, float]:
        """([radians a position for each pair], factor on cos and sin)."""
        R, s, theta = self.rotary_dim, self.scaling, self.theta
        if s is None:
            return [theta ** (-2.0 * i / R) for i in range(R // 2)], 1.0
        if s.kind == "ntk":
            theta = theta * s.factor ** (R / (R - 2))
            return [theta ** (-2.0 * i / R) for i in range(R // 2)], 1.0
        base = [theta ** (-2.0 * i / R) for i in range(R // 2)]
        if s.kind == "linear":
            return [f / s.factor for f in base], 1.0
        if s.kind == "llama3":
            keep = []
            for f in base:
                turns = s.original_max_position * f / (2 * math.pi)
                keep.append(min(1.0, max(0.0, (turns - s.low_freq_factor) / (s.high_freq_factor - s.low_freq_factor))))
            return [k * f + (1.0 - k) * f / s.factor for f, k in zip(base, keep)], 1.0

        def index_of(turns: float) -> float:  # the (real) index of the pair with that many turns
            return R * math.log(s.original_max_position / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo = max(0, math.floor(index_of(s.beta_fast)))
        hi = min(R - 1, math.ceil(index_of(s.beta_slow)))
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(R // 2)]
        m = s.magnitude if s.magnitude is not None else (0.1 * math.log(s.factor) + 1.0 if s.factor > 1 else 1.0)
        return [r * f / s.factor + (1.0 - r) * f for f, r in zip(base, ramp)], m

    def __getstate__(self):
        # a saved or copied plan lays its tables out anew: loaded onto another device they would be on the wrong one
        return {**self.__dict__, "_on": {}}

    def to(self, device) -> "RotaryEmbedding":
        self._table(torch.device(device))
        return self

    def _table(self, device: torch.device) -> torch.Tensor:
        t = self._on.get(device)
        if t is None:
            if device.type == "cuda" and device.index is None:
                return self._table(torch.device("cuda", torch.cuda.current_device()))
            # a table first used in inference mode is one that a later training step saves for its backward
            with torch.inference_mode(False):
                t = self._on[device] = self._turns.to(device)
        return t

    def cos_sin(self, positions: torch.Tensor, dtype=torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """(magnitude cos a, magnitude sin a) [..., rotary_dim / 2] at integer ``positions``; the angles
        are formed in 64 bits."""
        f = torch.tensor(self.frequencies, dtype=torch.float64, device=positions.device)
        a = positions[..., None].double() * f
        return (a.cos() * self.magnitude).to(dtype), (a.sin() * self.magnitude).to(dtype)


def _rotate_torch(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, rot: RotaryEmbedding) -> torch.Tensor:
    """x [..., T, H, D], cos and sin [..., T, R / 2]."""
    R = rot.rotary_dim
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    r = x[..., :R].to(c.dtype)
    if rot.interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    r = r.to(x.dtype)
    return r if R == x.shape[-1] else torch.cat((r, x[..., R:]), dim=-1)


def _check(q, k, rot, positions, inplace) -> None:
    if not isinstance(rot, RotaryEmbedding):
        raise TypeError("apply_rotary: rotary must be a RotaryEmbedding")
    for name, x in (("q", q), ("k", k)):
        if x is None and name == "k":
            continue
        if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4):
            raise ValueError(f"apply_rotary: {name} must be a [batch, seq, heads, head_dim] or [tokens, heads, head_dim] tensor")
        if x.dtype not in _DTYPES and not (x.dtype == torch.float64 and not x.is_cuda):
            raise TypeError(f"apply_rotary: {name} must be bf16, fp16 or fp32, got {x.dtype}")
        if x.shape[-1] != rot.head_dim:
            raise ValueError(f"apply_rotary: {name} has head_dim {x.shape[-1]}, the rotary embedding {rot.head_dim}")
    if k is not None and (k.shape[:-2] != q.shape[:-2] or k.dtype != q.dtype or k.device != q.device):
        raise ValueError("apply_rotary: q and k must have the same batch, sequence, dtype and device")
    if positions is not None:
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"apply_rotary: positions must be int64 or int32, got {positions.dtype}")
        if positions.device != q.device:
            raise ValueError("apply_rotary: positions must be on q's device")
        lead = q.shape[:-2]
        if positions.dim() < 1 or positions.dim() > len(lead) or \
                any(p not in (1, n) for p, n in zip(reversed(positions.shape), reversed(lead))):
            raise ValueError(f"apply_rotary: positions {tuple(positions.shape)} do not broadcast to {tuple(lead)}")
    if inplace:
        for x in (q, k):
            if x is None:
                continue
            if torch.is_grad_enabled() and x.requires_grad:
                raise RuntimeError("apply_rotary: inplace=True is for tensors outside autograd")
            if x.stride(-1) != 1 or any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
                raise ValueError("apply_rotary: inplace=True needs contiguous heads in memory of their own")
        if k is not None and q.numel() and q.data_ptr() == k.data_ptr():
            raise ValueError("apply_rotary: inplace=True needs q and k in memory of their own")


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], rotary: RotaryEmbedding,
                 positions: Optional[torch.Tensor] = None, inplace: bool = False):
    """Rotate q and k (None: q alone); returns ``(q, k)``, or ``q`` when k is None.

    q: [batch, seq, q_heads, head_dim] or [tokens, q_heads, head_dim], k the same with its own number
    of heads; any strides (views of a packed projection need no copy).  ``positions``: int64 or int32,
    broadcast over the leading dimensions (default 0, 1, ... along the sequence; any value, also
    negative).  ``inplace`` writes into q and k, which must not overlap (no gradient): the form for new
    tokens that go to a cache.  With autograd the results are new contiguous tensors.
    """
    if isinstance(q, torch.Tensor) and q.is_cuda and isinstance(rotary, RotaryEmbedding):
        try:
            return ext().rotary(q, k, positions, rotary._table(q.device), rotary.head_dim, rotary.rotary_dim,
                                rotary.interleaved, rotary.magnitude, inplace)
        except (RuntimeError, TypeError):
            _check(q, k, rotary, positions, inplace)  # names what was refused
            raise
    _check(q, k, rotary, positions, inplace)
    pos = torch.arange(q.shape[-3], device=q.device) if positions is None else positions
    cos, sin = rotary.cos_sin(pos, torch.float64 if q.dtype == torch.float64 else torch.float32)
    out = [_rotate_torch(x, cos, sin, rotary) for x in (q, k) if x is not None]
    if inplace:
        out = [x.copy_(o) for x, o in zip((q, k), out)]
    return tuple(out) if k is not None else out[0]
