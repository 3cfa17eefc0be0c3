"""Rotary positions for the attention path (sm_100a, forward and backward).

Each pair of a head's first ``rot_dim`` values turns by position x frequency:
(a, b) -> s (a cos - b sin, a sin + b cos).  The kernel (``csrc/kernels/rotary.cu``)
computes the angles itself, in 64-bit fixed point, from the positions and ``rot_dim / 2``
frequencies, so there is no table and no longest position.

    rope = RotaryPositions(128, scaling="yarn", factor=8, original_len=2048, device="cuda")
    q, k = rotary(q, k, rope, positions)              # new tensors, with gradients
    qkv = rotary_qkv(qkv, B, S, H, rope)              # the packed matrix of ``causal_attention``
    rotary_(q, k, rope, positions)                    # in place, no gradients (decoding)

``mtorus.ops.attention.causal_attention(..., rotary=rope)`` rotates inside the
attention's own forward and backward.

Tensors are bf16, fp16 or fp32, [tokens, heads, dim] or [batch, tokens, heads, dim]
with any strides (rows that are not dense in the head dim are copied first), head
dim at most 512; results are computed in fp32 and rounded once.  ``positions`` is
int64 or int32, [tokens], [batch, tokens] or [1, tokens] ([batch] too, for one token
per sequence); without it token i of a sequence has position ``offset + i`` (both
together are refused).
Positions are read on the device and may be any integer, negative ones included.  An
angle is off by at most 2^-26 of a revolution (its rounding to fp32) and, from the
64-bit frequency, a few 2^-53 of itself; up to positions of about 2^28 the latter is
the smaller, beyond it grows with the position.

A CUDA graph that records the backward must be the only holder of an autograd
graph of its leaves: drop eager results of the same leaves before the capture.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .._ext import cuda as _cuda

LAYOUTS = ("half", "interleaved")
SCALINGS = ("none", "linear", "ntk", "yarn")


class RotaryPositions:
    """Frequencies and layout of rotary positions, built once per model and device.

    head_dim:  values per head; rot_dim (even, default head_dim): the leading values that
               are rotated, the rest passes through.
    layout:    "half" pairs value i with value i + rot_dim / 2, "interleaved" 2i with 2i + 1.
    base:      frequency of pair i is base ** (-2 i / rot_dim).
    scaling:   for contexts longer than the model was trained on, by ``factor``:
               "none" -- frequencies as they are;
               "linear" -- all divided by factor;
               "ntk" -- base multiplied by factor ** (rot_dim / (rot_dim - 2)): the slowest pair is
               divided by factor, the fastest stays;
               "yarn" -- pairs that turn more than beta_fast times within ``original_len`` tokens
               stay, those that turn less than beta_slow times are divided by factor, a linear ramp
               over the pair index lies between; queries and keys are scaled by
               ``attention_scale`` (default 0.1 ln(factor) + 1).
    """

    def __init__(self, head_dim: int, *, rot_dim: Optional[int] = None, base: float = 10000.0, layout: str = "half",
                 scaling: str = "none", factor: float = 1.0, original_len: int = 2048, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attention_scale: Optional[float] = None, device="cuda"):
        rot_dim = head_dim if rot_dim is None else rot_dim
        if not 0 < rot_dim <= head_dim <= 512 or rot_dim % 2:
            raise ValueError(f"rot_dim must be even, at least 2 and at most head_dim, and head_dim at most 512 "
                             f"(got rot_dim {rot_dim}, head_dim {head_dim})")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}, not {layout!r}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}, not {scaling!r}")
        if not (base > 1.0 and math.isfinite(base)):
            raise ValueError(f"base must be finite and above 1, not {base}")
        if not (factor >= 1.0 and math.isfinite(factor)):
            raise ValueError(f"factor must be finite and at least 1, not {factor}")
        if original_len < 1 or not 0.0 < beta_slow < beta_fast:
            raise ValueError("original_len must be at least 1 and 0 < beta_slow < beta_fast")
        self.head_dim, self.rot_dim, self.layout = int(head_dim), int(rot_dim), layout
        self.scaling, self.factor, self.base = scaling, float(factor), float(base)
        self.scale = 1.0
        r, half = self.rot_dim, self.rot_dim // 2
        if scaling == "ntk" and r > 2:
            base = base * factor ** (r / (r - 2))
        freq = [base ** (-2.0 * i / r) for i in range(half)]
        if scaling == "linear":
            freq = [w / factor for w in freq]
        elif scaling == "yarn":
            def pair_of(turns):  # index of the pair that turns so often in original_len tokens
                return r * math.log(original_len / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

            low = max(math.floor(pair_of(beta_fast)), 0)
            high = min(math.ceil(pair_of(beta_slow)), r - 1)
            ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(half)]
            freq = [w / factor * m + w * (1.0 - m) for w, m in zip(freq, ramp)]
            self.scale = 0.1 * math.log(factor) + 1.0 if attention_scale is None else float(attention_scale)
        if scaling != "yarn" and attention_scale is not None:
            self.scale = float(attention_scale)
        if not math.isfinite(self.scale):
            raise ValueError("attention_scale must be finite")
        self.frequencies = freq
        # revolutions per position as 64-bit fixed-point fractions (the bits of a uint64)
        turns = [int(w / (2.0 * math.pi) * 2.0 ** 64) for w in freq]
        self.turns = torch.tensor([t - (t >> 63 << 64) for t in turns], dtype=torch.int64, device=device)
        self.args = (self.turns, self.rot_dim, layout == "interleaved", self.scale)

    def _check(self, dim: int) -> None:
        if dim != self.head_dim:
            raise ValueError(f"these rotary positions are for head dim {self.head_dim}, not {dim}")


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], rope: RotaryPositions,
           positions: Optional[torch.Tensor] = None, *, offset: int = 0
           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotated copies of q and k (k may be None; their head counts may differ); differentiable."""
    rope._check(q.shape[-1])
    return _cuda().rotary(q, k, *rope.args, positions, offset)


def rotary_qkv(qkv: torch.Tensor, B: int, S: int, H: int, rope: RotaryPositions,
               positions: Optional[torch.Tensor] = None, *, kv_heads: Optional[int] = None,
               offset: int = 0) -> torch.Tensor:
    """qkv [B*S, (H + 2 kv_heads) * dim] (q | k | v, heads contiguous) with q and k rotated and v
    copied, as one new matrix; differentiable.  kv_heads defaults to H."""
    return _cuda().rotary_qkv(qkv, B, S, H, H if kv_heads is None else kv_heads, rope.head_dim, *rope.args,
                              positions, offset)


def rotary_(q: torch.Tensor, k: Optional[torch.Tensor], rope: RotaryPositions,
            positions: Optional[torch.Tensor] = None, *, offset: int = 0, inverse: bool = False) -> None:
    """Rotates q and k where they lie (views of a cache or of a packed matrix included: any strides
    with a dense head dim); ``inverse`` undoes that: minus the angle, divided by the attention scale.
    Records no gradient and refuses tensors that require one; values outside the rotated heads are
    not touched.  q and k must not share memory."""
    rope._check(q.shape[-1])
    scale = rope.scale
    if inverse:
        if scale == 0.0:
            raise ValueError("rotary_: an attention scale of 0 cannot be undone")
        scale = 1.0 / scale
    _cuda().rotary_inplace(q, k, *rope.args[:3], scale, positions, offset, inverse)


def rotary_gradient_(dq: torch.Tensor, dk: torch.Tensor, rope: RotaryPositions,
                     positions: Optional[torch.Tensor] = None, *, offset: int = 0) -> None:
    """Turns the gradients of rotated q and k, where they lie, into those of q and k: minus the angle,
    times the attention scale (the transpose of the rotation, where ``rotary_``'s inverse undoes it)."""
    rope._check(dq.shape[-1])
    _cuda().rotary_inplace(dq, dk, *rope.args, positions, offset, True)
