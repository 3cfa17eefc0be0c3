"""Residual update of a block fused with the norms around it (sm_100a, forward and backward).

    y = residual_scale * x + branch_scale * gate * norm(branch; post_weight)
    n = norm(y; pre_weight)

with norm(v; w) = v / sqrt(mean(v^2) + eps) * w over the last dim (RMS norm).  One
kernel (``csrc/kernels/residual_norm.cu``) reads x and the branch and writes the
residual stream y and the next branch's input n; the backward is one kernel and a
small sum of the weights' partial gradients.  Every part but the sum is optional:
without ``post_weight`` the branch enters as it is, without ``gate`` it is not gated,
without ``pre_weight`` only y is computed.  ``rms_norm`` is the norm alone.

x and branch are bf16, fp16 or fp32 [..., d] with d up to 16384 (any strides; rows
that are not dense are copied first); the weights are fp32 master parameters [d].
``gate`` is an fp32 vector [d] (per channel), fp32 [..., 1] (per row), or of x's
shape and type (per element).  Arithmetic is fp32: the statistics, n and all gradients
see y before its rounding.  Weight gradients are summed in a fixed order, so
results repeat bit for bit.

A CUDA graph that records the backward must be the only holder of an autograd
graph of its leaves: drop eager results of the same leaves before the capture.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .._ext import cuda as _cuda


def residual_norm(x: torch.Tensor, branch: torch.Tensor, *, pre_weight: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  residual_scale: float = 1.0, branch_scale: float = 1.0, eps: float = 1e-6
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """-> (y, n); n is None without ``pre_weight``.  Differentiable in every tensor."""
    return _cuda().residual_norm(x, branch, pre_weight, post_weight, gate, residual_scale, branch_scale, eps)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last dim (the first norm of a model, which has no
    branch before it).  Differentiable."""
    return _cuda().rms_norm(x, weight, eps)
