"""Log probabilities of given tokens, with entropy and top alternatives (sm_100a, with gradients).

    r = token_logprobs(logits, tokens, temperature=1.0, top=8, entropy=True)
    r.logprob        fp32 like tokens: log softmax(logits / temperature) at the token
    r.entropy        fp32 like tokens (None unless asked for)
    r.top_logprobs   fp32 [..., top], falling; r.top_ids int64 [..., top] (None for top = 0)

One kernel reads the logits once (``csrc/kernels/token_logprobs.cu``); neither the
softmax nor fp32 logits are written.  ``logprob``, ``entropy`` and ``top_logprobs`` are
differentiable (one kernel writes the logits' gradient, in their type, rounded
once); the ids are not.

Logits are bf16, fp16 or fp32 [..., V] (any row stride; rows that are not dense are
copied first), tokens int64 [...], top at most 64 and at most V.  Sums are held in fp32.

* A token outside [0, V) is ignored: its logprob is 0 and has no gradient.  Entropy and
  alternatives of its row are computed all the same; where their gradients are absent or 0, the
  row's gradient is 0 whatever its logits are.
* Masked logits: -inf has probability 0; a row of -inf only has logprob -inf, entropy 0, no gradient.
  The type's lowest value is a value like any other: its probability is 0 too unless the row's largest
  is near it, measured in temperatures.  A row of nothing else is uniform; in fp16, where it is -65504,
  it reaches 1e-30 at a temperature of 950.
* Alternatives order by value, equal values by the lowest id.  Where fewer than ``top`` tokens are
  possible, impossible ones follow with logprob -inf.
* Otherwise a row with a NaN or +inf has NaN results and gradients (its ids rank NaN with -inf).

A CUDA graph that records the backward must be the only holder of an autograd
graph of its leaves: drop eager results of the same leaves before the capture.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .._ext import cuda as _cuda

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, top: int = 0,
                   entropy: bool = False) -> TokenLogprobs:
    return TokenLogprobs(*_cuda().token_logprobs(logits, tokens, temperature, top, entropy))
