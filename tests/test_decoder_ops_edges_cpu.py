"""More refusals of the decoder operators, and what their callers pass on (no GPU)."""
import pytest
import torch

from mtorus.ops.rotary import RotaryPositions, rotary_

BF = torch.bfloat16


def _rope(**kw):
    return RotaryPositions(64, device="cpu", **kw)


def test_rotary_inverse_of_a_zero_scale_is_refused():
    q = torch.zeros(5, 4, 64, dtype=BF)
    with pytest.raises(ValueError, match="cannot be undone"):
        rotary_(q, None, _rope(attention_scale=0.0), inverse=True)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_(q, None, _rope(attention_scale=0.0))
