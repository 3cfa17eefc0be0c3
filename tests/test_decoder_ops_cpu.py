"""Refusals and host-side set-up of the rotary, residual norm and log probability operators (no GPU)."""
import math

import pytest
import torch

from mtorus.ops.attention import causal_attention
from mtorus.ops.logprobs import token_logprobs
from mtorus.ops.residual_norm import residual_norm, rms_norm
from mtorus.ops.rotary import RotaryPositions, rotary, rotary_, rotary_qkv

BF = torch.bfloat16


def _rope(**kw):
    return RotaryPositions(64, device="cpu", **kw)


@pytest.mark.parametrize("kw", [dict(rot_dim=3), dict(rot_dim=66), dict(rot_dim=0), dict(layout="pairs"),
                                dict(scaling="dynamic"), dict(base=1.0), dict(base=float("inf")), dict(factor=0.5),
                                dict(factor=float("nan")), dict(original_len=0), dict(beta_fast=1.0, beta_slow=2.0),
                                dict(attention_scale=float("inf"))])
def test_rotary_positions_refuses(kw):
    with pytest.raises(ValueError):
        _rope(**kw)


def test_rotary_positions_head_dim_limit():
    with pytest.raises(ValueError, match="at most 512"):
        RotaryPositions(514, device="cpu")


def test_rotary_frequencies():
    w = [10000.0 ** (-2.0 * i / 64) for i in range(32)]
    assert _rope().frequencies == w and _rope().scale == 1.0
    assert _rope(scaling="linear", factor=4).frequencies == [x / 4 for x in w]
    ntk = _rope(scaling="ntk", factor=4).frequencies
    assert ntk[0] == 1.0 and abs(ntk[-1] * 4 / w[-1] - 1) < 1e-12  # fastest stays, slowest is divided by the factor
    r = _rope(scaling="yarn", factor=8, original_len=2048)
    turns = [2048 * x / (2 * math.pi) for x in w]
    assert r.scale == 0.1 * math.log(8) + 1.0
    assert r.frequencies[0] == w[0] and r.frequencies[-1] == w[-1] / 8
    for f, x, t in zip(r.frequencies, w, turns):
        assert x / 8 <= f <= x
        if t > 40:
            assert f == x
        if t < 0.8:
            assert f == x / 8
    assert _rope(rot_dim=2, scaling="ntk", factor=4).frequencies == [1.0]
    for t, x in zip(_rope().turns.tolist(), w):  # 64-bit fixed-point fractions of a revolution
        assert abs(t / 2.0 ** 64 - x / (2 * math.pi)) <= 2.0 ** -53 * x + 2.0 ** -64


def test_rotary_refuses():
    rope = _rope()
    q, k = torch.zeros(2, 5, 4, 64, dtype=BF), torch.zeros(2, 5, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match="head dim 64"):
        rotary(torch.zeros(5, 4, 32, dtype=BF), None, rope)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        rotary(q.double(), None, rope)
    with pytest.raises(TypeError, match="but k is"):
        rotary(q, k.float(), rope)
    with pytest.raises(ValueError, match="heads only"):
        rotary(q, k[:, :4], rope)
    with pytest.raises(ValueError, match="dim"):
        rotary(torch.zeros(64, dtype=BF), None, rope)
    with pytest.raises(TypeError, match="positions must be"):
        rotary(q, k, rope, torch.zeros(2, 5))
    for shape in [(4,), (3, 5), (2, 4), (5, 2), (2, 5, 1), (1,)]:
        with pytest.raises(ValueError, match="positions"):
            rotary(q, k, rope, torch.zeros(shape, dtype=torch.long))
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary(q, k, rope, torch.zeros(5, dtype=torch.long))
    with pytest.raises(ValueError, match="kv_heads"):
        rotary_qkv(torch.zeros(10, 7 * 64, dtype=BF), 2, 5, 4, rope, kv_heads=2)
    with pytest.raises(ValueError, match="kv_heads"):
        rotary_qkv(torch.zeros(11, 8 * 64, dtype=BF), 2, 5, 4, rope, kv_heads=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_qkv(torch.zeros(10, 8 * 64, dtype=BF), 2, 5, 4, rope, kv_heads=2)


def test_rotary_inplace_refuses():
    rope = _rope()
    q = torch.zeros(5, 4, 64, dtype=BF)
    with pytest.raises(ValueError, match="same memory"):
        rotary_(q, q, rope)
    with pytest.raises(RuntimeError, match="single memory location"):
        rotary_(torch.zeros(5, 1, 64, dtype=BF).expand(5, 4, 64), None, rope)
    with pytest.raises(RuntimeError, match="single memory location"):
        buf = torch.zeros(6, 4, 64, dtype=BF)
        rotary_(buf[:5], buf[1:], rope)
    with pytest.raises(RuntimeError, match="gradient"):
        rotary_(q.float().requires_grad_(), None, rope)
    with pytest.raises(ValueError, match="stride 1"):
        rotary_(torch.zeros(5, 4, 128, dtype=BF)[..., ::2], None, rope)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_(q, None, rope)


def _packed_heads(q_from, q_to, k_from, k_to, heads_first=False):
    rope = _rope()
    packed = torch.zeros(2, 8, 5, 64, dtype=BF).transpose(1, 2) if heads_first else torch.zeros(2, 5, 8, 64, dtype=BF)
    rotary_(packed[:, :, q_from:q_to], packed[:, :, k_from:k_to], rope)


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("heads", [(0, 4, 3, 5), (0, 4, 0, 2), (2, 4, 0, 3), (3, 4, 0, 8), (0, 8, 7, 8)])
def test_rotary_inplace_refuses_heads_in_common(heads, heads_first):
    with pytest.raises(ValueError, match="same memory"):
        _packed_heads(*heads, heads_first)


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("heads", [(0, 4, 4, 6), (4, 8, 0, 4), (0, 1, 1, 8), (7, 8, 6, 7)])
def test_rotary_inplace_takes_heads_side_by_side(heads, heads_first):
    with pytest.raises(RuntimeError, match="CUDA"):  # the last check: without a GPU nothing runs
        _packed_heads(*heads, heads_first)


def test_causal_attention_rotary_refuses():
    qkv = torch.zeros(128, 3 * 128, dtype=BF)
    with pytest.raises(ValueError, match="head dim 64"):
        causal_attention(qkv, 1, 128, 1, 128, rotary=_rope())
    with pytest.raises(ValueError, match="without rotary"):
        causal_attention(qkv, 1, 128, 1, 128, positions=torch.arange(128))


def test_residual_norm_refuses():
    x, w = torch.zeros(3, 5, 64, dtype=BF), torch.ones(64)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        residual_norm(x.double(), x.double())
    with pytest.raises(TypeError, match="but the branch"):
        residual_norm(x, x.float())
    with pytest.raises(ValueError, match="same shape"):
        residual_norm(x, x[:, :4])
    with pytest.raises(TypeError, match="must be fp32"):
        residual_norm(x, x, pre_weight=w.to(BF))
    with pytest.raises(ValueError, match=r"must be \[64\]"):
        residual_norm(x, x, post_weight=torch.ones(32))
    with pytest.raises(TypeError, match="per channel must be fp32"):
        residual_norm(x, x, gate=w.to(BF))
    with pytest.raises(TypeError, match="per row must be fp32"):
        residual_norm(x, x, gate=torch.ones(3, 5, 1, dtype=BF))
    with pytest.raises(TypeError, match="per element must have"):
        residual_norm(x, x, gate=torch.ones(3, 5, 64))
    for shape in [(5, 64), (3, 5), (1, 5, 64), (3, 1, 1), (1,)]:
        with pytest.raises(ValueError, match="gate must be"):
            residual_norm(x, x, gate=torch.ones(shape))
    with pytest.raises(ValueError, match="16384"):
        residual_norm(torch.zeros(1, 16385, dtype=BF), torch.zeros(1, 16385, dtype=BF))
    with pytest.raises(ValueError, match="16384"):
        rms_norm(torch.zeros(2, 0), torch.zeros(0))
    for kw in [dict(eps=-1.0), dict(eps=float("nan")), dict(residual_scale=float("inf")),
               dict(branch_scale=float("nan"))]:
        with pytest.raises(ValueError):
            residual_norm(x, x, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        residual_norm(x, x, pre_weight=w, post_weight=w, gate=w)
    with pytest.raises(RuntimeError, match="CUDA"):
        rms_norm(x, w)


def test_token_logprobs_refuses():
    x, t = torch.zeros(3, 5, 40, dtype=BF), torch.zeros(3, 5, dtype=torch.long)
    with pytest.raises(TypeError, match="logits must be"):
        token_logprobs(x.double(), t)
    with pytest.raises(TypeError, match="int64"):
        token_logprobs(x, t.int())
    with pytest.raises(ValueError, match="vocabulary"):
        token_logprobs(x, t[:2])
    with pytest.raises(ValueError, match="vocabulary"):
        token_logprobs(x[..., :0], t)
    for top in (-1, 41, 65):
        with pytest.raises(ValueError, match="top must be"):
            token_logprobs(x, t, top=top)
    for tau in (0.0, -1.0, float("nan"), float("inf"), 1e-7):
        with pytest.raises(ValueError, match="temperature"):
            token_logprobs(x, t, temperature=tau)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x, t, top=4, entropy=True)


def test_forward_mode_gradients_are_refused():
    import torch.autograd.forward_ad as fwd

    rope, w = _rope(), torch.ones(64)
    x = torch.zeros(5, 4, 64)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        calls = [lambda: rotary(dual, None, rope), lambda: rotary(x, dual, rope), lambda: rotary_(dual, None, rope),
                 lambda: rotary_qkv(dual.reshape(5, 256), 1, 5, 2, rope, kv_heads=1),
                 lambda: residual_norm(x, dual, pre_weight=w),
                 lambda: residual_norm(x, x, pre_weight=fwd.make_dual(w, w)),
                 lambda: rms_norm(dual, w),
                 lambda: token_logprobs(dual, torch.zeros(5, 4, dtype=torch.int64))]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
