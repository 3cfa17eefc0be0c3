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


# ------------------------------------------------------------------------------------------- scoring a model


def test_scoring_leaves_the_model_as_it_is_for_others(monkeypatch):
    """While a model scores, its dropout and FP8 states stay set: another thread may be in a training forward."""
    import mtorus.ops.fused as fused
    import mtorus.ops.kernels as kernels
    import mtorus.ops.logprobs as logprobs
    from mtorus.models.gpt import GptConfig, GptModel

    model = GptModel(GptConfig(40, 16, 2, 2, 32, 8, 0.5))
    model.flat = object()
    drop, fp8 = object(), object()
    model.dropout_state, model.fp8_state, model.fp8_head = drop, fp8, True
    model.lm_head.weight.w16 = model.lm_head.weight.data.to(BF)
    seen = []

    def look(*passed):
        assert model.dropout_state is drop and model.fp8_state is fp8
        seen.append(passed)

    class Embed:
        @staticmethod
        def apply(ids, anchor, weights, S, dropout):
            look(dropout)
            return torch.zeros(ids.numel(), 16, dtype=BF)

    class Norm:
        @staticmethod
        def apply(x, weights, eps):
            look(None)
            return x

    monkeypatch.setattr(fused, "EmbeddingFn", Embed)
    monkeypatch.setattr(fused, "LayerNormFn", Norm)
    monkeypatch.setattr(fused, "grad_anchor", lambda device: None)
    monkeypatch.setattr(kernels, "gemm", lambda a, b, bias=None: a @ b.t())
    monkeypatch.setattr(logprobs, "token_logprobs", lambda logits, tokens, **kw: (look(None), logits.shape)[1])
    for blk in model.blocks:
        def forward(x, B, S, fp8=None, drop=None):
            look(fp8, drop)
            return x
        monkeypatch.setattr(blk, "fused_forward", forward)
    ids = torch.zeros(2, 8, dtype=torch.long)
    assert model.fused_token_logprobs(ids, ids) == (2, 8, 40)
    assert len(seen) == 5 and all(v is None for passed in seen for v in passed)
    # and a model that never had FP8 does not get an attribute for it
    del model.fp8_state
    fp8 = None
    monkeypatch.setattr(Embed, "apply", staticmethod(lambda ids, *a: torch.zeros(ids.numel(), 16, dtype=BF)))
    for blk in model.blocks:
        monkeypatch.setattr(blk, "fused_forward", lambda x, B, S, fp8=None, drop=None: x)
    monkeypatch.setattr(Norm, "apply", staticmethod(lambda x, *a: x))
    monkeypatch.setattr(logprobs, "token_logprobs", lambda logits, tokens, **kw: logits.shape)
    model.fused_token_logprobs(ids, ids)
    assert not hasattr(model, "fp8_state")
    # training's own forward still takes both
    model.fp8_state = fp8 = object()
    got = []
    for blk in model.blocks:
        monkeypatch.setattr(blk, "fused_forward", lambda x, B, S, fp8=None, drop=None: (got.append((fp8, drop)), x)[1])
    model.dropout_state = None
    model.fused_hidden(ids)
    assert [f for f, _ in got] == [(fp8, "L0"), (fp8, "L1")]
