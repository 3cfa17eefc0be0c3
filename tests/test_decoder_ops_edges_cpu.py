"""More refusals of the decoder operators, and what their callers pass on (no GPU)."""
import random

import pytest
import torch

from mtorus.ops.rotary import RotaryPositions, rotary, rotary_, rotary_qkv

BF = torch.bfloat16


def _rope(**kw):
    return RotaryPositions(64, device="cpu", **kw)


def test_rotary_inverse_of_a_zero_scale_is_refused():
    q = torch.zeros(5, 4, 64, dtype=BF)
    with pytest.raises(ValueError, match="cannot be undone"):
        rotary_(q, None, _rope(attention_scale=0.0), inverse=True)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_(q, None, _rope(attention_scale=0.0))


def test_rotary_offset_with_positions_is_refused():
    q, pos = torch.zeros(5, 4, 64, dtype=BF), torch.arange(5)
    for call in (lambda **kw: rotary(q, None, _rope(), **kw), lambda **kw: rotary_(q, None, _rope(), **kw),
                 lambda **kw: rotary_qkv(q.view(5, 256), 1, 5, 2, _rope(), kv_heads=1, **kw)):
        with pytest.raises(ValueError, match="offset"):
            call(positions=pos, offset=3)
        for kw in (dict(positions=pos), dict(offset=3)):
            with pytest.raises(RuntimeError, match="CUDA"):
                call(**kw)


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


# --------------------------------------------------------------------------------- heads in common, in place


def _strided(buf, sizes, strides, at=0):
    return buf.as_strided(sizes, strides, at)


def _places(t):
    return set(torch.arange(t.untyped_storage().size() // 2).as_strided(t.size(), t.stride(), t.storage_offset())
               .reshape(-1).tolist())


def _pairs():
    """q and k of one buffer, and whether they have heads in common."""
    buf = torch.zeros(6, 12, 64, dtype=BF)
    four = torch.zeros(2, 5, 12, 64, dtype=BF)
    heads_first = buf.transpose(0, 1)
    flat = torch.zeros(4000, dtype=BF)

    def packed(at):
        return _strided(flat, (4, 2, 64), (768, 64, 1), at)

    return {
        "other head strides": (buf[:, :4], buf[:, 1:8:2], True),
        "other head strides, apart": (buf[:, 0:8:2], buf[:, 1:8:2], False),
        "a group's queries and all keys": (buf[:, 0:2], buf[:, 0:12:3], True),
        "a group's queries and all keys, apart": (buf[:, 0:2], buf[:, 2::4], False),
        "the next token": (buf[:-1, :4], buf[1:, :4], True),
        "the next token, other heads": (buf[:-1, :4], buf[1:, 4:8], False),
        "the next token, some heads": (buf[:-1, 2:6], buf[1:, 5:8], True),
        "the next sequence": (four[:1, :, :3], four[1:, :, :3], False),
        "tokens of the same sequence": (four[:, :3, :3], four[:, 2:, 1:3], True),
        "tokens apart in the same sequence": (four[:, :2, :3], four[:, 3:, 1:3], False),
        "other token strides": (buf[:3, :4], buf[::2, 2:6], True),
        "other token strides, apart": (buf[:3, :4], buf[::2, 4:8], False),
        "half a head": (packed(0), packed(96), True),
        "one value": (packed(0), packed(127), True),
        "side by side": (packed(0), packed(128), False),
        "into the next token": (packed(0), packed(641), True),
        "up to the next token": (packed(0), packed(640), False),
        "heads before tokens": (heads_first[:6, :3], heads_first[2:8, 3:6], False),
        "heads before tokens, shared": (heads_first[:6, :3], heads_first[2:8, 2:5], True),
    }


@pytest.mark.parametrize("name", list(_pairs()))
def test_rotary_inplace_heads_in_common(name):
    q, k, shared = _pairs()[name]
    assert bool(_places(q) & _places(k)) == shared
    for a, b in ((q, k), (k, q)):
        # refused before the last check, which is the one for the device: without a GPU nothing runs
        with pytest.raises((ValueError, RuntimeError), match="memory" if shared else "CUDA"):
            rotary_(a, b, _rope())


def test_rotary_inplace_heads_in_common_at_random():
    """Against the places themselves: layouts of every kind, nested and not."""
    rng = random.Random(7)
    flat = torch.zeros(60000, dtype=BF)
    rope = RotaryPositions(4, device="cpu")
    found = {True: 0, False: 0}
    while min(found.values()) < 150:
        tokens, n = rng.randint(1, 4), [rng.randint(1, 4), rng.randint(1, 4)]
        head = [rng.choice([4, 6, 8, 12, 20]) for _ in range(2)]
        token = [rng.choice([4, 16, 24, 36, 48, 60, 120]) for _ in range(2)]
        q, k = (_strided(flat, (tokens, n[i], 4), (token[i], head[i], 1), rng.randint(0, 150)) for i in range(2))
        # within itself each nests its axes
        if any(t.numel() != len(_places(t)) or
               (t.size(0) > 1 and t.size(1) > 1 and t.stride(0) < t.size(1) * t.stride(1) - t.stride(1) + 4 and
                t.stride(1) < t.size(0) * t.stride(0) - t.stride(0) + 4) for t in (q, k)):
            continue
        shared = bool(_places(q) & _places(k))
        found[shared] += 1
        with pytest.raises((ValueError, RuntimeError)) as e:
            rotary_(q, k, rope)
        assert ("memory" in str(e.value)) == shared, (q.size(), q.stride(), q.storage_offset(), k.stride(),
                                                      k.storage_offset())


def test_rotary_inplace_entangled_layouts_are_refused():
    """Long axes of unlike strides whose heads lie between one another's: no proof in a few thousand trials."""
    flat = torch.zeros(36 * 20000 + 16, dtype=BF)
    q = _strided(flat, (20000, 1, 4), (24, 4, 1))
    k = _strided(flat, (20000, 2, 4), (36, 4, 1), 4)
    with pytest.raises(ValueError, match="same memory"):
        rotary_(q, k, RotaryPositions(4, device="cpu"))


def test_rotary_inplace_windows_that_slide_are_refused():
    flat = torch.zeros(4096, dtype=BF)
    for sizes, strides in [((5, 2, 64), (64, 64, 1)), ((5, 1, 64), (32, 64, 1)), ((2, 5, 2, 64), (192, 128, 64, 1))]:
        with pytest.raises(ValueError, match="same memory"):
            rotary_(_strided(flat, sizes, strides), None, _rope())
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_(_strided(flat, (5, 1, 64), (64, 1, 1)), None, _rope())
