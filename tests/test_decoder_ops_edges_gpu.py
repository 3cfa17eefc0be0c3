"""More of the decoder operators' edges on the GPU, against the plain 64-bit forms and bounds of
``test_decoder_ops_gpu``: sparse masks in every type, padded batches, rotary undone."""
import pytest
import test_decoder_ops_gpu as ops
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


# ------------------------------------------------------------------------- masked logits before possible ones


def _masked(rows, V, dtype, mask, seed):
    """Logits of which ``mask`` leaves a part, each row's token among them."""
    x, _ = ops._logits(rows, V, dtype, seed)
    g = ops._gen(seed + 1)
    if mask == "leading":
        keep = torch.arange(V, device=DEV).expand(rows, V) >= (V * 2) // 5
    elif mask == "all but the last":
        keep = torch.arange(V, device=DEV).expand(rows, V) >= V - 5
    else:  # one in a thousand, and the last so that none is empty
        keep = torch.rand(rows, V, generator=g, device=DEV) < 1e-3
        keep[:, -1] = True
    t = torch.multinomial(keep.float(), 1, generator=g)[:, 0]
    return x.masked_fill(~keep, float("-inf")), t


@pytest.mark.parametrize("dtype", [HF, BF, F32])
@pytest.mark.parametrize("mask", ["leading", "all but the last", "sparse"])
@pytest.mark.parametrize("rows,V", [(3, 50000), (400, 50001), (5, 3000), (400, 2048), (401, 301)])
def test_logprobs_masked_before_possible(rows, V, mask, dtype):
    """Whole tiles, vectors and threads without a possible token, before or between the possible ones."""
    x, t = _masked(rows, V, dtype, mask, 30)
    # the temperatures put the exponents' range on both sides of fp16's lowest value; the least of them for the
    # smaller cases only
    for tau in (1.0, 0.05) if rows * V > 10 ** 7 else (1.0, 0.05, 1e-4, 30.0, 2000.0):
        r = ops._check_logprobs(x, t, tau=tau, top=4)
        assert torch.isfinite(r.logprob).all() and torch.isfinite(r.entropy).all()
    ops._check_logprobs(x, t, top=4, entropy=False)


@pytest.mark.parametrize("V", [5, 40, 301, 2048, 4099])
def test_logprobs_many_short_rows_fp16(V):
    ops.test_logprobs_many_short_rows(HF, V)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_logprobs_nan_and_inf_stay_in_their_row_fp16(bad):
    ops.test_logprobs_nan_and_inf_stay_in_their_row(bad, HF)


@pytest.mark.parametrize("V", [3000, 70000])
def test_logprobs_rise_over_the_whole_range_fp16(V):
    """Each thread's maximum rises from fp16's lowest value to its largest, with masked values between."""
    i = torch.arange(V, device=DEV).double()
    x = torch.stack([-65504 + 131008 * i / (V - 1), 65504 * i / (V - 1), -65504 + i / V, i * 0 + 65504]).to(HF)
    x[:, 1::3] = float("-inf")
    t = torch.tensor([V - 1 - (V - 1) % 3, 0, 3, 6], device=DEV)
    for tau in (1.0, 1e-3, 1e3):
        for ent in (True, False):
            ops._check_logprobs(x, t, tau=tau, top=4, entropy=ent)


# -------------------------------------------------------------------------------------------- padded batches


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V", [(6, 513), (6, 50257), (400, 1003)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_logprobs_padded_rows_have_no_gradient(bad, rows, V, dtype):
    """Rows behind the last sequence: whatever their logits hold, an ignored token brings no gradient into them, nor do
    zeros from the entropy and the alternatives."""
    from mtorus.ops.logprobs import token_logprobs

    x, t = ops._logits(rows, V, dtype, 40)
    clean = x.clone()
    pad = [1, rows - 1]
    x[pad[0]] = bad
    x[pad[1], V // 2:] = bad
    t[pad] = -100
    up = torch.randn(rows, generator=ops._gen(41), device=DEV)
    up_pad = up.index_fill(0, torch.tensor(pad, device=DEV), 0.0)
    grads = []
    for src in (x, clean):
        leaf = src.detach().requires_grad_()
        r = token_logprobs(leaf, t, top=3, entropy=True)
        assert (r.logprob[pad] == 0).all()
        d = [torch.autograd.grad(r.logprob, leaf, up, retain_graph=True)[0],
             torch.autograd.grad([r.logprob, r.entropy, r.top_logprobs], leaf,
                                 [up, up_pad, up_pad[:, None].expand(rows, 3)], retain_graph=True)[0]]
        if src is x:  # a gradient that does come into such a row is as undefined as its logits
            (own,) = torch.autograd.grad(r.entropy, leaf, up)
            assert torch.isnan(own[pad]).all()
        grads.append(d)
    for got, want in zip(*grads):
        assert (got[pad] == 0).all()
        others = [i for i in range(rows) if i not in pad]
        assert torch.equal(got[others], want[others])


# ------------------------------------------------------------------------------------- rotary there and back


@pytest.mark.parametrize("kw", [dict(), dict(scaling="yarn", factor=8.0), dict(attention_scale=-0.25)])
def test_rotary_inverse_undoes(kw):
    """Positions taken back and given anew, as for a cache that moves: fp32, so that only the arithmetic shows."""
    from mtorus.ops.rotary import rotary_

    rope = ops._rope(64, rot_dim=48, **kw)
    g = ops._gen(50)
    q = torch.randn(5, 3, 64, generator=g, device=DEV)
    k = torch.randn(5, 2, 64, generator=g, device=DEV)
    pos = torch.randint(0, 100000, (5,), generator=g, device=DEV)
    for x, other in ((q, k), (k, None)):
        a, b = x.clone(), None if other is None else other.clone()
        rotary_(a, b, rope, pos)
        rotary_(a, b, rope, pos, inverse=True)
        for got, want in ((a, x), (b, other)):
            if want is None:
                continue
            # each way rounds below 8 U of the pair's sum of absolute values (at most doubled by the way before it), and
            # the scale and its reciprocal are rounded once each
            half = want[..., :48].double().abs().unflatten(-1, (2, 24)).sum(-2).repeat(1, 1, 2)
            off = (got[..., :48].double() - want[..., :48].double()).abs()
            assert (off <= (3 * ops.ROT_ROUNDINGS + 2) * ops.U * half).all()
            assert torch.equal(got[..., 48:], want[..., 48:])


def test_causal_attention_gradient_with_scaled_rotary():
    """The gradient of the turn is the turn back, times the attention scale (not divided by it)."""
    from mtorus.ops.attention import causal_attention
    from mtorus.ops.rotary import rotary_qkv

    B, S, H = 1, 256, 2
    g = ops._gen(51)
    qkv = torch.randn(B * S, 3 * H * 128, generator=g, device=DEV).to(BF)
    dout = torch.randn(B * S, H * 128, generator=g, device=DEV).to(BF)
    rope = ops._rope(128, scaling="yarn", factor=16.0, original_len=64)
    a, b = (qkv.clone().requires_grad_() for _ in range(2))
    oa = causal_attention(a, B, S, H, 128, rotary=rope)
    ob = causal_attention(rotary_qkv(b, B, S, H, rope), B, S, H, 128)
    assert torch.equal(oa, ob)
    (ga,), (gb,) = torch.autograd.grad(oa, a, dout), torch.autograd.grad(ob, b, dout)
    # dQ's reduce-adds may come in another order: bf16 values of one fp32 sum, at most one step apart, then rotated
    assert ((ga.double() - gb.double()).norm() / gb.double().norm()).item() <= 2.0 ** -7
