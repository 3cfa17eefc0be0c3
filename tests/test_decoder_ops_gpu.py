"""Rotary positions, residual norm and token log probabilities against plain 64-bit forms.

Every bound is worst-case arithmetic: half a step of the output's type (``finfo.eps / 2`` of the
value) plus a number of fp32 roundings (U = 2^-24 each) of the sum of the absolute values that the
formula adds up, so that cancellation is allowed for and nothing else.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _half_step(t):
    return torch.finfo(t).eps / 2


def _close(got, ref, magnitude, roundings, name="", below=0.0):
    """|got - ref| <= half a step of got's type at ref + roundings * U * magnitude (+ the type's smallest step, and
    ``below``: what underflow takes away)."""
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    g, r = got.detach().double(), ref.detach().double()
    # what lies half a step or more beyond the type's largest value rounds to infinity
    top = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    r = torch.where(r.abs() >= top, torch.copysign(torch.full_like(r, math.inf), r), r)
    fine = torch.isfinite(r)
    assert torch.equal(torch.isnan(g), torch.isnan(r)), name
    assert torch.equal(g[~fine & ~torch.isnan(r)], r[~fine & ~torch.isnan(r)]), name
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    # the rounding to the type acts on the fp32 result: its error is relative to ref + the fp32 error
    err32 = roundings * U * torch.as_tensor(magnitude, device=r.device).double().expand_as(r)
    step = 0.0 if got.dtype == F32 else _half_step(got.dtype)
    bound = err32 + step * (r.abs() + err32) + tiny
    off = ((g - r).abs() - bound)[fine] - below
    assert off.numel() == 0 or off.max().item() <= 0, (name, off.max().item(), (g - r).abs()[fine].max().item())


# ------------------------------------------------------------------------------------------------ rotary
#
# fp32 roundings of one product x cos: fraction of a revolution (<= 2^-26, times 2 pi), sincospi (2 ulp of at most 1),
# scale, product, sum: below 8 U of (|a| + |b|) s.

ROT_ROUNDINGS = 8


def _ref_rotary(x, rope, pos, sign=1.0):
    """x [B, S, H, D] in 64 bits, pos [B, S]."""
    r = rope.rot_dim
    w = torch.tensor(rope.frequencies, dtype=torch.float64, device=DEV)
    ang = pos.double()[:, :, None, None] * w
    c, s = torch.cos(ang) * rope.scale, torch.sin(ang) * rope.scale * sign
    y, mag = x.clone(), torch.zeros_like(x)
    ia, ib = (slice(0, r // 2), slice(r // 2, r)) if rope.layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * rope.scale
    return y, mag


def _rope(dim, **kw):
    from mtorus.ops.rotary import RotaryPositions

    return RotaryPositions(dim, device=DEV, **kw)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32), (80, 20), (96, 24), (256, 64), (33, 10), (2, 2), (512, 512),
                                     (129, 129 - 1)])
def test_rotary_forward_and_gradient(dtype, layout, dim, rot):
    from mtorus.ops.rotary import rotary

    g = _gen(1)
    B, S, H, K = 2, 7, 5, 3
    rope = _rope(dim, rot_dim=rot, layout=layout, scaling="yarn", factor=4.0, original_len=256)
    q = torch.randn(B, S, H, dim, generator=g, device=DEV).to(dtype).requires_grad_()
    k = torch.randn(B, S, K, dim, generator=g, device=DEV).to(dtype).requires_grad_()
    pos = torch.randint(-1000, 200000, (B, S), generator=g, device=DEV)
    oq, ok = rotary(q, k, rope, pos)
    for got, x in ((oq, q), (ok, k)):
        ref, mag = _ref_rotary(x.detach().double(), rope, pos)
        _close(got, ref, mag, ROT_ROUNDINGS)
        assert torch.equal(got[..., rot:], x[..., rot:])
    dq = torch.randn(q.shape, generator=g, device=DEV).to(dtype)
    dk = torch.randn(k.shape, generator=g, device=DEV).to(dtype)
    gq, gk = torch.autograd.grad((oq, ok), (q, k), (dq, dk))
    for got, x in ((gq, dq), (gk, dk)):
        ref, mag = _ref_rotary(x.double(), rope, pos, -1.0)
        _close(got, ref, mag, ROT_ROUNDINGS)


@pytest.mark.parametrize("tokens", [1, 2, 4095, 4096, 4099])
def test_rotary_lengths_and_default_positions(tokens):
    from mtorus.ops.rotary import rotary

    rope = _rope(64)
    q = torch.randn(tokens, 3, 64, generator=_gen(2), device=DEV).to(BF)
    got, none = rotary(q, None, rope, offset=100)
    assert none is None
    ref, mag = _ref_rotary(q.double()[None], rope, 100 + torch.arange(tokens, device=DEV)[None])
    _close(got[None], ref, mag, ROT_ROUNDINGS)


def test_rotary_far_positions():
    """Positions beyond 32 bits keep their angle: 64-bit revolutions, of which the fraction is exact to 2^-20."""
    from mtorus.ops.rotary import rotary

    rope = _rope(64)
    pos = torch.tensor([2 ** 31 - 1, 2 ** 31, 2 ** 33 + 5, -2 ** 32], device=DEV)
    q = torch.randn(4, 2, 64, generator=_gen(3), device=DEV)
    got, _ = rotary(q, None, rope, pos)
    ref, mag = _ref_rotary(q.double()[None], rope, pos[None])
    # both sides round angle / revolutions of up to 2^33 at 2^-53: 2^-18 rad more on each
    _close(got[None], ref, mag, ROT_ROUNDINGS + 2 ** 7)


@pytest.mark.parametrize("shape", ["S", "BS", "1S", "int32", "strided"])
def test_rotary_position_forms(shape):
    from mtorus.ops.rotary import rotary

    g = _gen(4)
    rope = _rope(32)
    q = torch.randn(3, 6, 2, 32, generator=g, device=DEV).to(BF)
    full = torch.randint(0, 5000, (3, 6), generator=g, device=DEV)
    pos = {"S": full[1], "BS": full, "1S": full[1:2], "int32": full.int(),
           "strided": torch.stack([full, full + 1], -1).transpose(0, 1)[..., 0].transpose(0, 1)}[shape]
    got, _ = rotary(q, None, rope, pos)
    ref, mag = _ref_rotary(q.double(), rope, pos.long().expand(3, 6))
    _close(got, ref, mag, ROT_ROUNDINGS)


def test_rotary_one_token_per_sequence_positions():
    from mtorus.ops.rotary import rotary

    rope = _rope(32)
    q = torch.randn(5, 1, 2, 32, generator=_gen(5), device=DEV).to(BF)
    pos = torch.arange(5, device=DEV) * 1000
    got, _ = rotary(q, None, rope, pos)
    ref, mag = _ref_rotary(q.double(), rope, pos[:, None])
    _close(got, ref, mag, ROT_ROUNDINGS)


def test_rotary_strided_and_transposed_inputs():
    from mtorus.ops.rotary import rotary

    g = _gen(6)
    rope = _rope(64)
    base = torch.randn(2, 4, 9, 3 * 64 + 1, generator=g, device=DEV).to(BF)
    views = [base[..., :64].transpose(1, 2), base[..., 1:65].transpose(1, 2), base[..., 0:128:2].transpose(1, 2),
             base[:, :, :1, 64:128].transpose(1, 2).expand(2, 9, 4, 64)]
    pos = torch.arange(9, device=DEV).expand(2, 9)
    for v in views:
        leaf = v.detach().requires_grad_()
        got, _ = rotary(leaf, None, rope)
        ref, mag = _ref_rotary(v.double(), rope, pos)
        _close(got, ref, mag, ROT_ROUNDINGS)
        up = torch.ones(1, 1, 1, 1, dtype=BF, device=DEV).expand_as(got)  # a gradient without strides of its own
        (grad,) = torch.autograd.grad(got, leaf, up)
        ref, mag = _ref_rotary(up.double().contiguous(), rope, pos, -1.0)
        _close(grad, ref, mag, ROT_ROUNDINGS)


@pytest.mark.parametrize("H,K,dim", [(4, 4, 128), (4, 1, 64), (3, 1, 33)])
def test_rotary_packed(H, K, dim):
    from mtorus.ops.rotary import rotary_qkv

    g = _gen(7)
    B, S = 2, 11
    rope = _rope(dim, rot_dim=dim // 4 * 2, layout="interleaved")
    qkv = torch.randn(B * S, (H + 2 * K) * dim, generator=g, device=DEV).to(BF).requires_grad_()
    got = rotary_qkv(qkv, B, S, H, rope, kv_heads=K)
    pos = torch.arange(S, device=DEV).expand(B, S)

    def check(got, x, sign):
        x = x.detach().view(B, S, H + 2 * K, dim)
        got = got.view(B, S, H + 2 * K, dim)
        ref, mag = _ref_rotary(x.double(), rope, pos, sign)
        _close(got[:, :, :H + K], ref[:, :, :H + K], mag[:, :, :H + K], ROT_ROUNDINGS)
        assert torch.equal(got[:, :, H + K:], x[:, :, H + K:])

    check(got, qkv, 1.0)
    up = torch.randn(qkv.shape, generator=g, device=DEV).to(BF)
    (grad,) = torch.autograd.grad(got, qkv, up)
    check(grad, up, -1.0)


def test_rotary_inplace_touches_the_rotated_heads_only():
    from mtorus.ops.rotary import rotary, rotary_

    g = _gen(8)
    rope = _rope(64, rot_dim=32)
    cache = torch.randn(5, 7, 6, 64, generator=g, device=DEV).to(BF)
    before = cache.clone()
    q, k = cache[1:4, :, :3], cache[1:4, :, 4:5]
    want_q, want_k = rotary(q, k, rope, offset=9)
    version = cache._version
    rotary_(q, k, rope, offset=9)
    assert cache._version > version
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    rest = torch.ones_like(cache, dtype=torch.bool)
    rest[1:4, :, :3, :32] = False
    rest[1:4, :, 4:5, :32] = False
    assert torch.equal(cache[rest], before[rest])
    # back again: the fp32 result of two rotations of once-rounded values
    rotary_(q, k, rope, offset=9, inverse=True)
    a = before[1:4].double()
    bound = _half_step(BF) * 2.1 * math.sqrt(2) * a.abs().max()
    assert (cache[1:4].double() - a).abs().max() <= bound


def test_rotary_64bit_offsets():
    """Sequences of a cache further apart than 2^31 values."""
    from mtorus.ops.rotary import rotary_

    rope = _rope(64)
    buf = torch.empty(2 ** 31 + 4096, dtype=BF, device=DEV)
    x = buf.as_strided((2, 3, 2, 64), (2 ** 31 + 64, 128, 64, 1))
    val = torch.randn(2, 3, 2, 64, generator=_gen(9), device=DEV).to(BF)
    x.copy_(val)
    rotary_(x, None, rope, offset=5)
    ref, mag = _ref_rotary(val.double(), rope, 5 + torch.arange(3, device=DEV).expand(2, 3))
    _close(x, ref, mag, ROT_ROUNDINGS)


def test_rotary_empty():
    from mtorus.ops.rotary import rotary, rotary_qkv

    rope = _rope(64)
    q, k = rotary(torch.empty(2, 0, 4, 64, device=DEV), torch.empty(2, 0, 1, 64, device=DEV), rope)
    assert q.shape == (2, 0, 4, 64) and k.shape == (2, 0, 1, 64)
    q, _ = rotary(torch.empty(3, 0, 64, device=DEV), None, rope)
    assert q.shape == (3, 0, 64)
    assert rotary_qkv(torch.empty(0, 12 * 64, device=DEV, dtype=BF), 0, 5, 4, rope).shape == (0, 12 * 64)


def test_rotary_without_query_heads():
    from mtorus.ops.rotary import rotary

    rope = _rope(64, rot_dim=32)
    k = torch.randn(3, 2, 64, generator=_gen(10), device=DEV)
    q, got = rotary(torch.empty(3, 0, 64, device=DEV), k, rope)
    assert q.shape == (3, 0, 64)
    assert torch.equal(got, rotary(k, None, rope)[0]) and torch.equal(got[..., 32:], k[..., 32:])


def test_rotary_inplace_and_inference_mode():
    from mtorus.ops.rotary import rotary, rotary_

    rope = _rope(64)
    with torch.inference_mode():
        q = torch.randn(3, 2, 64, device=DEV)
        want, _ = rotary(q, None, rope)
        rotary_(q, None, rope)
        assert torch.equal(q, want)
    before = q.clone()
    with pytest.raises(RuntimeError, match="inference"):
        rotary_(q, None, rope)
    assert torch.equal(q, before)


def test_rotary_gradient_of_one_side_only():
    from mtorus.ops.rotary import rotary

    rope = _rope(64)
    q = torch.randn(3, 2, 64, device=DEV)
    k = torch.randn(3, 1, 64, device=DEV, requires_grad=True)
    oq, ok = rotary(q, k, rope)
    ok.sum().backward()
    assert q.grad is None and k.grad is not None
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(rotary(q, k, rope)[1].sum(), k, create_graph=True)


# ------------------------------------------------------------------------------------------ residual norm


def _rms(v, w, eps):
    r = 1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
    return v * r * w, r


def _ref_norm(x, h, pre, post, gate, beta, alpha, eps, dy=None, dn=None):
    """Outputs and gradients in 64 bits, each with the sum of absolute values it is made of."""
    T = x.shape[0]
    x, h, pre, post, gate, dy, dn = (None if t is None else t.detach().double()
                                     for t in (x, h, pre, post, gate, dy, dn))
    b, rh = (h, None) if post is None else _rms(h, post, eps)
    ag = alpha if gate is None else alpha * gate
    y = beta * x + ag * b
    ya = (beta * x).abs() + (ag * b).abs()
    out = {"y": (y, ya)}
    if pre is not None:
        n, ry = _rms(y, pre, eps)
        # an error of y moves the norm too: relative to the row's root mean square of absolute values
        rel = 1.0 + ry * ya.square().mean(-1, keepdim=True).sqrt()
        out["n"] = (n, ya * ry * pre.abs() + n.abs() * rel)
    if dy is None and dn is None:
        return out
    Y, Ya = (torch.zeros_like(x), torch.zeros_like(x)) if dy is None else (dy, dy.abs())
    if pre is not None and dn is not None:
        yh, yha = y * ry, ya * ry
        u = dn * pre
        m, ma = (u * yh).mean(-1, keepdim=True), (u.abs() * yha).mean(-1, keepdim=True)
        Y = Y + ry * (u - yh * m)
        Ya = Ya + ry * rel * (u.abs() + yha * ma * rel)
        out["dpre"] = ((dn * yh).sum(0), (dn.abs() * yha * rel).sum(0))
    out["dx"] = (beta * Y, abs(beta) * Ya)
    db, dba = ag * Y, (ag * torch.ones_like(Y)).abs() * Ya
    if gate is not None:
        dg, dga = alpha * b * Y, abs(alpha) * b.abs() * Ya
        if gate.shape == (x.shape[1],) and not (T == 1 and x.shape[1] == 1):
            out["dgate"] = (dg.sum(0), dga.sum(0))
        elif gate.shape == (T, 1):
            out["dgate"] = (dg.sum(1, keepdim=True), dga.sum(1, keepdim=True))
        else:
            out["dgate"] = (dg, dga)
    if post is not None:
        hh = h * rh
        out["dpost"] = ((db * hh).sum(0), (dba * hh.abs()).sum(0))
        v, va = db * post, dba * post.abs()
        mean, meana = (v * hh).mean(-1, keepdim=True), (va * hh.abs()).mean(-1, keepdim=True)
        out["dh"] = (rh * (v - hh * mean), rh * (va + hh.abs() * meana))
    else:
        out["dh"] = (db, dba)
    return out


# fp32 roundings: a row sum adds 8-16 values of a thread, 5 shuffles and up to 32 warps (below 64); each factor of
# a chain (statistics, weights, gate, scales) a few more, and the gradients chain two row sums.
FWD_ROUNDINGS, BWD_ROUNDINGS = 96, 320
# column sums: rows of a CTA, then up to 2368 / 8 partial sums of a warp, then 8 warps
COL_ROUNDINGS = BWD_ROUNDINGS + 512


def _norm_case(rows, d, dtype, post, pre, gate, seed=0):
    g = _gen(seed)

    def rand(*s):
        return torch.randn(*s, generator=g, device=DEV)

    t = dict(x=(rand(rows, d) * 2).to(dtype), h=rand(rows, d).to(dtype), pre=1 + 0.2 * rand(d) if pre else None,
             post=1 + 0.2 * rand(d) if post else None,
             gate={"none": None, "channel": rand(d), "row": rand(rows, 1), "full": rand(rows, d).to(dtype)}[gate])
    return t, rand(rows, d).to(dtype), rand(rows, d).to(dtype) if pre else None


def _check_norm(t, dy, dn, beta=0.75, alpha=-0.5, eps=1e-6):
    from mtorus.ops.residual_norm import residual_norm

    leaf = {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}
    y, n = residual_norm(leaf["x"], leaf["h"], pre_weight=leaf["pre"], post_weight=leaf["post"], gate=leaf["gate"],
                         residual_scale=beta, branch_scale=alpha, eps=eps)
    ref = _ref_norm(t["x"], t["h"], t["pre"], t["post"], t["gate"], beta, alpha, eps, dy, dn)
    _close(y, *ref["y"], FWD_ROUNDINGS, "y")
    assert (n is None) == (t["pre"] is None)
    if n is not None:
        _close(n, *ref["n"], FWD_ROUNDINGS, "n")
    outs = [(y, dy)] + ([] if n is None else [(n, dn)])
    outs = [(o, g) for o, g in outs if g is not None]
    names = [k for k, v in leaf.items() if v is not None]
    got = torch.autograd.grad([o for o, _ in outs], [leaf[k] for k in names], [g for _, g in outs], allow_unused=True)
    for k, v in zip(names, got):
        if "d" + k not in ref:
            assert v is None, k
            continue
        assert v.dtype == leaf[k].dtype
        column = k in ("pre", "post") or (k == "gate" and v.dim() == 1)
        _close(v, *ref["d" + k], COL_ROUNDINGS if column else BWD_ROUNDINGS, "d" + k)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 64), (2, 255), (9, 256), (3, 1000), (4, 1003), (700, 136),
                                    (17, 2048), (3, 4096), (2, 8192), (2, 8200), (3, 16384), (2, 16383)])
def test_residual_norm_sizes(dtype, rows, d):
    t, dy, dn = _norm_case(rows, d, dtype, True, True, "channel" if d > 1 else "none")
    _check_norm(t, dy, dn)


@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("d", [256, 1003])
def test_residual_norm_parts(post, pre, gate, d):
    t, dy, dn = _norm_case(33, d, BF, post, pre, gate, 1)
    _check_norm(t, dy, dn)


@pytest.mark.parametrize("gate", ["channel", "row", "full"])
@pytest.mark.parametrize("dtype,d", [(BF, 2048), (F32, 1003), (BF, 16384)])
def test_residual_norm_gates(gate, dtype, d):
    t, dy, dn = _norm_case(21, d, dtype, True, True, gate, 2)
    _check_norm(t, dy, dn, beta=1.0, alpha=1.0)


@pytest.mark.parametrize("which", ["y", "n"])
def test_residual_norm_one_gradient_only(which):
    t, dy, dn = _norm_case(19, 512, BF, True, True, "channel", 3)
    _check_norm(t, dy if which == "y" else None, dn if which == "n" else None)


@pytest.mark.parametrize("wanted", [("pre",), ("x",), ("h", "gate"), ("post", "gate"), ("x", "pre")])
def test_residual_norm_some_gradients(wanted):
    from mtorus.ops.residual_norm import residual_norm

    t, dy, dn = _norm_case(50, 256, BF, True, True, "channel", 16)
    ref = _ref_norm(t["x"], t["h"], t["pre"], t["post"], t["gate"], 1.0, 1.0, 1e-6, dy, dn)
    leaf = {k: v.detach().requires_grad_(k in wanted) for k, v in t.items()}
    y, n = residual_norm(leaf["x"], leaf["h"], pre_weight=leaf["pre"], post_weight=leaf["post"], gate=leaf["gate"])
    got = torch.autograd.grad([y, n], [leaf[k] for k in wanted], [dy, dn], allow_unused=True)
    for k, v in zip(wanted, got):
        _close(v, *ref["d" + k], BWD_ROUNDINGS if k in "xh" else COL_ROUNDINGS, k)


def test_residual_norm_many_rows():
    t, dy, dn = _norm_case(5003, 264, BF, True, True, "channel", 4)
    _check_norm(t, dy, dn)
    t, dy, dn = _norm_case(4096, 1032, BF, True, True, "channel", 4)
    _check_norm(t, dy, dn)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,d", [(7, 77), (9, 77), (2011, 77), (601, 1003), (333, 2047), (5, 8191), (1200, 4097),
                                    (2, 9), (300, 9), (37, 260)])
@pytest.mark.parametrize("gate", ["channel", "full"])
def test_residual_norm_rows_off_16_bytes(dtype, rows, d, gate):
    t, dy, dn = _norm_case(rows, d, dtype, True, True, gate, 14)
    _check_norm(t, dy, dn)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows,d", [(1, 8), (2, 40), (3, 64), (5, 48), (6, 128), (1, 128), (4097, 64), (2049, 72),
                                    (20001, 64), (10001, 120)])
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
def test_residual_norm_short_rows(dtype, rows, d, gate):
    t, dy, dn = _norm_case(rows, d, dtype, True, True, gate, 21)
    _check_norm(t, dy, dn)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [3, 9, 601])
def test_rms_norm_of_heads(rows, d):
    """[tokens, heads, d] views of a packed matrix, which stays as it was."""
    from mtorus.ops.residual_norm import rms_norm

    g = _gen(22)
    packed = torch.randn(rows, 5 * d, generator=g, device=DEV).to(BF)
    kept = packed.clone()
    w = torch.randn(d, generator=g, device=DEV)
    for part in (packed[:, :d], packed[:, d:4 * d].unflatten(1, (3, d)), packed.unflatten(1, (5, d))):
        x = part.detach().requires_grad_()
        n = rms_norm(x, w.requires_grad_(), eps=1e-6)
        dn = torch.randn(n.shape, generator=g, device=DEV).to(BF)
        dx, dw = torch.autograd.grad(n, [x, w], dn)
        flat = x.detach().reshape(-1, d)
        ref = _ref_norm(flat, torch.zeros_like(flat), w, None, None, 1.0, 0.0, 1e-6, None, dn.reshape(-1, d))
        _close(n.reshape(-1, d), *ref["n"], FWD_ROUNDINGS, "n")
        _close(dx.reshape(-1, d), *ref["dx"], BWD_ROUNDINGS, "dx")
        _close(dw, *ref["dpre"], COL_ROUNDINGS, "dw")
    assert torch.equal(packed, kept)


@pytest.mark.parametrize("d", [64, 120])
def test_residual_norm_short_rows_do_not_mix(d):
    """A row of NaN or infinity changes its own results only (and the column sums), whichever rows share its warp."""
    from mtorus.ops.residual_norm import residual_norm

    t, dy, dn = _norm_case(13, d, BF, True, True, "row", 23)

    def run(t):
        leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, n = residual_norm(leaf["x"], leaf["h"], pre_weight=leaf["pre"], post_weight=leaf["post"], gate=leaf["gate"])
        return [y, n, *torch.autograd.grad([y, n], [leaf["x"], leaf["h"], leaf["gate"]], [dy, dn])]

    want = run(t)
    for row, value in ((0, math.nan), (5, math.inf), (12, math.nan)):
        x = t["x"].clone()
        x[row] = value
        others = [i for i in range(13) if i != row]
        for a, b in zip(run(dict(t, x=x)), want):
            assert torch.equal(a[others], b[others])
            assert not torch.isfinite(a[row].float()).all()


def test_residual_norm_rows_off_16_bytes_of_a_wider_matrix():
    """Rows of 257 values, 769 apart: what lies between them is neither used nor, in the outputs, written."""
    g = _gen(15)
    wide = torch.full((40, 769), float("nan"), device=DEV, dtype=BF)
    t, dy, dn = _norm_case(40, 257, BF, True, True, "channel", 15)
    for at in (0, 512):
        x = wide.clone()
        x[:, at:at + 257] = torch.randn(40, 257, generator=g, device=DEV).to(BF)
        _check_norm(dict(t, x=x[:, at:at + 257]), dy, dn)
        _check_norm(dict(t, h=x[:, at:at + 257]), dy, dn)
        _check_norm(t, x[:, at:at + 257], dn)


def test_residual_norm_zero_gate_and_zero_rows():
    t, dy, dn = _norm_case(6, 320, F32, True, True, "row", 5)
    t["gate"][1] = 0.0
    t["h"][2] = 0.0
    t["x"][3] = 0.0
    t["h"][3] = 0.0
    _check_norm(t, dy, dn)


def test_residual_norm_strides():
    """Rows of a wider matrix, on and off 16-byte boundaries, transposed and expanded inputs."""
    g = _gen(6)
    wide = torch.randn(12, 3 * 256 + 1, generator=g, device=DEV).to(BF)
    base, dy, dn = _norm_case(12, 256, BF, True, True, "full", 7)
    for x in (wide[:, :256], wide[:, 1:257], wide[:, 0:512:2], wide[:256, :12].t().contiguous().t()[:12].expand(12, 12)
              [:, :1].expand(12, 256)):
        _check_norm(dict(base, x=x), dy, dn)
        _check_norm(dict(base, h=x, gate=wide[:, 512:768]), dy, dn)
        _check_norm(base, x, dn)
        _check_norm(base, dy, x)


def test_residual_norm_leading_dims():
    from mtorus.ops.residual_norm import residual_norm

    t, _, _ = _norm_case(12, 128, BF, True, True, "row", 8)
    x, h = t["x"].view(3, 4, 128), t["h"].view(3, 4, 128)
    y, n = residual_norm(x, h, pre_weight=t["pre"], post_weight=t["post"], gate=t["gate"].view(3, 4, 1))
    y2, n2 = residual_norm(t["x"], t["h"], pre_weight=t["pre"], post_weight=t["post"], gate=t["gate"])
    assert y.shape == x.shape and torch.equal(y.view(12, 128), y2) and torch.equal(n.view(12, 128), n2)
    # x as [B, S, d] with the sequence dimension first in memory
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    y3, _ = residual_norm(xt, h, pre_weight=t["pre"], post_weight=t["post"], gate=t["gate"].view(3, 4, 1))
    assert torch.equal(y3, y)


@pytest.mark.parametrize("rows,d,dtype", [(5, 2048, BF), (3, 77, F32), (0, 64, BF)])
def test_rms_norm(rows, d, dtype):
    from mtorus.ops.residual_norm import rms_norm

    t, _, dn = _norm_case(rows, d, dtype, False, True, "none", 9)
    x, w = t["x"].requires_grad_(), t["pre"].requires_grad_()
    n = rms_norm(x, w)
    ref = _ref_norm(x, torch.zeros_like(x), w, None, None, 1.0, 0.0, 1e-6, None, dn)
    _close(n, *ref["n"], FWD_ROUNDINGS)
    dx, dw = torch.autograd.grad(n, (x, w), dn)
    _close(dx, *ref["dx"], BWD_ROUNDINGS)
    _close(dw, *ref["dpre"], COL_ROUNDINGS)


def test_residual_norm_empty():
    t, dy, dn = _norm_case(0, 64, BF, True, True, "channel", 10)
    _check_norm(t, dy, dn)


def test_residual_norm_repeats_bit_for_bit():
    from mtorus.ops.residual_norm import residual_norm

    t, dy, dn = _norm_case(3001, 512, BF, True, True, "channel", 11)
    runs = []
    for _ in range(3):
        leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, n = residual_norm(leaf["x"], leaf["h"], pre_weight=leaf["pre"], post_weight=leaf["post"],
                             gate=leaf["gate"])
        runs.append([y, n] + list(torch.autograd.grad([y, n], list(leaf.values()), [dy, dn])))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_residual_norm_differences():
    """The gradient against central differences of the 64-bit function along random directions: the difference
    is off by O(h^2) of the function's third derivative (h = 1e-4) and the fp32 gradient by its roundings."""
    from mtorus.ops.residual_norm import residual_norm

    t, dy, dn = _norm_case(7, 96, F32, True, True, "channel", 12)
    leaf = {k: v.detach().requires_grad_() for k, v in t.items()}
    y, n = residual_norm(leaf["x"], leaf["h"], pre_weight=leaf["pre"], post_weight=leaf["post"], gate=leaf["gate"],
                         eps=1e-3)
    grads = torch.autograd.grad([y, n], list(leaf.values()), [dy, dn])

    def f(v):
        o = _ref_norm(v["x"], v["h"], v["pre"], v["post"], v["gate"], 1.0, 1.0, 1e-3)
        return ((o["y"][0] * dy.double()).sum() + (o["n"][0] * dn.double()).sum()).item()

    for (k, v), g in zip(t.items(), grads):
        e = torch.randn(v.shape, generator=_gen(13), device=DEV).double()
        e /= e.norm()
        up, down = (f({**t, k: v.double() + s * 1e-4 * e}) for s in (1, -1))
        assert abs((up - down) / 2e-4 - (g.double() * e).sum().item()) <= 1e-4 * max(1.0, g.double().norm().item()), k


# -------------------------------------------------------------------------------------- log probabilities


def _ref_logprobs(logits, tokens, tau, top, gl=None, gh=None, gk=None):
    x = logits.detach().double()
    V = x.shape[-1]
    z = x / tau
    m = z.amax(-1, keepdim=True)
    empty = m == float("-inf")
    zm = torch.where(empty, torch.full_like(z, float("-inf")), z - m.masked_fill(empty, 0.0))
    s = zm.exp().sum(-1, keepdim=True)
    lp = zm - s.log().masked_fill(empty, 0.0)
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, 0.0) if not torch.isnan(p).any() else p * lp
    ent = -plp.sum(-1)
    use = (tokens >= 0) & (tokens < V)
    at = torch.where(use, tokens, 0).unsqueeze(-1)
    out = {"logprob": torch.where(use, lp.gather(-1, at).squeeze(-1), 0.0), "entropy": ent, "lp": lp}
    if top:
        # descending by value, equal values by index: a stable sort; NaN ranks with -inf
        order = torch.sort(torch.where(torch.isnan(x), float("-inf"), x), dim=-1, descending=True, stable=True)
        out["top_ids"] = order.indices[..., :top]
        out["top_logprobs"] = lp.gather(-1, out["top_ids"])
    if gl is None and gh is None and gk is None:
        return out
    d, mag = torch.zeros_like(x), torch.zeros_like(x)
    total = torch.zeros_like(ent)
    factor = torch.zeros_like(x)  # what a probability is multiplied with, in absolute values
    if gl is not None:
        g = torch.where(use, gl.double(), 0.0)
        total = total + g
        d.scatter_add_(-1, at, g.unsqueeze(-1))
        mag.scatter_add_(-1, at, g.abs().unsqueeze(-1))
    if gk is not None:
        total = total + gk.double().sum(-1)
        d.scatter_add_(-1, out["top_ids"], gk.double())
        mag.scatter_add_(-1, out["top_ids"], gk.double().abs())
    ta = total.abs() + (0 if gk is None else gk.double().abs().sum(-1))
    d = d - p * total.unsqueeze(-1)
    mag = mag + p * ta.unsqueeze(-1)
    factor = factor + ta.unsqueeze(-1)
    if gh is not None:
        d = d - gh.double().unsqueeze(-1) * (plp + p * ent.unsqueeze(-1))
        mag = mag + gh.double().abs().unsqueeze(-1) * (plp.abs() + p * ent.unsqueeze(-1).abs())
        factor = factor + gh.double().abs().unsqueeze(-1) * (lp.abs().clamp(max=140.0) + ent.unsqueeze(-1).abs())
    # a probability below 2^-126 (and its logarithm below -140) counts as 0: at most 2^-126 times its factor is lost
    out["dlogits"] = (torch.where(empty, 0.0, d / tau), mag / tau, factor / tau * 2.0 ** -126)
    return out


def _lp_roundings(V):
    # a thread adds up to V / 512 exponentials, rescaled on the way, then 5 + 5 joins; an exponential is off by
    # |t| + 4 roundings, log2 and the products by a few more
    return V / 512 + 160


def _check_logprobs(logits, tokens, tau=1.0, top=0, entropy=True, grads="lhk", seed=0, dlogits_layout=None):
    from mtorus.ops.logprobs import token_logprobs

    V = logits.shape[-1]
    leaf = logits.detach().requires_grad_()
    r = token_logprobs(leaf, tokens, temperature=tau, top=top, entropy=entropy)
    g = _gen(seed + 100)
    gl = torch.randn(tokens.shape, generator=g, device=DEV) if "l" in grads else None
    gh = torch.randn(tokens.shape, generator=g, device=DEV) if "h" in grads and entropy else None
    gk = torch.randn(*tokens.shape, top, generator=g, device=DEV) if "k" in grads and top else None
    ref = _ref_logprobs(logits, tokens, tau, top, gl, gh, gk)
    n = _lp_roundings(V)
    lp_mag = 1.0 + ref["logprob"].abs().masked_fill(torch.isinf(ref["logprob"]), 0.0)
    _close(r.logprob, ref["logprob"], lp_mag.nan_to_num(), n, "logprob")
    if entropy:
        _close(r.entropy, ref["entropy"], (1.0 + math.log(V) + ref["entropy"].abs()).nan_to_num(), n, "entropy")
    else:
        assert r.entropy is None
    if top:
        assert torch.equal(r.top_ids, ref["top_ids"])
        mag = 1.0 + ref["top_logprobs"].abs().masked_fill(torch.isinf(ref["top_logprobs"]), 0.0)
        _close(r.top_logprobs, ref["top_logprobs"], mag.nan_to_num(), n, "top")
    else:
        assert r.top_ids is None and r.top_logprobs is None
    pairs = [(o, u) for o, u in ((r.logprob, gl), (r.entropy, gh), (r.top_logprobs, gk)) if u is not None]
    if pairs:
        (d,) = torch.autograd.grad([o for o, _ in pairs], leaf, [u for _, u in pairs])
        assert d.dtype == logits.dtype
        # a probability is off by the error of its log (n roundings) plus that of its own exponent (2 |log p|, and
        # p |log p| < 1 keeps that within n of the largest term)
        _close(d, ref["dlogits"][0], ref["dlogits"][1].nan_to_num(), 2 * n, "dlogits",
               ref["dlogits"][2].nan_to_num()[torch.isfinite(ref["dlogits"][0])])
    return r


def _logits(rows, V, dtype, seed=0, scale=3.0):
    g = _gen(seed)
    x = (torch.randn(rows, V, generator=g, device=DEV) * scale).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g, device=DEV)
    return x, t


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 5), (4, 17), (5, 64), (3, 1000), (2, 1003), (7, 4099),
                                    (300, 520), (3, 50257), (1, 50304), (2, 131072)])
def test_logprobs_sizes(dtype, rows, V):
    x, t = _logits(rows, V, dtype)
    _check_logprobs(x, t, top=min(5, V))
    _check_logprobs(x, t, tau=0.7, top=0, entropy=False)


@pytest.mark.parametrize("top", [1, 2, 20, 63, 64])
@pytest.mark.parametrize("rows,V", [(2, 64), (3, 700), (2, 30011), (400, 2048)])
def test_logprobs_top(top, rows, V):
    x, t = _logits(rows, V, BF, 1, 1.0)  # many equal values at 8 bits
    _check_logprobs(x, t, top=top, tau=1.5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [5, 40, 256, 301, 1003, 2048, 4099])
def test_logprobs_many_short_rows(dtype, V):
    """Enough rows for a warp each: every bound on the alternatives, ties, masks, rows off 16-byte offsets."""
    x, t = _logits(401, V, dtype, 12, 1.0)
    x[5] = float("-inf")
    x[6] = 1.0
    x[7, 3:] = float("-inf")
    x[8, ::2] = torch.finfo(dtype).min
    x[9] = torch.finfo(dtype).min
    t[10] = -1
    for top in sorted({0, 1, min(7, V), min(20, V), min(64, V)}):
        _check_logprobs(x, t, top=top, tau=0.8, entropy=top != 7)


def test_logprobs_ties_and_order():
    """Rows of one value, of two values, falling, rising, and with all large values in one thread's vectors."""
    V = 40000
    i = torch.arange(V, device=DEV)
    rows = [torch.zeros(V, device=DEV), (i % 2).float(), -i.float() / 64, i.float() / 64,
            torch.where(i % 4096 < 8, 5.0 + (i % 7).float(), -3.0), torch.where(i % 32768 < 8, 50.0, 0.0),
            torch.where(i == 39999, 9.0, -9.0), torch.where(i % 2 == 0, 0.0, -0.0)]
    x = torch.stack(rows)
    t = torch.arange(len(rows), device=DEV) * 100
    for dtype in (BF, F32):
        for top in (1, 17, 64):
            _check_logprobs(x.to(dtype), t, top=top)


def test_logprobs_more_candidates_than_room():
    """All large values in the vectors of a few threads, so that thousands lie above the bound."""
    V, step = 262144, 512 * 8
    x = torch.full((300, V), -1.0, device=DEV)
    at = torch.arange(V, device=DEV) % step < 80
    x[::2, at] = (torch.arange(int(at.sum()), device=DEV) % 251).float()
    t = torch.zeros(300, dtype=torch.long, device=DEV)
    _check_logprobs(x.to(BF), t, top=64, grads="")


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_logprobs_masks(dtype):
    """Masked columns, masked targets, a row with three possible tokens, an empty row and rows of lowest values."""
    V = 3001
    low = torch.finfo(dtype).min
    x, t = _logits(8, V, dtype, 2)
    x[0, 2000:] = float("-inf")
    t[0] = 5
    x[1, 10] = float("-inf")
    t[1] = 10
    x[2] = float("-inf")
    x[2, [7, 2999, 100]] = torch.tensor([1.0, 2.0, 3.0], device=DEV).to(dtype)
    t[2] = 100
    x[3] = float("-inf")
    t[3] = 4
    x[4] = low
    x[5] = low
    x[5, 77] = 0.5
    t[5] = 77
    x[6, ::2] = low
    x[7] = low
    x[7, 5:9] = float("-inf")
    x[7, 0] = float("-inf")
    r = _check_logprobs(x, t, top=6)
    assert r.logprob[1] == float("-inf") and r.logprob[3] == float("-inf") and r.entropy[3] == 0
    assert r.top_ids[2].tolist() == [100, 2999, 7, 0, 1, 2] and r.top_ids[3].tolist() == list(range(6))
    assert abs(r.entropy[4].item() - math.log(V)) < 1e-4


def test_logprobs_ignored_tokens():
    x, t = _logits(6, 513, F32, 3)
    t[0], t[1], t[2] = -100, 513, 2 ** 40
    r = _check_logprobs(x, t, top=3)
    assert (r.logprob[:3] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_nan_and_inf_stay_in_their_row(bad, dtype):
    from mtorus.ops.logprobs import token_logprobs

    x, t = _logits(4, 5000, dtype, 4)
    x[1, 4321] = bad
    x[2] = bad
    leaf = x.requires_grad_()
    r = token_logprobs(leaf, t, top=4, entropy=True)
    (d,) = torch.autograd.grad(r.logprob.sum() + r.entropy.sum() + r.top_logprobs.sum(), leaf)
    for row in (1, 2):
        for o in (r.logprob, r.entropy, r.top_logprobs, d):
            assert torch.isnan(o[row]).all()
        assert ((r.top_ids[row] >= 0) & (r.top_ids[row] < 5000)).all()
    if bad == float("inf"):
        assert r.top_ids[1, 0] == 4321
    assert r.top_ids[2].tolist() == [0, 1, 2, 3]
    keep = [0, 3]
    _check_logprobs(x.detach()[keep], t[keep], top=4)
    clean = token_logprobs(x.detach()[keep], t[keep], top=4, entropy=True)
    for a, b in zip(r, clean):
        assert torch.equal(a[keep], b)


def test_logprobs_peaked_and_extreme():
    """One certain token; values near the end of the range; small and large temperatures."""
    V = 1999
    x = torch.full((5, V), -40.0, device=DEV)
    x[0, 3] = 60.0
    x[1] = torch.linspace(-3e38, 3e38, V, device=DEV)
    x[2] = 1e30
    x[3] = torch.linspace(0, 1, V, device=DEV)
    x[4, :2] = 3.0
    t = torch.tensor([3, V - 1, 0, 5, 1], device=DEV)
    for tau in (1.0, 1e-3, 1e3):
        keep = [0, 1, 2, 3, 4] if tau == 1.0 else [0, 3, 4]
        _check_logprobs(x[keep], t[keep], tau=tau, top=3)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [3000, 70000])
def test_logprobs_large_values_that_keep_rising(dtype, V):
    """Each thread's maximum rises again and again far beyond where exponents are exact: still finite results."""
    i = torch.arange(V, device=DEV).double()
    x = torch.stack([1e30 * (1 + i), 1e32 * (1 + i / V), -1e30 * (V - i), 1e9 + 1e7 * i, i * 0 + 3e38]).to(dtype)
    for rows in (slice(0, 5), slice(0, 1)):
        xr = x[rows]
        t = torch.randint(0, V, (xr.shape[0],), generator=_gen(13), device=DEV)
        t[0] = V - 1
        for ent in (True, False):
            r = _check_logprobs(xr, t, top=4, entropy=ent)
            assert torch.isfinite(r.logprob).all()


@pytest.mark.parametrize("grads", ["l", "h", "k", "lk", "hk"])
def test_logprobs_parts_of_the_gradient(grads):
    x, t = _logits(9, 2051, BF, 5)
    # the token is also an alternative in some rows: its gradient is the sum of both
    t[::2] = x[::2].float().argmax(-1)
    _check_logprobs(x, t, top=4, grads=grads)


def test_logprobs_strides():
    """Columns of a wider matrix, rows off the gradient's 16-byte offsets, leading dimensions, expanded rows."""
    wide, t = _logits(6, 4000, BF, 6)
    for x in (wide[:, :1000], wide[:, 1:1004], wide[:, 3:1019], wide[:, 0:2000:2], wide[:1, 5:1005].expand(6, 1000)):
        _check_logprobs(x, t % 1000, top=3)
    _check_logprobs(wide[:, :1000].reshape(2, 3, 1000), (t % 1000).view(2, 3), top=3)
    _check_logprobs(wide[0], t[0], top=3)  # one row, no leading dimension


def test_logprobs_64bit_offsets():
    V = 4096
    buf = torch.empty(2 ** 31 + 3 * V, dtype=BF, device=DEV)
    x = buf.as_strided((2, V), (2 ** 31 + V, 1))
    val, t = _logits(2, V, BF, 7)
    x.copy_(val)
    _check_logprobs(x, t, top=4, grads="")


def test_logprobs_empty():
    from mtorus.ops.logprobs import token_logprobs

    x = torch.empty(0, 100, device=DEV, dtype=BF, requires_grad=True)
    r = token_logprobs(x, torch.empty(0, dtype=torch.long, device=DEV), top=3, entropy=True)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    r.logprob.sum().backward()
    assert x.grad.shape == (0, 100)


def test_logprobs_agrees_with_the_cross_entropy_kernel():
    from mtorus.ops import kernels as K
    from mtorus.ops.logprobs import token_logprobs

    x, t = _logits(64, 50304, BF, 8)
    lp = token_logprobs(x, t).logprob
    loss = K.xent_fused(x.clone(), t, write_grad=False)
    # that kernel evaluates half of its exponentials to 7.5e-5
    assert (lp + loss).abs().max() <= 1e-4 + 1e-6 * loss.abs().max()


def test_logprobs_repeats_bit_for_bit():
    from mtorus.ops.logprobs import token_logprobs

    for rows in (3, 500):
        x, t = _logits(rows, 20000, BF, 9, 1.0)
        runs = []
        for _ in range(3):
            leaf = x.detach().requires_grad_()
            r = token_logprobs(leaf, t, top=20, entropy=True)
            (d,) = torch.autograd.grad(r.logprob.sum() + r.top_logprobs.sum() - r.entropy.sum(), leaf)
            runs.append([*r, d])
        for o in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(o, runs[0]))


def test_logprobs_differences():
    """Against central differences of the 64-bit function (h = 1e-4: off by O(h^2) of its third derivative)."""
    from mtorus.ops.logprobs import token_logprobs

    x, t = _logits(4, 50, F32, 10, 1.0)
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, t, top=3, entropy=True, temperature=0.9)
    (d,) = torch.autograd.grad(r.logprob.sum() + 2 * r.entropy.sum() - r.top_logprobs.sum(), leaf)
    e = torch.randn(x.shape, generator=_gen(11), device=DEV).double()
    e /= e.norm()

    def f(v):
        o = _ref_logprobs(v, t, 0.9, 3)
        return (o["logprob"].sum() + 2 * o["entropy"].sum() - o["top_logprobs"].sum()).item()

    diff = (f(x.double() + 1e-4 * e) - f(x.double() - 1e-4 * e)) / 2e-4
    assert abs(diff - (d.double() * e).sum().item()) <= 1e-4


def test_double_backward_is_refused():
    from mtorus.ops.logprobs import token_logprobs
    from mtorus.ops.residual_norm import residual_norm

    x = torch.randn(3, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(token_logprobs(x, torch.zeros(3, dtype=torch.long, device=DEV)).logprob.sum(), x,
                            create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(residual_norm(x, x)[0].sum(), x, create_graph=True)


def test_changed_inputs_are_noticed():
    from mtorus.ops.logprobs import token_logprobs
    from mtorus.ops.residual_norm import residual_norm

    x = torch.randn(3, 64, device=DEV, requires_grad=True)
    for f in (lambda y: token_logprobs(y, torch.zeros(3, dtype=torch.long, device=DEV)).logprob,
              lambda y: residual_norm(y, y, post_weight=torch.ones(64, device=DEV))[0]):
        y = x * 1.0
        o = f(y)
        y.add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            o.sum().backward()


# ------------------------------------------------------------------------------------- streams and graphs


def _step(t, rope, dy):
    """All three operators, forward and backward, on tensors of the caller."""
    from mtorus.ops.logprobs import token_logprobs
    from mtorus.ops.residual_norm import residual_norm
    from mtorus.ops.rotary import rotary

    leaf = {k: v.detach().requires_grad_() for k, v in t.items() if k != "tokens"}
    y, n = residual_norm(leaf["x"], leaf["h"], pre_weight=leaf["pre"], post_weight=leaf["post"], gate=leaf["gate"])
    q, _ = rotary(n.view(-1, 4, 64), None, rope)
    r = token_logprobs(q.reshape(-1, 256), t["tokens"], top=3, entropy=True)
    grads = torch.autograd.grad([y, r.logprob, r.entropy, r.top_logprobs], list(leaf.values()),
                                [dy, dy[:, 0].float(), dy[:, 1].float(), dy[:, :3].float()])
    return [y.detach(), n.detach(), r.logprob.detach(), r.entropy.detach(), r.top_ids, *grads]


def _step_inputs(seed):
    t, dy, _ = _norm_case(300, 256, BF, True, True, "channel", seed)
    t["tokens"] = torch.randint(0, 256, (300,), generator=_gen(seed + 1), device=DEV)
    return t, dy


def test_two_streams_at_once():
    rope = _rope(64)
    work = [_step_inputs(20), _step_inputs(30)]
    want = [_step(t, rope, dy) for t, dy in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(4):
        for i, (s, (t, dy)) in enumerate(zip(streams, work)):
            with torch.cuda.stream(s):
                got[i].append(_step(t, rope, dy))
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_two_captured_graphs():
    """Forward and backward recorded twice and replayed in turn, with inputs that change in place."""
    rope = _rope(64)
    graphs = []
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for seed in (40, 50):
        t, dy = _step_inputs(seed)
        with torch.cuda.stream(side):
            _step(t, rope, dy)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = _step(t, rope, dy)
        graphs.append((g, t, dy, out))
    for seed in (60, 70):
        for i, (g, t, dy, out) in enumerate(graphs):
            new, ndy = _step_inputs(seed + i)
            for k in t:
                t[k].copy_(new[k])
            dy.copy_(ndy)
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i, (_, t, dy, out) in enumerate(graphs):
            want = _step(*(lambda a: (a[0], rope, a[1]))(_step_inputs(seed + i)))
            assert all(torch.equal(a, b) for a, b in zip(out, want))


# ------------------------------------------------------------------------------------ together, as used


class _Weight:
    """What the fused linear layer reads of a flattened parameter."""

    def __init__(self, n, k, seed):
        self.data = torch.randn(n, k, generator=_gen(seed), device=DEV) / math.sqrt(k)
        self.w16 = self.data.to(BF)
        self.main_grad = torch.zeros_like(self.data)
        self.shape = self.data.shape


def _decoder(x0, w, ws, rope, tokens, B, S, H):
    """norm -> qkv -> rotary attention -> projection -> post norm, gate, residual, next norm -> head -> log
    probabilities, on the framework's kernels."""
    from mtorus.ops.attention import causal_attention
    from mtorus.ops.fused import LinearFn
    from mtorus.ops.logprobs import token_logprobs
    from mtorus.ops.residual_norm import residual_norm, rms_norm

    n0 = rms_norm(x0, ws["first"])
    qkv = LinearFn.apply(n0, None, (w["qkv"], None))
    a = causal_attention(qkv, B, S, H, 128, rotary=rope)
    h = LinearFn.apply(a, None, (w["proj"], None))
    y, n = residual_norm(x0, h, pre_weight=ws["pre"], post_weight=ws["post"], gate=ws["gate"], branch_scale=0.7)
    logits = LinearFn.apply(n, None, (w["head"], None))
    return y, token_logprobs(logits, tokens, entropy=True, top=4)


def _decoder64(x0, w, ws, rope, tokens, B, S, H):
    d = H * 128
    n0, _ = _rms(x0, ws["first"], 1e-6)
    qkv = (n0 @ w["qkv"].t()).view(B, S, 3 * H, 128)
    freq = torch.tensor(rope.frequencies, dtype=torch.float64, device=DEV)
    ang = torch.arange(S, device=DEV).double()[None, :, None, None] * freq
    a, b = qkv[:, :, :2 * H, :64], qkv[:, :, :2 * H, 64:]
    qk = torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)
    q, k, v = (t.transpose(1, 2) for t in (qk[:, :, :H], qk[:, :, H:], qkv[:, :, 2 * H:]))
    sc = (q @ k.transpose(-1, -2) / math.sqrt(128)).masked_fill(
        torch.ones(S, S, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
    o = (torch.softmax(sc, -1) @ v).transpose(1, 2).reshape(B * S, d)
    y = x0 + 0.7 * ws["gate"] * _rms(o @ w["proj"].t(), ws["post"], 1e-6)[0]
    lp = torch.log_softmax(_rms(y, ws["pre"], 1e-6)[0] @ w["head"].t(), -1)
    return y, lp.gather(-1, tokens[:, None])[:, 0], -(lp.exp() * lp).sum(-1)


def test_decoder_block_with_all_three():
    B, S, H, V = 2, 128, 2, 1000
    d = H * 128
    g = _gen(80)
    x0 = torch.randn(B * S, d, generator=g, device=DEV).to(BF)
    tokens = torch.randint(0, V, (B * S,), generator=g, device=DEV)
    w = {"qkv": _Weight(3 * d, d, 81), "proj": _Weight(d, d, 82), "head": _Weight(V, d, 83)}
    ws = {k: 1 + 0.1 * torch.randn(d, generator=g, device=DEV) for k in ("first", "pre", "post", "gate")}
    rope = _rope(128)
    leaf = {k: v.clone().requires_grad_() for k, v in ws.items()}
    xl = x0.clone().requires_grad_()
    y, r = _decoder(xl, w, leaf, rope, tokens, B, S, H)
    (-(r.logprob.mean()) - 0.1 * r.entropy.mean()).backward()

    leaf64 = {k: v.double().requires_grad_() for k, v in ws.items()}
    w64 = {k: v.w16.double().requires_grad_() for k, v in w.items()}
    x64 = x0.double().requires_grad_()
    y64, lp64, ent64 = _decoder64(x64, w64, leaf64, rope, tokens, B, S, H)
    (-(lp64.mean()) - 0.1 * ent64.mean()).backward()

    def rel(a, b):
        return ((a.double() - b.double()).norm() / b.double().norm()).item()

    # bf16 roundings one after another on the way (norm, qkv, rotary, P, O, projection, y / n, logits): 8 of at most
    # 2^-8 each; the gradient passes the same tensors back
    fwd, bwd = 8 * 2.0 ** -8, 16 * 2.0 ** -8
    assert rel(y, y64) <= fwd and rel(r.logprob, lp64) <= fwd and rel(r.entropy, ent64) <= fwd
    assert rel(xl.grad, x64.grad) <= bwd
    for k in leaf:
        assert rel(leaf[k].grad, leaf64[k].grad) <= bwd, k
    for k in w:
        assert rel(w[k].main_grad, w64[k].grad) <= bwd, k


def test_causal_attention_rotary_equals_its_parts():
    from mtorus.ops.attention import causal_attention
    from mtorus.ops.rotary import rotary_qkv

    B, S, H = 2, 256, 3
    g = _gen(90)
    qkv = torch.randn(B * S, 3 * H * 128, generator=g, device=DEV).to(BF)
    dout = torch.randn(B * S, H * 128, generator=g, device=DEV).to(BF)
    rope = _rope(128, layout="interleaved", rot_dim=64)
    pos = torch.randint(0, 3000, (B, S), generator=g, device=DEV)
    a = qkv.clone().requires_grad_()
    oa = causal_attention(a, B, S, H, 128, rotary=rope, positions=pos)
    b = qkv.clone().requires_grad_()
    ob = causal_attention(rotary_qkv(b, B, S, H, rope, pos), B, S, H, 128)
    assert torch.equal(oa, ob)
    (ga,) = torch.autograd.grad(oa, a, dout)
    (gb,) = torch.autograd.grad(ob, b, dout)
    # dQ is accumulated with reduce-adds whose order may differ between the two calls (bf16 outputs of one fp32
    # sum: at most one step apart, then rotated)
    assert ((ga.double() - gb.double()).norm() / gb.double().norm()).item() <= 2.0 ** -7
    assert torch.equal(ga.view(B, S, 3 * H, 128)[:, :, 2 * H:], gb.view(B, S, 3 * H, 128)[:, :, 2 * H:])


def test_model_scores_tokens():
    from mtorus.models.gpt import GptConfig, GptModel

    cfg = GptConfig(1000, 256, 2, 2, 512, 128, 0.0)
    model = GptModel(cfg, init="normal").to(DEV)
    g = _gen(91)
    ids = torch.randint(0, 1000, (2, 129), generator=g, device=DEV)
    with torch.no_grad():
        lp = torch.log_softmax(model(ids[:, :-1]).float(), -1)
    model.flatten(DEV)
    tgt = ids[:, 1:].clone()
    tgt[0, :5] = -100
    r = model.fused_token_logprobs(ids[:, :-1], tgt, top=5, entropy=True)
    assert r.logprob.shape == (2, 128) and r.top_ids.shape == (2, 128, 5)
    use = tgt >= 0
    want = torch.where(use, lp.gather(-1, tgt.clamp(min=0)[..., None])[..., 0], 0.0)
    # logits of about 0.3 in bf16 after a chain of bf16 products: 16 roundings of 2^-9 of logits below 4
    assert (r.logprob - want).abs().max() <= 16 * 2.0 ** -9 * 4
    assert (r.top_logprobs[..., 0] - lp.amax(-1)).abs().max() <= 16 * 2.0 ** -9 * 4
    assert not r.logprob.requires_grad
    # in the middle of a training with dropout and FP8: the same scores, and the training's state untouched
    model.config.dropout = 0.5
    model.enable_dropout(3)
    model.enable_fp8(recipe="tensor")
    key, cursor = model.dropout_state.rng.clone(), model.fp8_state.state_dict()
    again = model.fused_token_logprobs(ids[:, :-1], tgt, top=5, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(r, again))
    assert torch.equal(key, model.dropout_state.rng)
    after = model.fp8_state.state_dict()
    assert str(after) == str(cursor)
