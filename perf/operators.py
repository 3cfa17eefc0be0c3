"""Cases that measure the decoder operators around the matrix products and the attention kernel.

Three operators, each forward and backward:

* ``rotary``   -- rotary positions on q and k, or on a packed q | k | v matrix (``mtorus.ops.rotary``);
* ``norm``     -- the residual update of a block with its post norm, gate and scales, and the next block's
  pre norm, in one operator (``mtorus.ops.residual_norm``);
* ``logprobs`` -- log probabilities of given tokens with entropy and top alternatives
  (``mtorus.ops.logprobs``).

``run`` computes them in plain torch (32 bits, rounded once at the end) while ``own`` is false and through the
framework's entry points while it is true.  ``exact`` computes the same from the definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoding step of 8 sequences far into a stretched context: grouped heads, a position per sequence
        dict(name="rotary decode 8x1", op="rotary", form="qk", grad=False, B=8, S=1, heads=32, kv_heads=8, dim=128,
             rot=128, layout="half", scaling="yarn", factor=16.0, original=8192, positions="random", dtype="bf16"),
        # the training batch of the 1B benchmark configuration: 8 x 2048 tokens, 16 heads, packed q | k | v
        dict(name="rotary train qkv 8x2048", op="rotary", form="qkv", grad=True, B=8, S=2048, heads=16, kv_heads=16,
             dim=128, rot=128, layout="half", scaling="none", factor=1.0, original=2048, positions="none", dtype="bf16"),
        # odd sequence length, half of each 64-wide head rotated, neighbouring pairs; q and k are views of one matrix
        dict(name="rotary interleaved 3x1021", op="rotary", form="qk", grad=True, B=3, S=1021, heads=32, kv_heads=32,
             dim=64, rot=32, layout="interleaved", scaling="linear", factor=4.0, original=2048, positions="none",
             dtype="fp16"),
        # prefill of one long document with positions of packed documents, grouped heads
        dict(name="rotary prefill 1x32769", op="rotary", form="qk", grad=False, B=1, S=32769, heads=32, kv_heads=8,
             dim=128, rot=128, layout="half", scaling="ntk", factor=8.0, original=4096, positions="documents",
             dtype="bf16"),
        # one decoding step: latency of the whole residual update
        dict(name="norm decode 8x2048", op="norm", grad=False, rows=8, d=2048, post=True, pre=True, gate="channel",
             beta=1.0, alpha=1.0, dtype="bf16"),
        # training batch of the 1B benchmark configuration, norms on both sides and a learned gate per channel
        dict(name="norm train 16384x2048", op="norm", grad=True, rows=16384, d=2048, post=True, pre=True,
             gate="channel", beta=1.0, alpha=1.0, dtype="bf16"),
        # width of the 6.7B configuration, no post norm, a scalar gate per token and a depth-scaled branch
        dict(name="norm train 4096x4096", op="norm", grad=True, rows=4096, d=4096, post=False, pre=True, gate="row",
             beta=1.0, alpha=0.125, dtype="bf16"),
        # ragged width in 32 bits with a gate computed per element
        dict(name="norm ragged 1531x1003", op="norm", grad=True, rows=1531, d=1003, post=True, pre=True, gate="full",
             beta=0.5, alpha=0.75, dtype="fp32"),
        # sampling step of 4 sequences over the padded 50304 vocabulary: chosen token, entropy, 8 alternatives
        dict(name="logprobs decode 4x50304", op="logprobs", grad=False, rows=4, vocab=50304, pad=47, tau=0.8, top=8,
             entropy=True, dtype="bf16"),
        # policy-gradient step: log probabilities and entropy of 8192 tokens with their gradient
        dict(name="logprobs train 8192x50304", op="logprobs", grad=True, rows=8192, vocab=50304, pad=47, tau=1.0,
             top=0, entropy=True, dtype="bf16"),
        # scoring a document over the unpadded vocabulary (rows off any 16-byte boundary) with 20 alternatives
        dict(name="logprobs score 2048x50257", op="logprobs", grad=False, rows=2048, vocab=50257, pad=0, tau=1.0,
             top=20, entropy=False, dtype="bf16"),
        # distillation from the top alternatives of 32-bit logits over a large vocabulary, gradient included
        dict(name="logprobs distil 257x131072", op="logprobs", grad=True, rows=257, vocab=131072, pad=0, tau=2.0,
             top=5, entropy=True, dtype="fp32"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    grad = rng.random() < 0.5
    if op == "rotary":
        form = rng.choice(["qk", "qkv"])
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 4])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        tokens = _log_uniform(rng, 1, min(32768, (1 << 26) // (dim * (heads + 2 * kv))))
        B = min(tokens, rng.choice([1, 1, 2, 3, 8, 32]))
        return dict(op=op, form=form, grad=grad, B=B, S=max(1, tokens // B), heads=heads, kv_heads=kv, dim=dim,
                    rot=rot, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), factor=rng.choice([2.0, 4.0, 8.0, 32.0]),
                    original=rng.choice([2048, 4096, 8192]), positions=rng.choice(["none", "random", "documents"]),
                    dtype=dtype)
    if op == "norm":
        d = _log_uniform(rng, 48, 8192)
        d = d if rng.random() < 0.3 else max(64, d // 64 * 64)
        rows = _log_uniform(rng, 1, min(32768, (1 << 25) // d))
        post = rng.random() < 0.6
        return dict(op=op, grad=grad, rows=rows, d=d, post=post, pre=True if not post else rng.random() < 0.8,
                    gate=rng.choice(["none", "channel", "row", "full"]), beta=rng.choice([1.0, 1.0, 0.5]),
                    alpha=rng.choice([1.0, 0.25, 0.75]), dtype=dtype)
    vocab = _log_uniform(rng, 256, 160000)
    vocab = vocab if rng.random() < 0.3 else max(256, vocab // 64 * 64)
    rows = _log_uniform(rng, 1, min(16384, (1 << 27) // vocab))
    return dict(op=op, grad=grad, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 7, 47]),
                tau=rng.choice([1.0, 1.0, 0.7, 2.0]), top=rng.choice([0, 0, 1, 5, 20]), entropy=rng.random() < 0.6,
                dtype=dtype)


# ---------------------------------------------------------------------------------------------------- inputs


def _frequencies(case):
    """Angle per position of each pair (64 bits) and the factor on the rotated values."""
    r, base = case["rot"], 10000.0
    f = case["factor"]
    i = torch.arange(0, r // 2, dtype=torch.float64)
    if case["scaling"] == "ntk":
        base = base * f ** (r / (r - 2)) if r > 2 else base
    w = base ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return w / f, 1.0
    if case["scaling"] == "yarn":
        def index_of(turns):
            return r * math.log(case["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(index_of(32.0)), 0), min(math.ceil(index_of(1.0)), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return w / f * ramp + w * (1 - ramp), 0.1 * math.log(f) + 1.0
    return w, 1.0


def _prepare_rotary(case, g, state):
    dt, dev = _DTYPES[case["dtype"]], "cuda"
    B, S, H, K, D = (case[k] for k in ("B", "S", "heads", "kv_heads", "dim"))
    width = (H + 2 * K) * D
    qkv = torch.randn(B * S, width, generator=g, device=dev).to(dt)
    state["dqkv"] = (torch.randn(B * S, width, generator=g, device=dev) * 0.01).to(dt)
    if case["positions"] == "random":  # a position per sequence, its tokens following one another
        start = torch.randint(0, 4 * case["original"], (B, 1), generator=g, device=dev)
        state["positions"] = start + torch.arange(S, device=dev)
    elif case["positions"] == "documents":  # several documents in a row, each from position 0
        cut = torch.rand(B, S, generator=g, device=dev) < 4.0 / S
        cut[:, 0] = True
        at = torch.arange(S, device=dev).expand(B, S)
        state["positions"] = at - torch.where(cut, at, 0).cummax(dim=1).values
    else:
        state["positions"] = None
    w, scale = _frequencies(case)
    state["w"], state["scale"] = w.to(dev), scale
    if case["form"] == "qkv":
        state["qkv"] = qkv.requires_grad_(case["grad"])
    else:  # views of the packed matrix: rows further apart than their own width
        q, k = qkv[:, : H * D].view(B, S, H, D), qkv[:, H * D: (H + K) * D].view(B, S, K, D)
        state["q"], state["k"] = (t.detach().requires_grad_(case["grad"]) for t in (q, k))
        state["dq"] = state["dqkv"][:, : H * D].reshape(B, S, H, D)
        state["dk"] = state["dqkv"][:, H * D: (H + K) * D].reshape(B, S, K, D)
    if own:  # the handle that a program builds once for a model
        from mtorus.ops.rotary import RotaryPositions

        state["rope"] = RotaryPositions(D, rot_dim=case["rot"], base=10000.0, layout=case["layout"],
                                        scaling=case["scaling"], factor=case["factor"],
                                        original_len=case["original"], device=dev)


def _prepare_norm(case, g, state):
    dt, dev, T, d = _DTYPES[case["dtype"]], "cuda", case["rows"], case["d"]

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev) * scale

    # a residual stream that has grown over some layers, with a few large channels
    x = rand(T, d, scale=3.0) * torch.where(torch.rand(d, generator=g, device=dev) < 0.01, 8.0, 1.0)
    state["x"], state["h"] = x.to(dt), rand(T, d).to(dt)
    state["pre"] = 1.0 + rand(d, scale=0.1) if case["pre"] else None
    state["post"] = 1.0 + rand(d, scale=0.1) if case["post"] else None
    state["gate"] = {"none": lambda: None, "channel": lambda: rand(d, scale=0.5),
                     "row": lambda: torch.rand(T, 1, generator=g, device=dev),
                     "full": lambda: torch.sigmoid(rand(T, d)).to(dt)}[case["gate"]]()
    state["dy"] = rand(T, d, scale=0.02).to(dt)
    state["dn"] = rand(T, d, scale=0.05).to(dt) if case["pre"] else None
    for k in ("x", "h", "pre", "post", "gate"):
        if state[k] is not None:
            state[k].requires_grad_(case["grad"])


def _prepare_logprobs(case, g, state):
    dt, dev, T, V = _DTYPES[case["dtype"]], "cuda", case["rows"], case["vocab"]
    x = torch.randn(T, V, generator=g, device=dev) * 2.5
    tokens = torch.randint(0, V - case["pad"], (T,), generator=g, device=dev)
    # tokens that a trained model finds likely, some of them nearly certain
    lift = torch.rand(T, 1, generator=g, device=dev) * 16.0
    x.scatter_add_(1, tokens[:, None], lift)
    if case["pad"]:  # columns that fill the vocabulary up are masked
        x[:, V - case["pad"]:] = float("-inf")
    # prompt tokens, which the loss leaves out
    state["tokens"] = torch.where(torch.rand(T, generator=g, device=dev) < 0.05, -100, tokens)
    state["logits"] = x.to(dt).requires_grad_(case["grad"])
    unit = 1.0 if dt == torch.float16 else 1.0 / T  # 16-bit training scales its loss, so that gradients are not lost
    state["dlogprob"] = torch.randn(T, generator=g, device=dev) * unit
    state["dentropy"] = torch.full((T,), -0.01 * unit, device=dev)
    state["dtop"] = -torch.rand(T, max(1, case["top"]), generator=g, device=dev) * unit


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    {"rotary": _prepare_rotary, "norm": _prepare_norm, "logprobs": _prepare_logprobs}[case["op"]](case, g, state)
    return state


# ---------------------------------------------------------------------------------------------------- plain forms


def _rotate(x, cos, sin, case):
    """x [B, S, H, D] in 32 bits; cos, sin [B or 1, S, 1, r / 2]."""
    r = case["rot"]
    if case["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], dim=-1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_rotary(state):
    case = state["case"]
    B, S, H, K, D = (case[k] for k in ("B", "S", "heads", "kv_heads", "dim"))
    pos = state["positions"]
    pos = torch.arange(S, device="cuda")[None] if pos is None else pos
    angle = pos[..., None, None].double() * state["w"]
    cos, sin = (torch.cos(angle) * state["scale"]).float(), (torch.sin(angle) * state["scale"]).float()
    dt = _DTYPES[case["dtype"]]
    if case["form"] == "qk":
        out = {"q": _rotate(state["q"].detach().float(), cos, sin, case).to(dt),
               "k": _rotate(state["k"].detach().float(), cos, sin, case).to(dt)}
        if case["grad"]:
            out["dq"] = _rotate(state["dq"].float(), cos, -sin, case).to(dt)
            out["dk"] = _rotate(state["dk"].float(), cos, -sin, case).to(dt)
        return out

    def packed(x, sin):
        x = x.view(B, S, H + 2 * K, D)
        turned = _rotate(x[:, :, : H + K].float(), cos, sin, case).to(dt)
        return torch.cat([turned, x[:, :, H + K:]], dim=2).view(B * S, -1)

    out = {"qkv": packed(state["qkv"].detach(), sin)}
    if case["grad"]:
        out["dqkv"] = packed(state["dqkv"], -sin)
    return out


def _plain_norm(state):
    case, eps = state["case"], 1e-6
    alpha, beta, dt = case["alpha"], case["beta"], _DTYPES[case["dtype"]]
    x, h = state["x"].detach().float(), state["h"].detach().float()
    pre, post, gate = (None if state[k] is None else state[k].detach().float() for k in ("pre", "post", "gate"))
    b = h
    if post is not None:
        rh = torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
        hh = h * rh
        b = hh * post
    ag = alpha if gate is None else alpha * gate
    y = beta * x + ag * b
    out = {"y": y.to(dt)}
    if pre is not None:
        ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        yh = y * ry
        out["n"] = (yh * pre).to(dt)
    if not case["grad"]:
        return out
    dy = state["dy"].float()
    if pre is not None:
        dn = state["dn"].float()
        u = dn * pre
        out["dpre"] = (dn * yh).sum(0)
        dy = dy + ry * (u - yh * (u * yh).mean(-1, keepdim=True))
    out["dx"] = (beta * dy).to(dt)
    if gate is not None:
        dg = alpha * b * dy
        out["dgate"] = {"channel": lambda: dg.sum(0), "row": lambda: dg.sum(1, keepdim=True),
                        "full": lambda: dg.to(dt)}[case["gate"]]()
    db = ag * dy
    if post is not None:
        out["dpost"] = (db * hh).sum(0)
        v = db * post
        db = rh * (v - hh * (v * hh).mean(-1, keepdim=True))
    out["dh"] = db.to(dt)
    return out


def _plain_logprobs(state):
    case = state["case"]
    k, inv_tau, V = case["top"], 1.0 / case["tau"], case["vocab"]
    logits, tokens = state["logits"].detach(), state["tokens"]
    z = logits.float()
    m = z.amax(-1, keepdim=True)
    lp = (z - m) * inv_tau
    lp = lp - torch.log(torch.exp(lp).sum(-1, keepdim=True))
    use = (tokens >= 0) & (tokens < V)
    at = torch.where(use, tokens, 0)[:, None]
    out = {"logprob": torch.where(use, lp.gather(1, at)[:, 0], 0.0)}
    if case["entropy"] or case["grad"]:
        p = torch.exp(lp)
    if case["entropy"]:
        out["entropy"] = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    if k:
        # one whole number per logit that orders by value, then by lowest index
        bits = z.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = (order << 20) | (V - 1 - torch.arange(V, device=z.device))
        out["top_ids"] = V - 1 - (torch.topk(key, k, dim=-1).values & 0xFFFFF)
        out["top_logprobs"] = lp.gather(1, out["top_ids"])
    if case["grad"]:
        g = torch.where(use, state["dlogprob"], 0.0)
        total = g + state["dtop"][:, :k].sum(-1) if k else g
        d = -total[:, None] * p
        if case["entropy"]:
            d -= state["dentropy"][:, None] * torch.where(p > 0, p * (lp + out["entropy"][:, None]), 0.0)
        d.scatter_add_(1, at, g[:, None])
        if k:
            d.scatter_add_(1, out["top_ids"], state["dtop"])
        out["dlogits"] = (d * inv_tau).to(logits.dtype)
    return out


# ---------------------------------------------------------------------------------------------------- the framework's calls


def _own_rotary(state):
    from mtorus.ops.rotary import rotary, rotary_qkv

    case = state["case"]
    if case["form"] == "qk":
        q, k = rotary(state["q"], state["k"], state["rope"], state["positions"])
        out = {"q": q, "k": k}
        if case["grad"]:
            out["dq"], out["dk"] = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
        return out
    qkv = rotary_qkv(state["qkv"], case["B"], case["S"], case["heads"], state["rope"], state["positions"],
                     kv_heads=case["kv_heads"])
    out = {"qkv": qkv}
    if case["grad"]:
        (out["dqkv"],) = torch.autograd.grad(qkv, state["qkv"], state["dqkv"])
    return out


def _own_norm(state):
    from mtorus.ops.residual_norm import residual_norm

    case = state["case"]
    y, n = residual_norm(state["x"], state["h"], pre_weight=state["pre"], post_weight=state["post"],
                         gate=state["gate"], residual_scale=case["beta"], branch_scale=case["alpha"], eps=1e-6)
    out = {"y": y} if n is None else {"y": y, "n": n}
    if case["grad"]:
        names = [k for k in ("x", "h", "pre", "post", "gate") if state[k] is not None]
        got = torch.autograd.grad([y] if n is None else [y, n], [state[k] for k in names],
                                  [state["dy"]] if n is None else [state["dy"], state["dn"]])
        out.update(zip(["d" + k for k in names], got))
    return out


def _own_logprobs(state):
    from mtorus.ops.logprobs import token_logprobs

    case, k = state["case"], state["case"]["top"]
    r = token_logprobs(state["logits"], state["tokens"], temperature=case["tau"], top=k, entropy=case["entropy"])
    out = {"logprob": r.logprob}
    outs, grads = [r.logprob], [state["dlogprob"]]
    if case["entropy"]:
        out["entropy"] = r.entropy
        outs.append(r.entropy)
        grads.append(state["dentropy"])
    if k:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        outs.append(r.top_logprobs)
        grads.append(state["dtop"])
    if case["grad"]:
        (out["dlogits"],) = torch.autograd.grad(outs, state["logits"], grads)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "norm": _own_norm, "logprobs": _own_logprobs}[op](state)
    return {"rotary": _plain_rotary, "norm": _plain_norm, "logprobs": _plain_logprobs}[op](state)


# ---------------------------------------------------------------------------------------------------- work and exact values


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "rotary":
        T, both = case["B"] * case["S"], 2 if case["grad"] else 1
        heads = case["heads"] + case["kv_heads"] * (2 if case["form"] == "qkv" else 1)
        turned = T * (case["heads"] + case["kv_heads"]) * case["rot"]
        return {"bytes": both * 2 * e * T * heads * case["dim"] + (0 if case["positions"] == "none" else 8 * T),
                "flops": both * 3 * turned}
    if case["op"] == "norm":
        n = case["rows"] * case["d"]
        moved = 2 + 1 + case["pre"]  # x, h; y, n
        weights = case["pre"] + case["post"] + (case["gate"] == "channel")
        small = 4 * case["rows"] * (case["gate"] == "row")
        full = case["gate"] == "full"
        flops = 4 + 3 * case["pre"] + 4 * case["post"]
        if case["grad"]:  # dy, dn; dx, dh
            moved, weights, small, flops = moved + 3 + case["pre"], 2 * weights, 2 * small, 3 * flops
        return {"bytes": e * n * (moved + full * (2 if case["grad"] else 1)) + 4 * weights * case["d"] + small,
                "flops": flops * n}
    n, T = case["rows"] * case["vocab"], case["rows"]
    rows = 8 + 4 + 4 * case["entropy"] + 12 * case["top"]
    if case["grad"]:
        rows += 4 + 4 * case["entropy"] + 4 * case["top"]
    flops = 4 + 2 * case["entropy"] + (case["grad"] and 5 + 2 * case["entropy"])
    return {"bytes": e * n * (2 if case["grad"] else 1) + rows * T, "flops": flops * n}


def _exact_rotary(case, state):
    B, S, H, K, D, r = (case[k] for k in ("B", "S", "heads", "kv_heads", "dim", "rot"))
    pos = state["positions"]
    pos = torch.arange(S, device="cuda").expand(B, S) if pos is None else pos
    angle = pos.double().unsqueeze(-1) * state["w"]  # [B, S, r / 2]
    turn = torch.polar(torch.full_like(angle, state["scale"]), angle).unsqueeze(2)

    def rotated(x, turn, heads):  # the pairs as complex numbers times a complex number
        x = x.detach().double().reshape(B, S, -1, D)
        out = x.clone()
        if case["layout"] == "half":
            c = torch.complex(x[:, :, :heads, : r // 2], x[:, :, :heads, r // 2: r]) * turn
            out[:, :, :heads, : r // 2], out[:, :, :heads, r // 2: r] = c.real, c.imag
        else:
            c = torch.view_as_complex(x[:, :, :heads, :r].reshape(B, S, heads, r // 2, 2).contiguous()) * turn
            out[:, :, :heads, :r] = torch.view_as_real(c).reshape(B, S, heads, r)
        return out

    if case["form"] == "qkv":
        out = {"qkv": rotated(state["qkv"], turn, H + K).view(B * S, -1)}
        if case["grad"]:
            out["dqkv"] = rotated(state["dqkv"], turn.conj(), H + K).view(B * S, -1)
        return out
    out = {"q": rotated(state["q"], turn, H), "k": rotated(state["k"], turn, K)}
    if case["grad"]:
        out["dq"], out["dk"] = rotated(state["dq"], turn.conj(), H), rotated(state["dk"], turn.conj(), K)
    return out


def _exact_norm(case, state):
    def rms(t, w):
        return t / torch.sqrt(torch.mean(t * t, dim=-1, keepdim=True) + 1e-6) * w

    names = [k for k in ("x", "h", "pre", "post", "gate") if state[k] is not None]
    v = {k: state[k].detach().double().requires_grad_(case["grad"]) for k in names}
    b = rms(v["h"], v["post"]) if case["post"] else v["h"]
    if "gate" in v:
        b = b * v["gate"]
    y = case["beta"] * v["x"] + case["alpha"] * b
    out, grads = {"y": y}, [state["dy"].double()]
    if case["pre"]:
        out["n"] = rms(y, v["pre"])
        grads.append(state["dn"].double())
    if case["grad"]:
        got = torch.autograd.grad(list(out.values()), [v[k] for k in names], grads)
        out.update(zip(["d" + k for k in names], got))
    return {k: t.detach() for k, t in out.items()}


def _exact_logprobs(case, state):
    x = state["logits"].detach()
    k, V = case["top"], case["vocab"]
    out = {}
    if k:  # a stable sort keeps the lowest index first among equals
        out["top_ids"] = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :k].contiguous()
    z = x.double()
    z = torch.where(torch.isinf(z), -1e5, z).requires_grad_(case["grad"])  # exp gives 0 in 64 bits
    lp = torch.log_softmax(z / case["tau"], dim=-1)
    tokens = state["tokens"]
    ignored = (tokens < 0) | (tokens >= V)
    out["logprob"] = lp.gather(1, tokens.masked_fill(ignored, 0)[:, None])[:, 0].masked_fill(ignored, 0.0)
    outs, grads = [out["logprob"]], [state["dlogprob"].double()]
    if case["entropy"]:
        out["entropy"] = -(lp.exp() * lp).sum(-1)
        outs.append(out["entropy"])
        grads.append(state["dentropy"].double())
    if k:
        out["top_logprobs"] = lp.gather(1, out["top_ids"])
        outs.append(out["top_logprobs"])
        grads.append(state["dtop"].double())
    if case["grad"]:
        (out["dlogits"],) = torch.autograd.grad(outs, z, grads)
    return {n: t.detach() for n, t in out.items()}


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "norm": _exact_norm, "logprobs": _exact_logprobs}[case["op"]](case, state)
