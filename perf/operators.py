"""Cases for the operators that carry a transformer block's activations in eight bits between its linear layers:

* ``linear`` / ``gemm``: the product of 8-bit integers with one scale per token and one per output channel, with and
  without the token-wise quantisation of its input;
* ``norm_forward`` / ``norm_backward``: the norm after a block, its gate and residual scale, the residual sum and the
  norm before the next block as one operator, and the gradient, from full tensors or from 8-bit checkpoints;
* ``silu``: a training step of SwiGLU that keeps an 8-bit checkpoint of its input instead of the input.

``own`` false: elementary torch operations in float32.  ``own`` true: the framework's entry points."""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
FLOOR = 1e-30
EPS = 1e-6
RESIDUAL = 0.75


def listed():
    return [
        # one token through a square projection: the latency of a decoding step
        {"name": "linear_one_token", "op": "linear", "m": 1, "k": 4096, "n": 4096, "dtype": "bf16", "smooth": False},
        # a small decoding batch through an up projection, smoothed
        {"name": "linear_six_tokens", "op": "linear", "m": 6, "k": 2048, "n": 8192, "dtype": "f16", "smooth": True},
        # a short prompt (or a verified draft) through a projection
        {"name": "linear_short_prompt", "op": "linear", "m": 200, "k": 4096, "n": 4096, "dtype": "bf16", "smooth": True},
        # codes at hand, float32 result, no size a multiple of a tile
        {"name": "gemm_ragged", "op": "gemm", "m": 1000, "k": 2064, "n": 1111, "dtype": "f32"},
        # a training or prefill batch of the repository's own width
        {"name": "linear_batch", "op": "linear", "m": 8192, "k": 4096, "n": 8192, "dtype": "bf16", "smooth": False},
        # a decoding step between two blocks
        {"name": "norm_fwd_decode", "op": "norm_forward", "s": 1, "b": 16, "n": 4096, "dtype": "bf16", "gate": "none"},
        # a training batch, one gate value per channel
        {"name": "norm_fwd_batch", "op": "norm_forward", "s": 8192, "b": 2, "n": 4096, "dtype": "bf16", "gate": "channel"},
        # the gradient of the same batch from the full tensors
        {"name": "norm_bwd_batch", "op": "norm_backward", "s": 8192, "b": 2, "n": 4096, "dtype": "bf16", "gate": "channel", "codes": "none"},
        # the gradient from 8-bit checkpoints, a gate for each sample, odd lengths, a wide row that is no power of two
        {"name": "norm_bwd_checkpoint", "op": "norm_backward", "s": 1001, "b": 5, "n": 5120, "dtype": "f16", "gate": "sample", "codes": "int8"},
        # a routed expert's few tokens, each with its routing weight
        {"name": "silu_few_rows", "op": "silu", "m": 77, "n": 512, "dtype": "bf16", "codes": "e4m3", "weighted": True},
        # the routed tokens of all experts, each with its routing weight
        {"name": "silu_routed", "op": "silu", "m": 40001, "n": 1408, "dtype": "bf16", "codes": "e4m3", "weighted": True},
        # the dense feed-forward of a training batch
        {"name": "silu_dense", "op": "silu", "m": 16384, "n": 8192, "dtype": "bf16", "codes": "int8", "weighted": False},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _type(rng):
    return rng.choice(["bf16", "bf16", "f16", "f32"])


def draw(rng):
    op = rng.choice(["linear", "linear", "gemm", "norm_forward", "norm_backward", "norm_backward", "silu", "silu"])
    if op in ("linear", "gemm"):
        m, k, n = _log(rng, 1, 8192), 16 * _log(rng, 8, 512), _log(rng, 32, 8192)
        if rng.random() < 0.5:
            n = max(64, n // 64 * 64)
        m = min(m, 8192 * 4096 * 8192 // (k * n))
        case = {"op": op, "m": m, "k": k, "n": n, "dtype": _type(rng)}
        if op == "linear":
            case["smooth"] = rng.random() < 0.5
        return case
    if op == "silu":
        n = 128 * _log(rng, 1, 64)
        return {"op": op, "m": min(_log(rng, 1, 65536), 16384 * 8192 // 2 // n), "n": n, "dtype": _type(rng),
                "codes": rng.choice(["int8", "e4m3"]), "weighted": rng.random() < 0.5}
    n, b = 128 * _log(rng, 1, 64), rng.randint(1, 8)
    s = max(1, min(_log(rng, 1, 16384), 16384 * 4096 // 2 // (b * n)))
    case = {"op": op, "s": s, "b": b, "n": n, "dtype": _type(rng), "gate": rng.choice(["none", "channel", "sample", "token"])}
    if op == "norm_backward":
        case["codes"] = rng.choice(["none", "int8", "e4m3"])
    return case


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _over(amax, top):
    # a quotient of two tensors is rounded once; a tensor over a Python number is multiplied by a rounded reciprocal
    return (amax / torch.full_like(amax, top)).clamp_min(FLOOR)


def _codes(x, kind):
    """8-bit codes and the float32 scale of each 1 x 128 block of the rows of x."""
    blocks = x.float().reshape(x.shape[0], -1, 128)
    scale = _over(blocks.abs().amax(2), TOP[kind])
    q = blocks / scale[:, :, None]
    q = q.round() if kind == "int8" else q
    return q.to(CODES[kind]).reshape(x.shape), scale


def _values(q, scale):
    return (q.float().reshape(q.shape[0], -1, 128) * scale[:, :, None]).reshape(q.shape)


def _token_codes(x, smooth):
    """8-bit integers and one float32 scale per row of x, after the division by the smoothing factors."""
    x = x.float()
    if smooth is not None:
        x = x / smooth.clamp_min(FLOOR)
    scale = _over(x.abs().amax(1), 127.0)
    return (x / scale[:, None]).round(), scale


def _norm_state(case, g):
    s, b, n, t = case["s"], case["b"], case["n"], TYPES[case["dtype"]]
    gate = {"none": None, "channel": (n,), "sample": (b, n), "token": (s, b, n)}[case["gate"]]
    st = {
        "x": _normal(g, s, b, n).to(t),
        "o": (_normal(g, s, b, n) * (0.3 + 3 * torch.rand((s, b, 1), generator=g, device="cuda"))).to(t),
        "post": (1 + 0.2 * _normal(g, n)).to(t),
        "pre": (1 + 0.2 * _normal(g, n)).to(t),
        "gate": None if gate is None else torch.sigmoid(_normal(g, *gate)).to(t),
    }
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st, op = {"case": case}, case["op"]
    if op in ("linear", "gemm"):
        m, k, n, t = case["m"], case["k"], case["n"], TYPES[case["dtype"]]
        w = _normal(g, n, k) * (0.5 + torch.rand((n, 1), generator=g, device="cuda")) / math.sqrt(k)
        x = _normal(g, m, k) * torch.exp(0.7 * _normal(g, k))
        st["smooth"] = None
        if case.get("smooth"):
            st["smooth"] = (x.abs().amax(0).clamp_min(1e-3) / w.abs().amax(0)).sqrt()
            w = w * st["smooth"]
        q, st["w_scale"] = _token_codes(w, None)
        st["w"] = q.to(torch.int8)
        if op == "gemm":
            q, st["x_scale"] = _token_codes(x, None)
            st["x"] = q.to(torch.int8)
        else:
            st["x"] = x.to(t)
        return st
    if op == "silu":
        m, n, t = case["m"], case["n"], TYPES[case["dtype"]]
        st["x"] = _normal(g, m, 2 * n).mul_(1.5).to(t)
        st["g"] = _normal(g, m, n).mul_(0.02).to(t)
        st["w"] = torch.rand(m, generator=g, device="cuda") if case["weighted"] else None
        return st
    st.update(_norm_state(case, g))
    if op == "norm_forward":
        return st
    # what the forward pass left behind
    rows, n = case["s"] * case["b"], case["n"]
    o = st["o"].float()
    st["rms_post"] = torch.rsqrt(o.square().mean(2) + EPS).reshape(rows)
    p = o * st["rms_post"].reshape(case["s"], case["b"], 1) * st["post"].float() * RESIDUAL
    if st["gate"] is not None:
        p = p * st["gate"].float()
    h = (st.pop("x").float() + p).to(st["o"].dtype)
    st["rms_pre"] = torch.rsqrt(h.float().square().mean(2) + EPS).reshape(rows)
    st["h"], st["o_scale"], st["h_scale"] = h, None, None
    if case["codes"] != "none":
        for name in ("o", "h"):
            q, st[name + "_scale"] = _codes(st[name].reshape(rows, n), case["codes"])
            st[name] = q.reshape(h.shape)
    st["grad_y"] = (0.05 * _normal(g, *h.shape)).to(h.dtype)
    st["grad_h"] = (0.05 * _normal(g, *h.shape)).to(h.dtype)
    return st


def run(st):
    op = st["case"]["op"]
    if own:
        return _run_own(st, op)
    if op == "linear":
        q, scale = _token_codes(st["x"], st["smooth"])
        return ((q @ st["w"].float().t()) * scale[:, None] * st["w_scale"]).to(st["x"].dtype)
    if op == "gemm":
        acc = st["x"].float() @ st["w"].float().t()
        return (acc * st["x_scale"][:, None] * st["w_scale"]).to(TYPES[st["case"]["dtype"]])
    if op == "silu":
        return _plain_silu(st)
    return _plain_norm_forward(st) if op == "norm_forward" else _plain_norm_backward(st)


def _plain_silu(st):
    x, g, w, n = st["x"].float(), st["g"].float(), st["w"], st["g"].shape[1]
    y = x[:, :n] / (1 + torch.exp(-x[:, :n])) * x[:, n:]
    if w is not None:
        y = y * w[:, None]
    # the backward pass sees the checkpoint only
    c = _values(*_codes(st["x"], st["case"]["codes"]))
    a, b = c[:, :n], c[:, n:]
    sig = 1 / (1 + torch.exp(-a))
    dw = None
    if w is not None:
        dw = (g * a * sig * b).sum(1)
        g = g * w[:, None]
    dx = torch.cat([g * b * sig * (1 + a * (1 - sig)), g * a * sig], 1)
    out = (y.to(st["x"].dtype), dx.to(st["x"].dtype))
    return out if dw is None else out + (dw,)


def _plain_norm_forward(st):
    t = st["x"].dtype
    o = st["o"].float()
    r_post = torch.rsqrt(o.square().mean(2, keepdim=True) + EPS)
    p = o * r_post * st["post"].float() * RESIDUAL
    if st["gate"] is not None:
        p = p * st["gate"].float()
    h = (st["x"].float() + p).to(t)
    hf = h.float()
    r_pre = torch.rsqrt(hf.square().mean(2, keepdim=True) + EPS)
    return h, (hf * r_pre * st["pre"].float()).to(t), r_post.reshape(-1), r_pre.reshape(-1)


def _plain_norm_backward(st):
    t, shape, n = st["grad_y"].dtype, st["h"].shape, st["h"].shape[2]
    if st["o_scale"] is None:
        o, h = st["o"].float(), st["h"].float()
    else:
        o = _values(st["o"].reshape(-1, n), st["o_scale"]).reshape(shape)
        h = _values(st["h"].reshape(-1, n), st["h_scale"]).reshape(shape)
    dy, post, gate = st["grad_y"].float(), st["post"].float(), st["gate"]
    r_pre, r_post = st["rms_pre"].reshape(shape[0], shape[1], 1), st["rms_post"].reshape(shape[0], shape[1], 1)
    hn, on = h * r_pre, o * r_post
    t1 = dy * st["pre"].float()
    dh = st["grad_h"].float() + r_pre * (t1 - hn * (t1 * hn).mean(2, keepdim=True))
    dpre = (dy * hn).reshape(-1, n).sum(0)
    dp = dh * RESIDUAL
    dgate = None
    if gate is not None:
        dgate = dp * on * post
        lead = dgate.dim() - gate.dim()
        dgate = (dgate.sum(tuple(range(lead))) if lead else dgate).to(gate.dtype)
        dp = dp * gate.float()
    dpost = (dp * on).reshape(-1, n).sum(0)
    t2 = dp * post
    do = r_post * (t2 - on * (t2 * on).mean(2, keepdim=True))
    out = (dh.to(t), do.to(t), dpost, dpre)
    return out if dgate is None else out + (dgate,)


def _run_own(st, op):
    if op == "linear":
        from linghe_b200.gemm.int8_gemm import int8_linear
        return int8_linear(st["x"], st["w"], st["w_scale"], smooth_scale=st["smooth"])
    if op == "gemm":
        from linghe_b200.gemm.int8_gemm import int8_gemm
        return int8_gemm(st["x"], st["w"], st["x_scale"], st["w_scale"], out_dtype=TYPES[st["case"]["dtype"]])
    if op == "silu":
        from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
        y, q, scale = silu_and_checkpoint_forward(st["x"], st["w"], checkpoint=CODES[st["case"]["codes"]])
        dx, dw = silu_and_checkpoint_backward(st["g"], q, scale, st["w"])
        return (y, dx) if dw is None else (y, dx, dw)
    if op == "norm_forward":
        from linghe_b200.utils.norm import rms_norm_pair_forward
        return rms_norm_pair_forward(st["x"], st["o"], st["post"], st["pre"], gate=st["gate"], residual_scale=RESIDUAL, eps=EPS)[:4]
    from linghe_b200.utils.norm import rms_norm_pair_backward
    out = rms_norm_pair_backward(st["grad_y"], st["grad_h"], st["o"], st["h"], st["post"], st["pre"], st["rms_post"], st["rms_pre"],
                                 gate=st["gate"], residual_scale=RESIDUAL, o_scale=st["o_scale"], h_scale=st["h_scale"])
    return out[:4] if out[4] is None else out


def work(case):
    op, e = case["op"], {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if op in ("linear", "gemm"):
        m, k, n = case["m"], case["k"], case["n"]
        read = m * k + 4 * m if op == "gemm" else m * k * e + (4 * k if case["smooth"] else 0)
        return {"bytes": read + n * k + 4 * n + m * n * e, "flops": 2 * m * n * k}
    if op == "silu":
        m, n = case["m"], case["n"]
        codes = m * 2 * n + 4 * m * 2 * n // 128
        forward, backward = m * 3 * n * e + codes, codes + m * 3 * n * e
        return {"bytes": forward + backward + (12 * m if case["weighted"] else 0), "flops": 30 * m * n}
    rows, n = case["s"] * case["b"], case["n"]
    gate = e * n * {"none": 0, "channel": 1, "sample": case["b"], "token": rows}[case["gate"]]
    if op == "norm_forward":
        return {"bytes": 4 * rows * n * e + 2 * n * e + gate + 8 * rows, "flops": 12 * rows * n}
    kept = 2 * rows * n * e if case["codes"] == "none" else 2 * (rows * n + 4 * rows * n // 128)
    return {"bytes": 4 * rows * n * e + kept + 2 * n * e + 8 * n + 2 * gate + 8 * rows, "flops": 35 * rows * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_codes(x, kind, block):
    """The values that the codes of each run of `block` elements stand for.  A code is defined by float32 numbers, the scale and
    the quotient that is rounded to it; each of the two is the nearest to its value in 64 bits."""
    v = x.double().unflatten(1, (-1, block))
    scale = (v.abs().amax(2, keepdim=True) / (127 if kind == "int8" else 448)).clamp_min(FLOOR).float().double()
    q = torch.div(v, scale).float().double()
    if kind == "int8":
        q = torch.round(q)
    else:  # nearest e4m3 number, ties to the even mantissa: steps of 2^(exponent - 3), none finer than 2^-9
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
        q = torch.round(q / step) * step
    return (q * scale).flatten(1)


def _stored(st, name):
    q, scale = st[name].flatten(0, 1).double(), st[name + "_scale"]
    return q if scale is None else (q.unflatten(1, (-1, 128)) * scale.double().unsqueeze(2)).flatten(1)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("linear", "gemm"):
        w = st["w"].double() * st["w_scale"].double().unsqueeze(1)
        if op == "gemm":
            x = st["x"].double() * st["x_scale"].double().unsqueeze(1)
        else:
            x = st["x"].double()
            if st["smooth"] is not None:  # the smoothed value is a float32 number too
                x = torch.div(x, st["smooth"].double()).float().double()
            x = _exact_codes(x, "int8", x.shape[1])
        return torch.einsum("mk,nk->mn", x, w)
    if op == "silu":
        n = case["n"]
        w = None if st["w"] is None else st["w"].double().requires_grad_()
        out = []
        for kept in (st["x"].double(), _exact_codes(st["x"], case["codes"], 128)):
            leaf = kept.requires_grad_()
            y = torch.sigmoid(leaf[:, :n]) * leaf[:, :n] * leaf[:, n:]
            out.append((leaf, y if w is None else y * w.unsqueeze(1)))
        (_, y), (leaf, again) = out
        grads = torch.autograd.grad(again, [leaf] if w is None else [leaf, w], st["g"].double())
        return (y.detach(),) + tuple(grads)
    n = case["n"]
    post, pre = st["post"].double(), st["pre"].double()
    gate = torch.ones(n, dtype=torch.float64, device="cuda") if st["gate"] is None else st["gate"].double()
    if op == "norm_forward":
        o = st["o"].double()
        r_post = (o.pow(2).sum(-1) / n + EPS).pow(-0.5)
        h = st["x"].double() + RESIDUAL * gate * torch.einsum("sbn,sb,n->sbn", o, r_post, post)
        # the second norm is that of the stored sum
        kept = h.to(st["x"].dtype).double()
        r_pre = (kept.pow(2).sum(-1) / n + EPS).pow(-0.5)
        return h, torch.einsum("sbn,sb,n->sbn", kept, r_pre, pre), r_post.flatten(), r_pre.flatten()
    s, b = case["s"], case["b"]
    h, o = _stored(st, "h"), _stored(st, "o")
    dy = st["grad_y"].flatten(0, 1).double()
    gate = gate.expand(s, b, n).reshape(-1, n)
    hat = {"h": torch.einsum("rn,r->rn", h, st["rms_pre"].double()), "o": torch.einsum("rn,r->rn", o, st["rms_post"].double())}

    def through(grad, xhat, r, gamma):  # gradient of xhat * gamma with respect to x, xhat = r x
        up = grad * gamma
        return r.double().unsqueeze(1) * (up - xhat * torch.einsum("rn,rn->r", up, xhat).unsqueeze(1) / n)

    dh = st["grad_h"].flatten(0, 1).double() + through(dy, hat["h"], st["rms_pre"], pre)
    dp = RESIDUAL * gate * dh
    out = [dh.reshape(s, b, n), through(dp, hat["o"], st["rms_post"], post).reshape(s, b, n),
           torch.einsum("rn,rn->n", dp, hat["o"]), torch.einsum("rn,rn->n", dy, hat["h"])]
    if st["gate"] is not None:
        dgate = (RESIDUAL * dh * hat["o"] * post).reshape(s, b, n)
        out.append({"channel": lambda v: v.sum((0, 1)), "sample": lambda v: v.sum(0), "token": lambda v: v}[case["gate"]](dgate))
    return tuple(out)
