"""Plain CPU forms of the operators that keep activations in eight bits, in float64 where a value is computed and
in float32 where a float32 number is part of the definition (scales, quotients, stored rounding).  With each result
comes, where a kernel may round, how far a float32 evaluation may be from it.

Bounds.  U = 2^-24 is the largest relative error of one float32 rounding.  A kernel evaluates every expression
here in at most CHAIN roundings in a row, the sum over a row included (at most 16 terms per thread, then a tree), so a
term of size |t| is off by at most CHAIN * U * |t|, and a sum by that of the sum of its terms' sizes.  A sum over M
rows adds at most M more roundings (`depth` where the number of additions in a row is known).  Rounding the result to its
type adds half a step, eps / 2 of its size.

A bound that grows with the number of terms cannot tell a lost row from rounding where the terms have both signs.
`whole_rows` makes inputs for which every sum over rows is exact in float32 and every row adds to every column with the same
sign: there a lost, doubled or wrongly scaled row is a wrong number."""

import math

import torch

U = 2.0 ** -24
CHAIN = 64
FLOOR = 1e-30


def half_step(ref, dtype):
    """Half a step of `dtype` at each value of `ref`, and half the smallest step below the normal numbers."""
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps / 2) + fi.tiny * fi.eps / 2


def codes(x, kind, block=128):
    """(codes, float32 scales [rows, n / block]) of the rows of x; kind torch.int8 or torch.float8_e4m3fn."""
    v = x.float().reshape(x.shape[0], -1, block)
    top = torch.tensor(127.0 if kind == torch.int8 else 448.0)
    scale = (v.abs().amax(2) / top).clamp_min(FLOOR)
    q = v / scale[:, :, None]
    if kind == torch.int8:
        q = q.round()
    return q.to(kind).reshape(x.shape), scale


def values(q, scale):
    rows = q.shape[0]
    return (q.double().reshape(rows, scale.shape[1], -1) * scale.double()[:, :, None]).reshape(rows, -1)


def token_quant(x, smooth=None):
    v = x.float()
    if smooth is not None:
        v = v / smooth.clamp_min(FLOOR)
    q, s = codes(v, torch.int8, x.shape[1])
    return q, s[:, 0]


def int8_gemm(a, b, a_s, b_s):
    """(c, bound before the result is rounded to its type): an exact integer, its conversion and two products."""
    c = (a.double() @ b.double().t()) * a_s.double()[:, None] * b_s.double()
    return c, 3.01 * U * c.abs()


def pair_forward(x, o, post, pre, gate, alpha, eps):
    """rows [M, n], gate [M, n] or None.  (h, bound, r_post): the second norm is that of the stored h (norm_of)."""
    o, x = o.double(), x.double()
    r = (o.square().mean(1) + eps).rsqrt()
    p = alpha * o * r[:, None] * post.double()
    if gate is not None:
        p = p * gate.double()
    return x + p, CHAIN * U * (p.abs() + x.abs()), r


def norm_of(h, weight, eps):
    h = h.double()
    r = (h.square().mean(1) + eps).rsqrt()
    y = h * r[:, None] * weight.double()
    return y, CHAIN * U * y.abs(), r


def row_depth(M, sms=148):
    """Additions in a row behind a sum over M rows in lh_rmsnorm_pair_bwd: at most ceil(M / sms) rows of a CTA (there are at least
    as many CTAs as SMs, or one per row) and as many groups of gate rows, then up to 16 CTAs an SM in 32 strands, then the strands."""
    return 2 * math.ceil(M / sms) + math.ceil(16 * sms / 32) + 32


def pair_backward(dy, dh, o, h, post, pre, r_post, r_pre, gate, alpha, depth=None):
    """All [M, n] in float64 (gate too, expanded; dh and gate may be None).  {name: (value, bound)}: dgate per element.
    depth: additions in a row behind a sum over rows, M if not given."""
    M = dy.shape[0] if depth is None else depth
    dy, post, pre = dy.double(), post.double(), pre.double()
    r_post, r_pre = r_post.double()[:, None], r_pre.double()[:, None]
    gate = torch.ones_like(dy) if gate is None else gate.double()
    dh = torch.zeros_like(dy) if dh is None else dh.double()
    hn, on, t = h * r_pre, o * r_post, dy * pre
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    dx = dh + r_pre * (t - hn * mean(t * hn))
    b_dx = CHAIN * U * (dh.abs() + r_pre * (t.abs() + hn.abs() * mean((t * hn).abs())))
    dp, b_dp = alpha * gate * dx, abs(alpha) * gate.abs() * b_dx
    u, b_u = dp * post, b_dp * post.abs()
    size_u = b_u / (CHAIN * U)
    do = r_post * (u - on * mean(u * on))
    b_do = 2 * CHAIN * U * r_post * (size_u + on.abs() * mean(size_u * on.abs()))
    rows = (CHAIN + M) * U
    size_dp = b_dp / (CHAIN * U)
    size_dx = b_dx / (CHAIN * U)
    dgate = alpha * dx * on * post
    return {
        "dx": (dx, b_dx), "do": (do, b_do),
        "dpost": ((dp * on).sum(0), 2 * rows * (size_dp * on.abs()).sum(0)),
        "dpre": ((dy * hn).sum(0), rows * (dy * hn).abs().sum(0)),
        "dgate": (dgate, 2 * rows * abs(alpha) * (size_dx * on * post).abs()),
    }


def whole_rows(lead, n, gate, with_dh=True, seed=1, device="cpu"):
    """Inputs of the norm pair's gradient and its results, all float64: (inputs, dx and the sums over rows, the terms of the sums).

    o and h are 1 or 2 in neighbouring columns alike, times a power of two per row (1/rms) and, as codes, per block of 128;
    dy is +1, -1 in neighbouring columns and pre the same in both, so that the row's sum of dy * pre * h * r_pre is zero and
    dx = dh + r_pre * dy * pre a whole number of 1 to 10 (without dh: one of -4 to 4, no zero, of one sign in a column).  Terms are multiples of 1/4: dx * on <= 20, with the gate and
    alpha = 1/2 again at most 20; 60000 rows sum to 1.2e6, 4.8e6 quarters, below 2^24.  dy, weights, gates, o, h and the codes
    (1 to 8) are exact in every type."""
    gen = torch.Generator(device=device).manual_seed(seed)
    rows = math.prod(lead)

    def pick(values, *shape):
        return torch.tensor(values, dtype=torch.float64, device=device)[torch.randint(len(values), shape, generator=gen, device=device)]

    pairs = lambda t: t.repeat_interleave(2, dim=-1)  # noqa: E731
    sign = torch.tensor([1.0, -1.0], dtype=torch.float64, device=device).repeat(n // 2)
    d = {"o": pairs(pick([1, 2], rows, n // 2)), "h": pairs(pick([1, 2], rows, n // 2)), "dy": sign.expand(rows, n),
         "dh": pick([5, 6], rows, n) if with_dh else None, "post": pick([1, 2], n), "pre": pairs(pick([1, 2], n // 2)),
         "r_post": pick([0.5, 1], rows), "r_pre": pick([1, 2], rows), "alpha": 0.5,
         "o_scale": pick([0.25, 0.5, 1], rows, n // 128), "h_scale": pick([0.25, 0.5, 1], rows, n // 128)}
    shape = {"none": None, "channel": (n,), "sample": (lead[-1], n), "token": (*lead, n)}[gate]
    d["gate"] = None if shape is None else pick([1, 2], *shape)
    full = torch.ones((), dtype=torch.float64, device=device) if shape is None else d["gate"].expand(*lead, n).reshape(rows, n)
    on, hn = d["o"] * d["r_post"][:, None], d["h"] * d["r_pre"][:, None]
    dx = d["r_pre"][:, None] * d["dy"] * d["pre"] + (d["dh"] if with_dh else 0)
    terms = {"dpre": d["dy"] * hn, "dpost": d["alpha"] * full * dx * on, "dgate": d["alpha"] * dx * on * d["post"]}
    sums = {"dx": dx, "dpre": terms["dpre"].sum(0), "dpost": terms["dpost"].sum(0)}
    if shape is not None:
        G = d["gate"].numel() // n
        sums["dgate"] = terms["dgate"].view(rows // G, G, n).sum(0).view(shape)
    return d, sums, terms


def silu_terms(x1):
    """sigmoid, and how far a float32 one from a base-2 exponential may be, relative: the exponent |x1| * log2(e) is
    rounded, which moves the result by up to |x1| * U, and a handful of other roundings and 2-ulp approximations."""
    return torch.sigmoid(x1), (x1.abs() + CHAIN) * U


def silu_forward(x, w):
    n = x.shape[1] // 2
    x1, x2 = x.double()[:, :n], x.double()[:, n:]
    s, rel = silu_terms(x1)
    y = x1 * s * x2
    if w is not None:
        y = y * w.double()[:, None]
    return y, rel * y.abs()


def silu_backward(g, x, w):
    """x: float64 values of the checkpoint.  {name: (value, bound)}"""
    n = x.shape[1] // 2
    g, x1, x2 = g.double(), x[:, :n], x[:, n:]
    s, rel = silu_terms(x1)
    dw = g * x1 * s * x2
    gw = g if w is None else g * w.double()[:, None]
    d1, d2 = gw * x2 * s * (1 + x1 * (1 - s)), gw * x1 * s
    b1 = 2 * rel * (gw * x2).abs() * (s + (x1 * s).abs())
    return {"dx": (torch.cat([d1, d2], 1), torch.cat([b1, rel * d2.abs()], 1)),
            "dw": (dw.sum(1), (rel * dw.abs()).sum(1) + CHAIN * U * dw.abs().sum(1))}
