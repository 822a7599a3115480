"""Plain CPU forms of the operators that keep activations in eight bits, in float64 where a value is computed and
in float32 where a float32 number is part of the definition (scales, quotients, stored rounding).  With each result
comes, where a kernel may round, how far a float32 evaluation may be from it.

Bounds.  U = 2^-24 is the largest relative error of one float32 rounding.  A kernel evaluates every expression
here in at most CHAIN roundings in a row, the sum over a row included (at most 16 terms per thread, then a tree), so a
term of size |t| is off by at most CHAIN * U * |t|, and a sum by that of the sum of its terms' sizes.  A sum over M
rows adds at most M more roundings.  Rounding the result to its type adds half a step, eps / 2 of its size."""

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


def pair_backward(dy, dh, o, h, post, pre, r_post, r_pre, gate, alpha):
    """All [M, n] in float64 (gate too, expanded; dh and gate may be None).  {name: (value, bound)}: dgate per element."""
    M = dy.shape[0]
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
