"""Operators that keep activations in eight bits (norm pair, SwiGLU with a checkpoint, int8 product) against their
plain forms in 64 bits.  Every tolerance is the oracle's bound plus half a step of the result's type; codes, scales
and integers are equal bit for bit."""

import pytest
import torch

from oracle import eight_bits as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
KINDS = [torch.int8, torch.float8_e4m3fn]
name = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def rand(seed, *shape, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def near(got, want, bound, what, extra=0.0):
    got, tol = got.detach().cpu(), bound + O.half_step(want, got.dtype) + extra
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / tol)[bad].max()):.3g} of the bound"


def same(got, want, what):
    a, b = got.detach().cpu().contiguous(), want.contiguous()
    assert a.shape == b.shape and a.dtype == b.dtype, (what, a.shape, a.dtype, b.shape, b.dtype)
    bad = a.view(torch.uint8) != b.view(torch.uint8)
    assert not bad.any(), f"{what}: {int(bad.sum())} bytes of {bad.numel()} differ"


def ok():
    from linghe_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.device_status(0) == 0


# ---- norm pair ---------------------------------------------------------------------------------
SHAPES = [((1,), 128), ((2, 3), 384), ((37,), 1408), ((101, 5), 256), ((999,), 2048), ((160, 4), 5120), ((77,), 8192)]
GATES = ["none", "channel", "sample", "token"]


def pair_inputs(lead, n, dtype, gate, seed=1):
    shape = (*lead, n)
    x, o = rand(seed, *shape).to(dtype), (rand(seed + 1, *shape) * torch.linspace(0.1, 4, lead[0]).reshape(-1, *[1] * len(lead))).to(dtype)
    post, pre = (1 + 0.3 * rand(seed + 2, n)).to(dtype), (1 + 0.3 * rand(seed + 3, n)).to(dtype)
    if len(lead) > 1 or gate != "sample":
        gshape = {"none": None, "channel": (n,), "sample": (lead[-1], n), "token": shape}[gate]
    else:
        gshape = shape
    g = None if gshape is None else torch.sigmoid(rand(seed + 4, *gshape)).to(dtype)
    rows = x.numel() // n
    full = None if g is None else g.expand(shape).reshape(rows, n)
    return x, o, post, pre, g, full


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("lead,n", SHAPES)
def test_pair_forward(lead, n, dtype, gate):
    from linghe_b200.utils.norm import rms_norm_pair_forward
    x, o, post, pre, g, full = pair_inputs(lead, n, dtype, gate)
    o.view(-1, n)[0] = 0                                  # a row of zeros: its norm is zero, h is x
    put = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    for kind in (None, *KINDS):
        h, y, rp, rh, saved = rms_norm_pair_forward(put(x), put(o), put(post), put(pre), gate=put(g), residual_scale=-0.6, eps=1e-5,
                                                    checkpoint=kind)
        assert h.shape == y.shape == x.shape and (saved is None) == (kind is None)
        want, bound, r = O.pair_forward(x.view(-1, n), o.view(-1, n), post, pre, full, -0.6, 1e-5)
        near(h.view(-1, n), want, bound, "h")
        near(rp, r, O.CHAIN * O.U * r, "rms_post")
        want, bound, r = O.norm_of(h.cpu().view(-1, n), pre, 1e-5)
        near(y.view(-1, n), want, bound, "y")
        near(rh, r, O.CHAIN * O.U * r, "rms_pre")
        same(h.view(-1, n)[:1], x.view(-1, n)[:1], "h of a zero row")
        if kind is not None:
            for (q, s), t in zip((saved[:2], saved[2:]), (o, h.cpu())):
                wq, ws = O.codes(t.view(-1, n), kind)
                same(q.view(-1, n), wq, "codes")
                same(s, ws, "scales")
    ok()


def pair_backward_case(lead, n, dtype, gate, kind, with_dh=True, alpha=0.8):
    from linghe_b200.utils.norm import rms_norm_pair_backward
    x, o, post, pre, g, full = pair_inputs(lead, n, dtype, gate, seed=11)
    rows = o.numel() // n
    h = x
    rp, rh = [((t.double().view(rows, n).square().mean(1) + 1e-6).rsqrt()).float() for t in (o, h)]
    dy, dh = rand(21, *x.shape, scale=0.1).to(dtype), rand(22, *x.shape, scale=0.1).to(dtype)
    osc = hsc = None
    ov, hv = o.double().view(rows, n), h.double().view(rows, n)
    ot, ht = o, h
    if kind is not None:
        (oq, osc), (hq, hsc) = O.codes(o.view(rows, n), kind), O.codes(h.view(rows, n), kind)
        ov, hv, ot, ht = O.values(oq, osc), O.values(hq, hsc), oq.view(o.shape), hq.view(h.shape)
    put = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    args = [put(t) for t in (dy, dh if with_dh else None, ot, ht, post, pre, rp, rh)]
    kw = dict(gate=put(g), residual_scale=alpha, o_scale=put(osc), h_scale=put(hsc))
    out = rms_norm_pair_backward(*args, **kw)
    want = O.pair_backward(dy.view(rows, n), dh.view(rows, n) if with_dh else None, ov, hv, post, pre, rp, rh, full, alpha)
    near(out[0].view(rows, n), *want["dx"], "dx")
    near(out[1].view(rows, n), *want["do"], "do")
    near(out[2], *want["dpost"], "dpost")
    near(out[3], *want["dpre"], "dpre")
    if g is None:
        assert out[4] is None
    else:
        G = g.numel() // n
        dg, bound = [v.view(rows // G, G, n).sum(0).view(g.shape) for v in want["dgate"]]
        near(out[4], dg, bound, "dgate")
    again = rms_norm_pair_backward(*args, **kw)
    for a, b in zip(out, again):
        if a is not None:
            same(a, b.cpu(), "the same call again")
    ok()


@pytest.mark.parametrize("kind", [None, *KINDS], ids=name)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("lead,n", SHAPES)
def test_pair_backward(lead, n, dtype, gate, kind):
    pair_backward_case(lead, n, dtype, gate, kind)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("kind", [None, torch.int8], ids=name)
def test_pair_backward_without_a_gradient_of_h(gate, kind):
    pair_backward_case((50, 3), 640, torch.bfloat16, gate, kind, with_dh=False)


# groups of rows that end inside a CTA's share, at its border, and span several CTAs
@pytest.mark.parametrize("lead", [(2, 700), (700, 2), (3, 333), (1200, 1), (1, 1200), (149, 7), (4, 296)])
def test_pair_backward_gate_groups(lead):
    pair_backward_case(lead, 2048, torch.float32, "sample", None)


# many rows to a CTA, so that every slot of its rings is used again several times
@pytest.mark.parametrize("kind", [None, *KINDS], ids=name)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=name)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("lead,n", [((12000, 5), 128), ((1400, 5), 1408), ((301, 5), 5120), ((300, 4), 8192)])
def test_pair_backward_long_walks(lead, n, dtype, gate, kind):
    pair_backward_case(lead, n, dtype, gate, kind)


# widths on both sides of where a thread has one vector of a row instead of two; the second ends inside a warp
@pytest.mark.parametrize("kind", [None, torch.int8], ids=name)
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("n", [4096, 4224, 4992, 5248])
def test_pair_backward_widths(n, dtype, gate, kind):
    pair_backward_case((180, 5), n, dtype, gate, kind)


def test_pair_no_rows():
    from linghe_b200.utils.norm import rms_norm_pair_backward, rms_norm_pair_forward
    x = torch.empty((0, 256), dtype=torch.bfloat16, device=DEV)
    w = torch.ones(256, dtype=torch.bfloat16, device=DEV)
    h, y, rp, rh, saved = rms_norm_pair_forward(x, x, w, w, gate=w, checkpoint=torch.int8)
    assert h.shape == y.shape == (0, 256) and rp.numel() == rh.numel() == 0 and saved[1].shape == (0, 2)
    out = rms_norm_pair_backward(x, x, x, x, w, w, rp, rh, gate=w)
    assert out[0].shape == (0, 256)
    for t in out[2:]:
        assert t.shape == (256,) and not t.any()
    ok()


def test_pair_values_that_are_not_finite():
    """A NaN or an infinity stays in its row, and a checkpoint of it gives nothing finite back in its block."""
    from linghe_b200.utils.norm import rms_norm_pair_forward
    n = 512
    x, o, post, pre, _, _ = pair_inputs((8,), n, torch.float32, "none")
    o[2, 300], o[5, 7], x[6, 1] = float("nan"), float("inf"), float("-inf")
    for kind in KINDS:
        h, y, rp, rh, saved = rms_norm_pair_forward(x.to(DEV), o.to(DEV), post.to(DEV), pre.to(DEV), checkpoint=kind)
        fine = torch.tensor([True, True, False, True, True, False, False, True])
        assert torch.isfinite(y.cpu()[fine]).all() and not torch.isfinite(y.cpu()[~fine]).all(1).any()
        assert torch.isnan(y.cpu()[2]).all()
        v = O.values(saved[0].cpu(), saved[1].cpu()).view(8, 4, 128)
        assert torch.isnan(v[2, 2]).all() and torch.isnan(v[5, 0]).all()
        assert torch.isfinite(v[2, [0, 1, 3]]).all() and torch.isfinite(v[5, 1:]).all() and torch.isfinite(v[fine]).all()
    ok()


# ---- SwiGLU with a checkpoint ------------------------------------------------------------------
@pytest.mark.parametrize("weight", [None, torch.float32, torch.bfloat16], ids=["none", "f32", "bf16"])
@pytest.mark.parametrize("kind", KINDS, ids=name)
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("M,n", [(1, 128), (3, 256), (77, 512), (130, 1408), (65, 4096), (9, 8192), (5, 14336), (5001, 1408), (4800, 384)])
def test_silu_checkpoint(M, n, dtype, kind, weight):
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    x, g = rand(1, M, 2 * n, scale=3).to(dtype), rand(2, M, n).to(dtype)
    x[0, :128] = 0                                        # a block of zeros
    w = None if weight is None else torch.rand(M, generator=torch.Generator().manual_seed(3)).to(weight)
    put = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    y, q, s = silu_and_checkpoint_forward(put(x), put(w), checkpoint=kind)
    near(y, *O.silu_forward(x, w), "y")
    wq, ws = O.codes(x, kind)
    same(q, wq, "codes")
    same(s, ws, "scales")
    dx, dw = silu_and_checkpoint_backward(put(g), q, s, put(w))
    want = O.silu_backward(g, O.values(wq, ws), w)
    near(dx, *want["dx"], "dx")
    assert (dw is None) == (w is None)
    if w is not None:
        near(dw, *want["dw"], "dw")
    ok()


@pytest.mark.parametrize("kind", KINDS, ids=name)
def test_silu_checkpoint_extremes(kind):
    """Large arguments (the sigmoid 0 or 1), codes at both ends, and a routing weight of zero."""
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    x = rand(5, 16, 512, scale=60)
    g, w = rand(6, 16, 256), torch.linspace(0, 1, 16)
    y, q, s = silu_and_checkpoint_forward(x.to(DEV), w.to(DEV), checkpoint=kind)
    near(y, *O.silu_forward(x, w), "y", extra=1e-30)
    dx, dw = silu_and_checkpoint_backward(g.to(DEV), q, s, w.to(DEV))
    want = O.silu_backward(g, O.values(*O.codes(x, kind)), w)
    near(dx, *want["dx"], "dx", extra=1e-30)
    near(dw, *want["dw"], "dw", extra=1e-30)
    assert not dx.cpu()[0].any()
    x[3, 5] = float("nan")
    x[4, 300] = float("inf")
    _, q, s = silu_and_checkpoint_forward(x.to(DEV), None, checkpoint=kind)
    v = O.values(q.cpu(), s.cpu())
    assert torch.isnan(v[3, :128]).all() and torch.isfinite(v[3, 128:]).all()
    assert torch.isnan(v[4, 256:384]).all() and torch.isfinite(v[4, :256]).all()
    ok()


def test_silu_checkpoint_takes_the_group_quantiser_s_codes():
    from linghe_b200.quant.group import triton_group_quant
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    x, g = rand(1, 64, 1024).to(torch.bfloat16).to(DEV), rand(2, 64, 512).to(torch.bfloat16).to(DEV)
    _, q, s = silu_and_checkpoint_forward(x, checkpoint=torch.float8_e4m3fn)
    q2, s2 = triton_group_quant(x)
    same(q2, q.cpu(), "codes")
    same(s2, s.cpu(), "scales")
    same(silu_and_checkpoint_backward(g, q2, s2)[0], silu_and_checkpoint_backward(g, q, s)[0].cpu(), "dx")


def test_silu_checkpoint_no_rows():
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    x, w = torch.empty((0, 512), device=DEV), torch.empty(0, device=DEV)
    y, q, s = silu_and_checkpoint_forward(x, w)
    dx, dw = silu_and_checkpoint_backward(y, q, s, w)
    assert y.shape == (0, 256) and dx.shape == (0, 512) and dw.shape == (0,)
    ok()


# ---- int8 ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("smooth", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("M,K", [(1, 16), (3, 208), (33, 512), (7, 1040), (130, 4096), (5, 8192), (3, 16400), (2, 40000)])
def test_token_quant(M, K, dtype, smooth):
    from linghe_b200.quant.token import token_quant_int8
    x = (rand(1, M, K) * torch.exp(rand(2, K))).to(dtype)
    x[M - 1, : K // 2] = 0
    if M > 2:
        x[1] = 0
    sm = torch.exp(rand(3, K)) if smooth else None
    if smooth:
        sm[0] = 0.0                                       # the floor of the divisor; its column is zero below
        x[:, 0] = 0
    q, s = token_quant_int8(x.to(DEV), None if sm is None else sm.to(DEV))
    wq, ws = O.token_quant(x, sm)
    same(q, wq, "codes")
    same(s, ws, "scales")
    ok()


def test_token_quant_ties_and_ends():
    from linghe_b200.quant.token import token_quant_int8
    x = torch.zeros(4, 272)
    x[0, :255] = torch.arange(-127, 128) / 2 * 2.0        # every code
    x[1, :254] = torch.arange(-127, 127) + 0.5            # quotients on a tie, amax 127 from the last element
    x[1, 254] = 127.0
    x[2, 0], x[2, 1] = 1e-38, -3e-39                      # below the floor of the scale
    x[3, 7], x[3, 8] = float("nan"), 1.0
    q, s = token_quant_int8(x.to(DEV))
    wq, ws = O.token_quant(x[:3])
    same(q[:3], wq, "codes")
    same(s[:3], ws, "scales")
    assert torch.isnan(s[3]).item()
    big = torch.full((1, 16), 3.0e38)
    big[0, 3] = float("-inf")
    assert torch.isnan(token_quant_int8(big.to(DEV))[1]).item()
    ok()


def gemm_inputs(M, N, K, seed=1):
    gen = torch.Generator().manual_seed(seed)
    a, b = [torch.randint(-128, 128, s, generator=gen, dtype=torch.int8) for s in ((M, K), (N, K))]
    return a, b, torch.rand(M, generator=gen) + 0.1, torch.rand(N, generator=gen) + 0.1


# one to sixteen tokens, then every kernel and its ragged edges: rows, columns, k within a stage and past it
GEMMS = [(1, 16, 16), (1, 4096, 4096), (3, 17, 80), (8, 1000, 2064), (9, 256, 512), (16, 33, 1040),
         (17, 40, 16), (17, 4096, 4096), (64, 512, 8192), (100, 1111, 528), (128, 64, 128), (129, 300, 2048), (200, 4096, 1024), (257, 63, 4096),
         (640, 4096, 272), (1000, 1111, 2064), (2048, 2500, 384), (1500, 4352, 144), (3000, 5000, 16),
         (4100, 8200, 144), (4100, 4099, 400), (2100, 16400, 528), (6000, 6016, 1040)]     # many tiles to a CTA


@pytest.mark.parametrize("out_dtype", TYPES, ids=name)
@pytest.mark.parametrize("M,N,K", GEMMS)
def test_int8_gemm(M, N, K, out_dtype):
    from linghe_b200.gemm.int8_gemm import int8_gemm
    a, b, sa, sb = gemm_inputs(M, N, K)
    if out_dtype == torch.float16:
        sa = sa * 2e-4                                     # stay below 65504
    c = int8_gemm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV), out_dtype=out_dtype)
    assert c.dtype == out_dtype
    da, db = a.to(DEV).double(), b.to(DEV).double()
    exact = (da @ db.t()).cpu() * sa.double()[:, None] * sb.double()
    near(c, exact, 3.01 * O.U * exact.abs(), "c")
    ok()


def test_int8_gemm_largest_sums():
    """k at its limit and every product 2^14: the sum is 128 short of 2^31 / 2^14 products."""
    from linghe_b200.gemm.int8_gemm import int8_gemm
    K = 131056
    one = torch.ones(256, device=DEV)
    for M in (2, 20, 200):
        a, b = torch.full((M, K), -128, dtype=torch.int8, device=DEV), torch.full((48, K), -128, dtype=torch.int8, device=DEV)
        c = int8_gemm(a, b, one[:M], one[:48], out_dtype=torch.float32)
        assert (c == float(K) * 16384.0).all()
    ok()


def test_int8_gemm_is_the_same_for_any_number_of_rows():
    from linghe_b200.gemm.int8_gemm import int8_gemm
    a, b, sa, sb = [t.to(DEV) for t in gemm_inputs(700, 2080, 1040)]
    whole = int8_gemm(a, b, sa, sb, out_dtype=torch.float32)
    for rows in (1, 5, 13, 16, 17, 130, 300):
        same(int8_gemm(a[:rows], b, sa[:rows], sb, out_dtype=torch.float32), whole[:rows].cpu(), f"{rows} rows")
    ok()


@pytest.mark.parametrize("smooth", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("lead,N,K", [((1,), 4096, 4096), ((2, 3), 272, 528), ((11,), 2048, 16400), ((3, 50), 1000, 1040), ((900,), 3000, 272)])
def test_int8_linear(lead, N, K, dtype, smooth):
    from linghe_b200.gemm.int8_gemm import int8_gemm, int8_linear
    from linghe_b200.quant.token import token_quant_int8
    x = rand(1, *lead, K).to(dtype).to(DEV)
    _, b, _, sb = gemm_inputs(1, N, K)
    b, sb = b.to(DEV), (sb / K).to(DEV)
    sm = torch.exp(rand(3, K)).to(DEV) if smooth else None
    got = int8_linear(x, b, sb, smooth_scale=sm)
    q, s = token_quant_int8(x, sm)
    same(got, int8_gemm(q, b, s, sb, out_dtype=dtype).cpu(), "the two calls in one")
    assert got.shape == (*lead, N) and got.dtype == dtype
    wq, ws = O.token_quant(x.cpu().view(-1, K), None if sm is None else sm.cpu())
    exact = (wq.to(DEV).double() @ b.double().t()).cpu() * ws.double()[:, None] * sb.cpu().double()
    near(got.view(-1, N), exact, 3.01 * O.U * exact.abs(), "c")
    ok()


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("N,K,smooth", [(1, 16, False), (33, 80, True), (4096, 4096, False), (4736, 16384, True), (4752, 1024, False), (512, 16400, True), (1111, 2064, False)])
def test_int8_linear_of_one_token(N, K, smooth, dtype):
    """One kernel up to two CTAs of 16 channels per SM and 16384 of k, two beyond: the bits of the two calls, also for a token that is
    zero and for one with a NaN or an infinity (every result is NaN or infinite then)."""
    from linghe_b200.gemm.int8_gemm import int8_gemm, int8_linear
    from linghe_b200.quant.token import token_quant_int8
    _, b, _, sb = gemm_inputs(1, N, K)
    b, sb = b.to(DEV), (sb / K).to(DEV)
    sm = torch.exp(rand(3, K)).to(DEV) if smooth else None
    x = rand(1, 1, K).to(dtype).to(DEV)
    for fill in (None, 0.0, float("nan"), float("-inf")):
        if fill == 0.0:
            x.zero_()
        elif fill is not None:
            x[0, K // 2] = fill
        got = int8_linear(x, b, sb, smooth_scale=sm)
        q, s = token_quant_int8(x, sm)
        if fill is None or fill == 0.0:
            same(got, int8_gemm(q, b, s, sb, out_dtype=dtype).cpu(), "the two calls in one")
        else:
            assert torch.isnan(s).all() and not torch.isfinite(got).any()
    ok()


def test_int8_no_rows():
    from linghe_b200.gemm.int8_gemm import int8_gemm, int8_linear
    from linghe_b200.quant.token import token_quant_int8
    b, sb = torch.ones((32, 64), dtype=torch.int8, device=DEV), torch.ones(32, device=DEV)
    x = torch.empty((0, 64), device=DEV)
    q, s = token_quant_int8(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    assert int8_gemm(q, b, s, sb).shape == (0, 32) and int8_linear(x, b, sb).shape == (0, 32)
    ok()
