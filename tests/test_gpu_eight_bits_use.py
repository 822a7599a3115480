"""The 8-bit operators as a program uses them: refusals, autograd, a block of them together, streams, captured graphs, offsets past
32 bits, alignment, and the two ways of argument handling."""

import pytest
import torch

from oracle import eight_bits as O
from tests.test_gpu_eight_bits import DEV, KINDS, TYPES, gemm_inputs, name, near, ok, pair_inputs, rand, same

pytestmark = pytest.mark.gpu


def calls():
    """(name, function of a dict of tensors) for every operator, and the tensors."""
    from linghe_b200.gemm.int8_gemm import int8_gemm, int8_linear
    from linghe_b200.quant.token import token_quant_int8
    from linghe_b200.utils.norm import rms_norm_pair_backward, rms_norm_pair_forward
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    x, o, post, pre, gate, _ = pair_inputs((12, 5), 512, torch.bfloat16, "sample")
    a, b, sa, sb = gemm_inputs(200, 512, 512)
    t = dict(x=x, o=o, post=post, pre=pre, gate=gate, dy=rand(5, 12, 5, 512).bfloat16(), dh=rand(6, 12, 5, 512).bfloat16(),
             u=rand(7, 60, 1024).bfloat16(), g=rand(8, 60, 512).bfloat16(), w=torch.rand(60), a=a, b=b, sa=sa, sb=sb / 512, sm=torch.rand(512) + 0.5)
    t = {k: v.to(DEV) for k, v in t.items()}

    def backward(d):
        h, y, rp, rh, kept = rms_norm_pair_forward(d["x"], d["o"], d["post"], d["pre"], d["gate"], 0.7, 1e-6, torch.int8)
        return (h, y, rp, rh, *kept) + rms_norm_pair_backward(d["dy"], d["dh"], kept[0], kept[2], d["post"], d["pre"], rp, rh, d["gate"], 0.7, kept[1], kept[3])

    def silu(d):
        y, q, s = silu_and_checkpoint_forward(d["u"], d["w"], torch.float8_e4m3fn)
        return (y, q, s) + silu_and_checkpoint_backward(d["g"], q, s, d["w"])

    return {"pair": backward, "silu": silu, "token": lambda d: token_quant_int8(d["x"], d["sm"]),
            "gemm": lambda d: (int8_gemm(d["a"], d["b"], d["sa"], d["sb"], out_dtype=torch.float32),),
            "rows": lambda d: (int8_gemm(d["a"][:5], d["b"], d["sa"][:5], d["sb"], out_dtype=torch.float32),),
            "linear": lambda d: (int8_linear(d["x"], d["b"], d["sb"], smooth_scale=d["sm"]),),
            "linear few": lambda d: (int8_linear(d["x"][0], d["b"], d["sb"]),)}, t


@pytest.mark.parametrize("which", ["pair", "silu", "token", "gemm", "rows", "linear", "linear few"])
def test_without_the_host_module(which, monkeypatch):
    from linghe_b200 import _lib
    fns, t = calls()
    first = fns[which](t)
    assert _lib.host() is not None
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(_lib, "_fn_cache", {})
    second = fns[which](t)
    assert len(first) == len(second)
    for i, (p, q) in enumerate(zip(first, second)):
        same(q, p.cpu(), f"{which} {i}")
    ok()


@pytest.mark.parametrize("which", ["pair", "silu", "token", "gemm", "rows", "linear", "linear few"])
def test_on_another_stream_and_replayed(which):
    """The same bits on a side stream, and from a captured graph whose inputs change between its replays."""
    fns, t = calls()
    want = [v.cpu() for v in fns[which](t)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fns[which](t)
    side.synchronize()
    for p, q in zip(got, want):
        same(p, q, "side stream")
    held = {k: v.clone() for k, v in t.items()}
    with torch.cuda.stream(side):
        fns[which](held)
        side.synchronize()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = fns[which](held)
            graphs.append((g, out))
    other = {k: (v.flip(0).contiguous() if k not in ("sb", "w") else v) for k, v in t.items()}
    expect = [v.cpu() for v in fns[which](other)]
    for source, result in ((t, want), (other, expect)):
        for k in held:
            held[k].copy_(source[k])
        torch.cuda.synchronize()
        for g, _ in graphs:          # both graphs at once: neither uses the other's scratch
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for p, q in zip(out, result):
                same(p, q, "replayed")
    ok()


@pytest.mark.parametrize("with_host_module", [True, False])
def test_refusals(with_host_module, monkeypatch):
    from linghe_b200 import _lib
    from linghe_b200.gemm.int8_gemm import int8_gemm, int8_linear
    from linghe_b200.quant.token import token_quant_int8
    from linghe_b200.utils.norm import rms_norm_pair_backward, rms_norm_pair_forward
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    if not with_host_module:
        monkeypatch.setattr(_lib, "_host", None)
        monkeypatch.setattr(_lib, "_fn_cache", {})
    d = dict(dtype=torch.bfloat16, device=DEV)
    x, w, r = torch.ones((4, 3, 256), **d), torch.ones(256, **d), torch.ones(12, device=DEV)
    q, s = torch.ones((4, 3, 256), dtype=torch.int8, device=DEV), torch.ones((12, 2), device=DEV)
    u, f = torch.ones((4, 512), **d), torch.ones(4, device=DEV)
    uq, us = torch.ones((4, 512), dtype=torch.int8, device=DEV), torch.ones((4, 4), device=DEV)
    a, b, one = torch.ones((4, 64), dtype=torch.int8, device=DEV), torch.ones((32, 64), dtype=torch.int8, device=DEV), torch.ones(32, device=DEV)
    bad = {
        "another type": lambda: rms_norm_pair_forward(x, x.float(), w, w),
        "weight type": lambda: rms_norm_pair_forward(x, x, w.float(), w),
        "weight length": lambda: rms_norm_pair_forward(x, x, w[:128].contiguous(), w),
        "width": lambda: rms_norm_pair_forward(x[..., :192].contiguous(), x[..., :192].contiguous(), w[:192].contiguous(), w[:192].contiguous()),
        "strides": lambda: rms_norm_pair_forward(x.transpose(0, 1), x.transpose(0, 1), w, w),
        "gate of the middle": lambda: rms_norm_pair_forward(x, x, w, w, gate=torch.ones((4, 1, 256), **d)),
        "gate of another batch": lambda: rms_norm_pair_forward(x, x, w, w, gate=torch.ones((2, 256), **d)),
        "gate of scalars": lambda: rms_norm_pair_forward(x, x, w, w, gate=torch.ones((4, 3, 1), **d)),
        "checkpoint type": lambda: rms_norm_pair_forward(x, x, w, w, checkpoint=torch.uint8),
        "one scale": lambda: rms_norm_pair_backward(x, None, q, q, w, w, r, r, o_scale=s),
        "scales of values": lambda: rms_norm_pair_backward(x, None, x, x, w, w, r, r, o_scale=s, h_scale=s),
        "codes without scales": lambda: rms_norm_pair_backward(x, None, q, q, w, w, r, r),
        "scale shape": lambda: rms_norm_pair_backward(x, None, q, q, w, w, r, r, o_scale=s.t().contiguous(), h_scale=s.t().contiguous()),
        "rms length": lambda: rms_norm_pair_backward(x, None, x, x, w, w, r[:4].contiguous(), r),
        "grad type": lambda: rms_norm_pair_backward(x, x.float(), x, x, w, w, r, r),
        "no checkpoint": lambda: silu_and_checkpoint_forward(u, checkpoint=None),
        "silu width": lambda: silu_and_checkpoint_forward(u[:, :384].contiguous()),
        "weight rows": lambda: silu_and_checkpoint_forward(u, f[:3].contiguous()),
        "weight half": lambda: silu_and_checkpoint_forward(u, f.half()),
        "g rows": lambda: silu_and_checkpoint_backward(u[:2, :256].contiguous(), uq, us),
        "scales layout": lambda: silu_and_checkpoint_backward(u[:, :256].contiguous(), uq, us[:, :2].contiguous()),
        "K": lambda: token_quant_int8(torch.ones((4, 24), **d)),
        "smooth type": lambda: token_quant_int8(u, torch.ones(512, **d)),
        "smooth length": lambda: token_quant_int8(u, torch.ones(256, device=DEV)),
        "out type": lambda: token_quant_int8(u, out=torch.empty((4, 512), dtype=torch.uint8, device=DEV)),
        "columns": lambda: int8_gemm(a, b[:, :32].contiguous(), f, one),
        "a scales": lambda: int8_gemm(a, b, one, one),
        "b scales": lambda: int8_gemm(a, b, f, f),
        "floats": lambda: int8_gemm(a.float(), b, f, one),
        "out dtype": lambda: int8_gemm(a, b, f, one, out_dtype=torch.float64),
        "b strides": lambda: int8_gemm(a, b.t().contiguous().t(), f, one),
        "linear columns": lambda: int8_linear(u, b, one),
        "linear ints": lambda: int8_linear(a, b, one),
        "linear host": lambda: int8_linear(u[:, :64].contiguous(), b.cpu(), one),
    }
    for what, call in bad.items():
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"accepted: {what}")
    ok()


@pytest.mark.parametrize("dtype", TYPES, ids=name)
def test_pointers_aligned_to_16_bytes_only(dtype):
    from linghe_b200.gemm.int8_gemm import int8_linear
    from linghe_b200.quant.token import token_quant_int8
    from linghe_b200.utils.norm import rms_norm_pair_forward
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward

    def off(t):      # the same values 16 bytes past an allocation's start
        step = 16 // t.element_size()
        buf = torch.empty(t.numel() + step, dtype=t.dtype, device=DEV)
        buf[step:] = t.reshape(-1).to(DEV)
        v = buf[step:].view(t.shape)
        assert v.data_ptr() % 32 == 16
        return v

    x, o, post, pre, gate, _ = [t.to(DEV) if t is not None else None for t in pair_inputs((9, 3), 640, dtype, "sample")]
    for kind in (None, torch.int8):
        p = rms_norm_pair_forward(x, o, post, pre, gate, checkpoint=kind)
        q = rms_norm_pair_forward(off(x), off(o), off(post), off(pre), off(gate), checkpoint=kind)
        for u, v in zip(p[:4] + (p[4] or ()), q[:4] + (q[4] or ())):
            same(v, u.cpu(), "pair")
    u, g = rand(3, 33, 768).to(dtype).to(DEV), rand(4, 33, 384).to(dtype).to(DEV)
    p = silu_and_checkpoint_forward(u)
    for a, b in zip(silu_and_checkpoint_forward(off(u)), p):
        same(a, b.cpu(), "silu")
    same(silu_and_checkpoint_backward(off(g), off(p[1]), off(p[2]))[0], silu_and_checkpoint_backward(g, p[1], p[2])[0].cpu(), "silu gradient")
    for a, b in zip(token_quant_int8(off(u)), token_quant_int8(u)):
        same(a, b.cpu(), "token")
    for M in (4, 33):
        _, w, _, ws = gemm_inputs(1, 100, 768)
        same(int8_linear(off(u[:M]), off(w), off(ws)), int8_linear(u[:M].contiguous(), w.to(DEV), ws.to(DEV)).cpu(), "linear")
    ok()


# ---- autograd -----------------------------------------------------------------------------------
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
def test_pair_autograd_against_differences(gate):
    """The gradient along a random direction against central differences of the definition in 64 bits (step 1e-4: the truncation
    is below 1e-7 of the terms).  Allowed: the oracle's bounds along the direction, and 1e-6 of the terms for h, which is a rounded
    float32 number in the kernel (2^-24, in at most four factors of a term) and not in the differences."""
    from linghe_b200.facade.norm import rms_norm_pair
    lead, n, alpha, eps = (7, 3), 256, 0.6, 1e-5
    x, o, post, pre, g, full = pair_inputs(lead, n, torch.float32, gate)
    dh, dy = rand(31, *x.shape), rand(32, *x.shape)
    leaves = [t.to(DEV).requires_grad_() for t in (x, o, post, pre) + (() if g is None else (g,))]
    h, y = rms_norm_pair(*leaves[:4], gate=None if g is None else leaves[4], residual_scale=alpha, eps=eps)
    grads = torch.autograd.grad([h, y], leaves, [dh.to(DEV), dy.to(DEV)])
    dirs = [rand(40 + i, *t.shape).double() for i, t in enumerate(leaves)]

    def loss(step):
        v = [t.detach().cpu().double() + step * d for t, d in zip(leaves, dirs)]
        r = (v[1].square().mean(-1, keepdim=True) + eps).rsqrt()
        hh = v[0] + alpha * (v[4] if g is not None else 1.0) * v[1] * r * v[2]
        yy = hh * (hh.square().mean(-1, keepdim=True) + eps).rsqrt() * v[3]
        return (hh * dh.double()).sum() + (yy * dy.double()).sum()

    numeric = (loss(1e-4) - loss(-1e-4)) / 2e-4
    analytic = sum((a.cpu().double() * d).sum() for a, d in zip(grads, dirs))
    rows = x.numel() // n
    rp = (o.double().view(rows, n).square().mean(1) + eps).rsqrt()
    hv = h.detach().cpu().view(rows, n)
    rh = (hv.double().square().mean(1) + eps).rsqrt()
    want = O.pair_backward(dy.view(rows, n), dh.view(rows, n), o.double().view(rows, n), hv.double(), post, pre, rp, rh, full, alpha)
    allowed = 0.0
    for key, d in zip(("dx", "do", "dpost", "dpre"), dirs):
        value, bound = want[key]
        d = d.view(value.shape).abs()
        allowed += ((bound + 1e-6 * value.abs()) * d).sum()
    if g is not None:
        value, bound = [t.view(x.shape) for t in want["dgate"]]
        allowed += ((bound + 1e-6 * value.abs()) * dirs[4].expand(x.shape).abs()).sum()
    assert abs(numeric - analytic) <= allowed + 1e-7 * abs(numeric), (float(numeric), float(analytic), float(allowed))
    ok()


def test_pair_autograd_edges():
    """Only one of the two results used, a gradient that is expanded, weights in bf16, a checkpoint."""
    from linghe_b200.facade.norm import rms_norm_pair
    x, o, post, pre, g, _ = [t.to(DEV).requires_grad_() if t is not None else None for t in pair_inputs((6, 4), 384, torch.bfloat16, "channel")]
    for kind in (None, *KINDS):
        for use in ("h", "y", "both"):
            h, y = rms_norm_pair(x, o, post, pre, gate=g, residual_scale=0.5, checkpoint=kind)
            out = {"h": h.sum(), "y": y.float().square().sum(), "both": (h + y).sum()}[use]
            grads = torch.autograd.grad(out, [x, o, post, pre, g])
            for a, b in zip(grads, (x, o, post, pre, g)):
                assert a.shape == b.shape and a.dtype == b.dtype and torch.isfinite(a).all()
            if use == "h":
                assert not grads[3].any() and (grads[0] == 1).all()
    x2 = x.detach()      # nothing but the weights is trained
    h, y = rms_norm_pair(x2, x2, post, pre)
    torch.autograd.grad(y.sum(), [post, pre])
    ok()


@pytest.mark.parametrize("kind", KINDS, ids=name)
def test_checkpointed_silu_autograd(kind):
    """Against differences of the 64-bit definition at the checkpoint's values, along a random direction (step 1e-4)."""
    from linghe_b200.facade.silu import checkpointed_silu
    x, w, g = rand(1, 5, 3, 512), torch.rand(5, 3, generator=torch.Generator().manual_seed(2)), rand(3, 5, 3, 256)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = checkpointed_silu(xd, wd, kind)
    assert y.shape == (5, 3, 256)
    dx, dw = torch.autograd.grad(y, [xd, wd], g.to(DEV))
    v = O.values(*O.codes(x.view(15, 512), kind))
    d, dd = rand(4, 15, 512).double(), rand(5, 15).double()

    def loss(step):
        a = v + step * d
        return (torch.nn.functional.silu(a[:, :256]) * a[:, 256:] * (w.view(15).double() + step * dd)[:, None] * g.view(15, 256).double()).sum()

    numeric = (loss(1e-4) - loss(-1e-4)) / 2e-4
    analytic = (dx.cpu().double().view(15, 512) * d).sum() + (dw.cpu().double().view(15) * dd).sum()
    want = O.silu_backward(g.view(15, 256), v, w.view(15))
    allowed = sum(((want[k][1] + O.half_step(want[k][0], torch.float32)) * e.abs()).sum() for k, e in (("dx", d), ("dw", dd)))
    assert abs(numeric - analytic) <= allowed + 1e-7 * abs(numeric), (float(numeric), float(analytic), float(allowed))
    ok()


def test_backward_captured_while_an_eager_graph_of_the_leaves_lives():
    from linghe_b200.facade.norm import rms_norm_pair
    from linghe_b200.facade.silu import checkpointed_silu
    x, o, post, pre, g, _ = [t.to(DEV).requires_grad_() if t is not None else None for t in pair_inputs((8, 2), 512, torch.bfloat16, "sample")]
    leaves = [x, o, post, pre, g]

    def step():
        h, y = rms_norm_pair(x, o, post, pre, gate=g, checkpoint=torch.int8)
        out = checkpointed_silu(y.view(16, 512))
        return torch.autograd.grad([out, h], leaves, [torch.ones_like(out), torch.ones_like(h)])

    # torch ties a leaf's gradient to the stream of the first graph that holds it, here the one that is captured later
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager_h, eager_y = rms_norm_pair(x, o, post, pre, gate=g)      # stays alive over the capture
        want = [t.cpu() for t in step()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        same(a, b, "captured")
    with torch.cuda.stream(side):
        torch.autograd.grad([eager_h.sum(), eager_y.sum()], leaves)
    ok()


def test_a_block_of_them_together():
    """Norm pair, int8 up projection, SwiGLU with a checkpoint, int8 down projection, norm pair: every step against the 64-bit form of
    the step on the tensors that came before it."""
    from linghe_b200.facade.norm import rms_norm_pair
    from linghe_b200.facade.silu import checkpointed_silu
    from linghe_b200.gemm.int8_gemm import int8_linear
    from linghe_b200.quant.token import token_quant_int8
    S, B, n, f = 33, 2, 512, 768
    x, o, post, pre, gate, full = pair_inputs((S, B), n, torch.bfloat16, "sample")
    up, down = rand(1, 2 * f, n).bfloat16() / n ** 0.5, rand(2, n, f).bfloat16() / f ** 0.5
    (uq, us), (dq, ds) = [token_quant_int8(w.to(DEV)) for w in (up, down)]
    xd, od, postd, pred, gated = [t.to(DEV).requires_grad_() for t in (x, o, post, pre, gate)]
    h, y = rms_norm_pair(xd, od, postd, pred, gate=gated, checkpoint=torch.float8_e4m3fn)
    with torch.no_grad():
        u = int8_linear(y, uq, us)
    u = u.requires_grad_()
    act = checkpointed_silu(u)
    with torch.no_grad():
        out = int8_linear(act, dq, ds)
    out = out.requires_grad_()
    h2, y2 = rms_norm_pair(h, out, postd, pred, gate=gated, checkpoint=torch.float8_e4m3fn)

    def linear(v, w, ws):
        q, s = O.token_quant(v.detach().cpu().view(S * B, -1))
        return O.int8_gemm(q, w.cpu(), s, ws.cpu())

    near(u.view(S * B, -1), *linear(y, uq, us), "up")
    near(act.view(S * B, -1), *O.silu_forward(u.detach().cpu().view(S * B, -1), None), "act")
    near(out.view(S * B, -1), *linear(act, dq, ds), "down")
    hv, bound, _ = O.pair_forward(h.detach().cpu().view(S * B, n), out.detach().cpu().view(S * B, n), post, pre, full, 1.0, 1e-6)
    near(h2.view(S * B, n), hv, bound, "h2")
    grads = torch.autograd.grad([h2, y2], [h, out, postd, pred, gated], [torch.ones_like(h2), torch.ones_like(y2)], retain_graph=True)
    du = torch.autograd.grad(act, u, torch.ones_like(act))[0]
    dx = torch.autograd.grad([h, y], [xd, od], [grads[0], torch.ones_like(y)])
    for t in (*grads, du, *dx):
        assert torch.isfinite(t).all()
    ok()


# ---- offsets past 32 bits -------------------------------------------------------------------------
def test_pair_past_32_bits():
    from linghe_b200.utils.norm import rms_norm_pair_backward, rms_norm_pair_forward
    n, M, last = 8192, 270_000, 4          # 2.2e9 elements
    make = lambda seed: rand(seed, last, n).bfloat16()  # noqa: E731
    post, pre = (1 + 0.1 * rand(1, n)).bfloat16(), (1 + 0.1 * rand(2, n)).bfloat16()
    tails = [make(s) for s in (3, 4, 5, 6)]
    x, o, dy, dh = [torch.zeros((M, n), dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    for t, v in zip((x, o, dy, dh), tails):
        t[-last:] = v.to(DEV)
    h, y, rp, rh, saved = rms_norm_pair_forward(x, o, post.to(DEV), pre.to(DEV), checkpoint=torch.int8)
    want, bound, _ = O.pair_forward(tails[0], tails[1], post, pre, None, 1.0, 1e-6)
    near(h[-last:], want, bound, "h")
    wq, ws = O.codes(tails[1], torch.int8)
    same(saved[0][-last:], wq, "codes")
    same(saved[1][-last:], ws, "scales")
    assert not h[:100].any() and not y[:100].any()
    dx, do, dpost, dpre, _ = rms_norm_pair_backward(dy, dh, o, h, post.to(DEV), pre.to(DEV), rp, rh)
    want = O.pair_backward(tails[2], tails[3], tails[1].double(), h[-last:].cpu().double(), post, pre, rp[-last:].cpu(), rh[-last:].cpu(), None, 1.0)
    near(dx[-last:], *want["dx"], "dx")
    near(do[-last:], *want["do"], "do")
    near(dpost, *want["dpost"], "dpost")       # the other rows are zero and add nothing
    near(dpre, *want["dpre"], "dpre")
    ok()


def test_silu_past_32_bits():
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    n, M, last = 8192, 140_000, 3
    tail, gt = rand(1, last, 2 * n).bfloat16(), rand(2, last, n).bfloat16()
    x, g = torch.zeros((M, 2 * n), dtype=torch.bfloat16, device=DEV), torch.zeros((M, n), dtype=torch.bfloat16, device=DEV)
    x[-last:], g[-last:] = tail.to(DEV), gt.to(DEV)
    y, q, s = silu_and_checkpoint_forward(x)
    near(y[-last:], *O.silu_forward(tail, None), "y")
    wq, ws = O.codes(tail, torch.int8)
    same(q[-last:], wq, "codes")
    same(s[-last:], ws, "scales")
    dx, _ = silu_and_checkpoint_backward(g, q, s)
    near(dx[-last:], *O.silu_backward(gt, O.values(wq, ws), None)["dx"], "dx")
    ok()


@pytest.mark.parametrize("M,N,K", [(70_016, 32_768, 16), (3, 140_032, 16_384), (150_016, 64, 16_384)])
def test_int8_gemm_past_32_bits(M, N, K):
    """c, b and a of more than 2^31 elements: the last rows and columns."""
    from linghe_b200.gemm.int8_gemm import int8_gemm
    gen = torch.Generator(device=DEV).manual_seed(1)
    a, b = [torch.randint(-128, 128, s, generator=gen, dtype=torch.int8, device=DEV) for s in ((M, K), (N, K))]
    sa, sb = torch.rand(M, device=DEV, generator=gen) + 0.1, torch.rand(N, device=DEV, generator=gen) + 0.1
    c = int8_gemm(a, b, sa, sb, out_dtype=torch.bfloat16)
    i, j = max(0, M - 130), max(0, N - 70)
    exact = ((a[i:].double() @ b[j:].double().t()) * sa[i:].double()[:, None] * sb[j:].double()).cpu()
    near(c[i:, j:].contiguous(), exact, 3.01 * O.U * exact.abs(), "c")
    ok()
