"""Sums over rows of the norm pair's gradient.  Where every sum is exact in float32 the kernel's has to be equal, whatever the order
of its additions; elsewhere it is held to a bound that counts the additions the kernel makes."""

import pytest
import torch

from oracle import eight_bits as O
from tests.test_gpu_eight_bits import DEV, KINDS, TYPES, name, near, ok, pair_inputs, rand, same

pytestmark = pytest.mark.gpu

GATES = ["none", "channel", "sample", "token"]


# one row; fewer rows than SMs; groups of gate rows inside a CTA's share and over several; many rows to a CTA; one and two
# vectors of a row to a thread; in float32 one row to the shared memory
@pytest.mark.parametrize("with_dh", [True, False], ids=["dh", "no dh"])
@pytest.mark.parametrize("kind", [None, *KINDS], ids=name)
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("lead,n", [((1, 1), 128), ((7, 9), 640), ((700, 2), 2048), ((2, 700), 512), ((149, 7), 384), ((12000, 5), 128), ((1400, 5), 1408),
                                    ((301, 5), 5120), ((300, 4), 8192)])
def test_whole_rows(lead, n, gate, dtype, kind, with_dh):
    from linghe_b200.utils.norm import rms_norm_pair_backward
    d, want, _ = O.whole_rows(lead, n, gate, with_dh, device=DEV)
    rows, shape = d["o"].shape[0], (*lead, n)
    o, h, scales = d["o"].to(dtype), d["h"].to(dtype), {}
    if kind is not None:
        o, h = [(d[k] / d[k + "_scale"].repeat_interleave(128, 1)).to(kind) for k in ("o", "h")]
        scales = {k: d[k].float() for k in ("o_scale", "h_scale")}
    out = rms_norm_pair_backward(d["dy"].to(dtype).contiguous().view(shape), d["dh"].to(dtype).view(shape) if with_dh else None, o.view(shape), h.view(shape),
                                 d["post"].to(dtype), d["pre"].to(dtype), d["r_post"].float(), d["r_pre"].float(),
                                 gate=None if d["gate"] is None else d["gate"].to(dtype), residual_scale=d["alpha"], **scales)
    same(out[0].view(rows, n), want["dx"].to(dtype).cpu(), "dx")
    same(out[2], want["dpost"].float().cpu(), "dpost")
    same(out[3], want["dpre"].float().cpu(), "dpre")
    if gate != "none":
        same(out[4], want["dgate"].to(dtype).cpu(), "dgate")
    ok()


@pytest.mark.parametrize("kind", [None, torch.int8], ids=name)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=name)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("lead,n", [((37, 1), 1408), ((12000, 5), 128), ((1400, 5), 1408), ((301, 5), 5120), ((300, 4), 8192)])
def test_sums_within_the_additions_made(lead, n, gate, dtype, kind):
    from linghe_b200.utils.norm import rms_norm_pair_backward
    x, o, post, pre, g, full = pair_inputs(lead, n, dtype, gate, seed=51)
    rows, alpha = o.numel() // n, 0.8
    rp, rh = [((t.double().view(rows, n).square().mean(1) + 1e-6).rsqrt()).float() for t in (o, x)]
    dy, dh = rand(61, *x.shape, scale=0.1).to(dtype), rand(62, *x.shape, scale=0.1).to(dtype)
    ov, hv, ot, ht, osc, hsc = o.double().view(rows, n), x.double().view(rows, n), o, x, None, None
    if kind is not None:
        (oq, osc), (hq, hsc) = O.codes(o.view(rows, n), kind), O.codes(x.view(rows, n), kind)
        ov, hv, ot, ht = O.values(oq, osc), O.values(hq, hsc), oq.view(o.shape), hq.view(x.shape)
    put = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    out = rms_norm_pair_backward(*[put(t) for t in (dy, dh, ot, ht, post, pre, rp, rh)], gate=put(g), residual_scale=alpha, o_scale=put(osc), h_scale=put(hsc))
    args = [put(t) for t in (dy.view(rows, n), dh.view(rows, n), ov, hv, post, pre, rp, rh, full)]
    sums = O.pair_backward(*args, alpha, depth=O.row_depth(rows))
    near(out[2], *[t.cpu() for t in sums["dpost"]], "dpost")
    near(out[3], *[t.cpu() for t in sums["dpre"]], "dpre")
    if g is not None:
        G = g.numel() // n
        value, bound = sums["dgate"] if G < rows else O.pair_backward(*args, alpha, depth=0)["dgate"]
        near(out[4], *[t.view(rows // G, G, n).sum(0).view(g.shape).cpu() for t in (value, bound)], "dgate")
    ok()
