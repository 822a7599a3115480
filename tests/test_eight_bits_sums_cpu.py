"""That the inputs and bounds of the tests of sums over rows can tell a wrong sum from rounding (no GPU)."""

import pytest
import torch

from oracle import eight_bits as O

GATES = ["none", "channel", "sample", "token"]


@pytest.mark.parametrize("with_dh", [True, False], ids=["dh", "no dh"])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("lead,n", [((999,), 256), ((700, 2), 384), ((12000, 5), 128)])
def test_every_row_shows_in_every_sum(lead, n, gate, with_dh):
    if len(lead) == 1 and gate == "sample":
        lead = (1, *lead)
    d, sums, terms = O.whole_rows(lead, n, gate, with_dh)
    hn = d["h"] * d["r_pre"][:, None]
    assert not (d["dy"] * d["pre"] * hn).sum(1).any()                    # no mean enters dx
    for key, t in terms.items():
        assert t.abs().min() >= 0.25 and (t.sign() == t.sign()[0]).all(), key       # no row is lost unseen
        assert torch.equal(t * 4, (t * 4).round()) and float(t.abs().sum(0).max()) * 4 < 2 ** 24, key      # exact in any order
    for t in (d["dy"], d["post"], d["pre"], d["o"], d["h"], sums["dx"], d["dh"] if with_dh else sums["dx"]):
        for dtype in (torch.bfloat16, torch.float16):
            assert torch.equal(t.to(dtype).double(), t)
    for v, s in ((d["o"], d["o_scale"]), (d["h"], d["h_scale"])):
        q = v / s.repeat_interleave(128, 1)
        for dtype in (torch.int8, torch.float8_e4m3fn):
            assert torch.equal(O.values(q.to(dtype), s.float()), v)


def test_the_bounds_reject_lost_sums():
    """Zero in place of a sum, and a sum without one CTA's rows, at values of both signs."""
    M, n = 7000, 256
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    dy, dh, o, h = 0.1 * r(M, n), 0.1 * r(M, n), r(M, n), r(M, n)
    post, pre, gate = 1 + 0.3 * r(n), 1 + 0.3 * r(n), torch.sigmoid(r(M, n))
    rp, rh = [(t.square().mean(1) + 1e-6).rsqrt() for t in (o, h)]
    want = O.pair_backward(dy, dh, o, h, post, pre, rp, rh, gate, 0.8, depth=O.row_depth(M))
    part = O.pair_backward(dy[48:], dh[48:], o[48:], h[48:], post, pre, rp[48:], rh[48:], gate[48:], 0.8)      # without the 48 rows of a CTA
    for key in ("dpost", "dpre"):
        value, bound = want[key]
        assert (value.abs() > bound).double().mean() > 0.97, key
        assert ((value - part[key][0]).abs() > bound).double().mean() > 0.9, key


def test_a_gate_per_element_is_no_sum():
    """Its gradient is one product per element: dh or on rounded to bf16 on the way is outside the bound."""
    M, n = 64, 256
    gen = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    dy, dh, o, h = 0.1 * r(M, n), 0.1 * r(M, n), r(M, n), r(M, n)
    post, pre, gate = 1 + 0.3 * r(n), 1 + 0.3 * r(n), torch.sigmoid(r(M, n))
    rp, rh = [(t.square().mean(1) + 1e-6).rsqrt() for t in (o, h)]
    value, bound = O.pair_backward(dy, dh, o, h, post, pre, rp, rh, gate, 0.8, depth=0)["dgate"]
    off = (value.bfloat16().double() - value).abs()
    assert (off > bound + O.half_step(value, torch.float32)).double().mean() > 0.9
