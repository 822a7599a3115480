"""The issuing threads of the 8-bit operators' pipelined kernels leave when their copies and MMAs are complete, also behind a wait that gave up: which
uses of the ring's barriers they wait for, by a model of the barriers, and that every kernel does so."""

import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "linghe_b200", "csrc", "lh_int8gemm.cu")


def loop(stages, uses):
    """s, ph, first of a warp behind `uses` steps of its loop."""
    s, ph, first = 0, 0, True
    for _ in range(uses):
        s += 1
        if s == stages:
            s, ph, first = 0, ph ^ 1, False
    return s, ph, first


@pytest.mark.parametrize("stages", [4, 5, 6])
def test_what_is_waited_for(stages):
    for uses in range(4 * stages + 2):
        s, ph, first = loop(stages, uses)
        # use u of the ring is on barrier u % stages and completes its phase u // stages, whose parity a wait names
        last = {u % stages: (u // stages) & 1 for u in range(max(0, uses - stages), uses)}
        copies = {i: ph if i < s else ph ^ 1 for i in range(stages) if i < s or not first}
        assert copies == last, (stages, uses)
        mmas = (s - 1, ph) if s > 0 else (stages - 1, ph ^ 1) if not first else None
        assert mmas == (None if uses == 0 else ((uses - 1) % stages, ((uses - 1) // stages) & 1)), (stages, uses)


def test_every_kernel_waits():
    with open(SOURCE) as fh:
        text = fh.read()
    kernels = [body for body in re.split(r"(?=__global__ )", text)[1:] if "STAGES; ++i) { mbar_init(&full[i]" in body]
    assert len(kernels) == 3
    for body in kernels:
        loads, rest = body.split("} else if (warp == 1) {", 1)
        assert "drain_copies<C::STAGES>(full, s, ph, " in loads
        assert "drain_mmas<C::STAGES>(empty, s, ph, " in rest
        # the flag of the first pass falls where the stage wraps
        assert len(re.findall(r"if \(\+\+s == C::STAGES\) \{ s = 0; ph \^= 1u; (?:first|fresh) = false; \}", body)) == 2


def test_the_ring_of_rows():
    """The norm pair's gradient fetches no row once its wait has given up, and then waits for the rows on their way."""
    with open(os.path.join(os.path.dirname(SOURCE), "lh_pair.cu")) as fh:
        text = fh.read()
    body = text[text.index("pair_bwd_kernel(const PairParams p)"):text.index("pair_reduce_kernel(")]
    in_loops = body[body.index("bool dead = false;"):]
    assert len(re.findall(r"\bfetch\(", in_loops)) == len(re.findall(r"if \(t == 0 && !dead && .*\) fetch\(", in_loops)) == 2
    assert re.search(r"if \(t == 0 && dead\) \{.*?\n.*?\n +for \(int i = max\(0, fetched - S\); i < fetched; \+\+i\) "
                     r"mbar_wait_inline\(&full\[i % S\], uint32_t\(i / S\) & 1u, DEVERR_FULL_WAIT\);", in_loops)
