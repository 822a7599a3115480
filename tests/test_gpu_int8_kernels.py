"""Every kernel of the int8 product at small ragged sizes, and that the sizes reach the kernel they are meant for."""

import json
import re

import pytest
import torch

from oracle import eight_bits as O
from tests.test_gpu_eight_bits import DEV, TYPES, gemm_inputs, name, near, ok

pytestmark = pytest.mark.gpu

# (kernel, columns of a tile where it has several widths, parts of k), sizes.  An odd N has rows that no tensor map describes in any type,
# one of 4 k + 2 in the 16-bit types only; the last tile of rows, columns and k is ragged everywhere.
VARIANTS = [
    (("pair", 256, 1), (1000, 4097, 4096)), (("pair", 256, 1), (6000, 6017, 2064)), (("pair", 256, 1), (4100, 6016, 2064)), (("pair", 256, 1), (900, 4100, 4112)),
    (("tile", 128, 1), (4100, 4099, 400)), (("tile", 128, 1), (2048, 2500, 384)),
    (("split", 128, 1), (512, 4099, 528)), (("split", 128, 1), (511, 4108, 144)), (("split", 128, 2), (500, 2051, 2064)), (("split", 128, 4), (17, 3499, 6160)),
    (("split", 64, 1), (200, 4099, 112)), (("split", 64, 1), (201, 4100, 80)),
    (("split", 64, 2), (257, 129, 240)), (("split", 64, 3), (257, 129, 272)), (("split", 64, 4), (40, 515, 496)), (("split", 64, 6), (130, 515, 720)),
    (("split", 64, 6), (30, 516, 720)), (("split", 64, 6), (129, 303, 2064)), (("split", 64, 8), (97, 300, 4112)),
    (("rows", 8, 1), (8, 1111, 2064)), (("rows", 16, 1), (15, 1111, 528)),
]


@pytest.mark.parametrize("out_dtype", TYPES, ids=name)
@pytest.mark.parametrize("variant,size", VARIANTS)
def test_ragged(variant, size, out_dtype):
    from linghe_b200.gemm.int8_gemm import int8_gemm
    M, N, K = size
    a, b, sa, sb = gemm_inputs(M, N, K, seed=5)
    if out_dtype == torch.float16:
        sa = sa * 2e-4                                     # stay below 65504
    behind = torch.full((M * N + 64,), 7.0, dtype=out_dtype, device=DEV)
    c = int8_gemm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV), out_dtype=out_dtype)
    exact = (a.to(DEV).double() @ b.to(DEV).double().t()).cpu() * sa.double()[:, None] * sb.double()
    near(c, exact, 3.01 * O.U * exact.abs(), "c")
    # the rows end where they should: the same call into the front of a larger buffer leaves what is behind it
    from linghe_b200 import _lib
    args = [t.to(DEV) for t in (a, b, sa, sb)]
    _lib.call("lh_int8_gemm", behind, *[_lib.ptr(t) for t in args], _lib.ptr(behind), M, N, K, _lib._DTYPES[out_dtype])
    assert torch.equal(behind[:M * N].view(M, N), c) and (behind[M * N:] == 7).all()
    ok()


def test_the_sizes_reach_their_kernels(tmp_path):
    from torch.profiler import ProfilerActivity, profile
    from linghe_b200.gemm.int8_gemm import int8_gemm
    wrong = []
    for (kind, width, parts), (M, N, K) in VARIANTS:
        args = [t.to(DEV) for t in gemm_inputs(M, N, K)]
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            int8_gemm(*args)
            torch.cuda.synchronize()
        prof.export_chrome_trace(str(tmp_path / "trace.json"))
        with open(tmp_path / "trace.json") as fh:
            launched = [e for e in json.load(fh)["traceEvents"] if e.get("cat") == "kernel" and "int8_" in e["name"]]
        if not launched:
            pytest.skip("no kernel is recorded on this machine")
        found = re.search(r"int8_(pair|tile|split|rows)_kernel(?:ILi(\d+)E|<(\d+)>)?", launched[0]["name"])
        of = int(found.group(2) or found.group(3) or 256)
        tiles = -(-M // 128) * -(-N // of)
        got = (found.group(1), of * 8 if found.group(1) == "rows" else of, launched[0]["args"]["grid"][0] // tiles if found.group(1) == "split" else 1)
        if got != (kind, width, parts):
            wrong.append(((M, N, K), (kind, width, parts), got))
    assert not wrong, wrong
