"""The alignment that the header and the docstrings state is the alignment that is checked: every pointer of the 8-bit operators in turn,
half a boundary off, is refused unless it is one of those that lie anywhere."""

import os
import re

import pytest

from linghe_b200 import _lib
from tests.test_eight_bits_cpu import BF16, F32, P

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "linghe_b200.h")
ANYWHERE = {"os", "hs", "s", "a_s", "b_s", "dpost", "dpre", "r_post", "r_pre", "w", "dw"}
SIZES = {"M": 32, "n": 256, "N": 64, "K": 256, "G": 1, "dtype": BF16, "w_dtype": F32, "out_dtype": BF16, "alpha": 1.0, "eps": 1e-6, "codes": 1,
         "scratch_bytes": 1 << 40}
NAMES = ["lh_rmsnorm_pair_fwd", "lh_rmsnorm_pair_bwd", "lh_silu_checkpoint_fwd", "lh_silu_checkpoint_bwd", "lh_token_quant_int8", "lh_int8_gemm",
         "lh_int8_linear"]


def parameters(name):
    """(name, is a pointer) of every parameter but the stream."""
    with open(HEADER) as fh:
        text = re.sub(r"/\*.*?\*/", "", fh.read(), flags=re.S)
    args = re.search(name + r"\s*\(([^)]*)\)\s*;", text).group(1)
    return [(re.search(r"(\w+)\s*$", a).group(1), "*" in a) for a in args.split(",")][:-1]


@pytest.mark.parametrize("name", NAMES)
def test_every_pointer(name):
    lib, params = _lib.load(), parameters(name)
    pointers = [p for p, is_ptr in params if is_ptr]

    def call(**given):
        rc = getattr(lib, name)(*[given.get(p, P if is_ptr else SIZES.get(p)) for p, is_ptr in params], None)
        assert rc == _lib.LH_ERR_ARG, (name, given, rc)
        return lib.lh_last_error().decode()

    for p in pointers:
        if p not in ANYWHERE:
            assert "16-byte" in call(**{p: P + 8}), (name, p)


def test_the_documents_name_the_smoothing_factors():
    from linghe_b200.gemm.int8_gemm import int8_linear
    from linghe_b200.quant.token import token_quant_int8
    for f in (int8_linear, token_quant_int8):
        assert re.search(r"`smooth_scale` \(float32 \[K\], at a 16-byte boundary", f.__doc__)
    with open(HEADER) as fh:
        text = fh.read()
    assert "the smoothing factors' too" in text
