"""Shared memory that kernels read in vectors of 16 bytes has an alignment that the source states: a dynamic array of a narrower type
begins wherever the kernel's static shared memory ends."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "linghe_b200", "csrc")
FILES = ["lh_int8gemm.cu", "lh_pair.cu", "lh_silu8.cu"]
BY_HAND = "{0} + ((1024u - (smem_u32({0}) & 1023u)) & 1023u)"


@pytest.mark.parametrize("file", FILES)
def test_dynamic_arrays_are_aligned(file):
    with open(os.path.join(CSRC, file)) as fh:
        text = fh.read()
    # split by kernel: each declares its own array
    for body in re.split(r"(?=__global__ )", text)[1:]:
        for align, array in re.findall(r"extern __shared__ (?:__align__\((\d+)\) )?\w+ (\w+)\[\];", body):
            assert (align and int(align) >= 16) or BY_HAND.format(array) in body, f"{file}: {array} of {body[:200]}"
