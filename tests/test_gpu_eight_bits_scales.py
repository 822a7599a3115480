"""Scales, sums and per-row values lie at any float32: pieces of packed buffers give the bits of tensors of their own."""

import pytest
import torch

from tests.test_gpu_eight_bits import DEV, KINDS, TYPES, gemm_inputs, name, ok, pair_inputs, rand, same

pytestmark = pytest.mark.gpu


def off(t, by):
    """The same values `by` elements past the start of an allocation."""
    buf = torch.empty(t.numel() + by, dtype=t.dtype, device=DEV)
    buf[by:] = t.reshape(-1).to(DEV)
    v = buf[by:].view(t.shape)
    assert v.data_ptr() % 16 != 0
    return v


@pytest.mark.parametrize("by", [1, 3])
@pytest.mark.parametrize("kind", KINDS, ids=name)
def test_pair(kind, by):
    from linghe_b200.utils.norm import rms_norm_pair_backward, rms_norm_pair_forward
    x, o, post, pre, g, _ = [None if t is None else t.to(DEV) for t in pair_inputs((31, 5), 640, torch.bfloat16, "sample")]
    h, y, rp, rh, (oq, os_, hq, hs) = rms_norm_pair_forward(x, o, post, pre, g, checkpoint=kind)
    want = rms_norm_pair_backward(y, h, oq, hq, post, pre, rp, rh, g, 1.0, os_, hs)
    got = rms_norm_pair_backward(y, h, oq, hq, post, pre, off(rp, by), off(rh, by), g, 1.0, off(os_, by), off(hs, by))
    for a, b in zip(got, want):
        same(a, b.cpu(), "gradient")
    ok()


@pytest.mark.parametrize("by", [1, 3])
@pytest.mark.parametrize("weight", [torch.float32, torch.bfloat16], ids=name)
def test_silu(weight, by):
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    u, g, w = rand(3, 33, 768).bfloat16().to(DEV), rand(4, 33, 384).bfloat16().to(DEV), torch.rand(33).to(weight).to(DEV)
    y, q, s = silu_and_checkpoint_forward(u, w)
    for a, b in zip(silu_and_checkpoint_forward(u, off(w, by)), (y, q, s)):
        same(a, b.cpu(), "forward")
    for a, b in zip(silu_and_checkpoint_backward(g, q, off(s, by), off(w, by)), silu_and_checkpoint_backward(g, q, s, w)):
        same(a, b.cpu(), "gradient")
    ok()


@pytest.mark.parametrize("by", [1, 3])
@pytest.mark.parametrize("out_dtype", TYPES, ids=name)
@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (12, 300, 512), (40, 516, 496), (200, 4100, 112), (512, 4100, 528), (2048, 2504, 384), (900, 4104, 4112)])
def test_int8(M, N, K, out_dtype, by):
    from linghe_b200.gemm.int8_gemm import int8_gemm, int8_linear
    a, b, sa, sb = [t.to(DEV) for t in gemm_inputs(M, N, K)]
    sb = sb / K
    same(int8_gemm(a, b, off(sa, by), off(sb, by), out_dtype=out_dtype), int8_gemm(a, b, sa, sb, out_dtype=out_dtype).cpu(), "product")
    x = rand(9, M, K).to(out_dtype).to(DEV)
    same(int8_linear(x, b, off(sb, by)), int8_linear(x, b, sb).cpu(), "linear")
    ok()
