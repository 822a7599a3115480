"""What the 8-bit operators refuse, without a GPU: sizes, formats, alignment and NULL pointers at the C ABI, and tensors
on the host at the Python entry points."""

import ctypes

import pytest
import torch

from linghe_b200 import _lib

BF16, F16, F32, RAW = 0, 1, 2, 3
P = 1 << 12        # an aligned address that is never read: every call here is refused


def refused(name, *args, says):
    lib = _lib.load()
    rc = getattr(lib, name)(*args, None)
    assert rc == _lib.LH_ERR_ARG, (name, rc, lib.lh_last_error())
    assert says in lib.lh_last_error().decode(), lib.lh_last_error()


def pair_fwd(x=P, o=P, post=P, pre=P, gate=0, dtype=BF16, M=8, n=256, G=0, codes=0, h=P, y=P, rp=P, rh=P, oq=0, os=0, hq=0, hs=0):
    return x, o, post, pre, gate, dtype, M, n, G, 1.0, 1e-6, codes, h, y, rp, rh, oq, os, hq, hs


def pair_bwd(dy=P, dh=0, o=P, os=0, h=P, hs=0, post=P, pre=P, gate=0, rp=P, rh=P, dtype=BF16, M=8, n=256, G=0, codes=0, dx=P, do=P, dpost=P,
             dpre=P, dgate=0, scratch=P, nbytes=1 << 40):
    return dy, dh, o, os, h, hs, post, pre, gate, rp, rh, dtype, M, n, G, 1.0, codes, dx, do, dpost, dpre, dgate, scratch, nbytes


@pytest.mark.parametrize("case,says", [
    (dict(n=200), "128"), (dict(n=0), "128"), (dict(n=8320), "8192"), (dict(M=-1), "M=-1"), (dict(dtype=RAW), "dtype"), (dict(codes=3), "codes"),
    (dict(M=1 << 31), "too many rows"), (dict(gate=P, G=3), "gate"), (dict(gate=P, G=0), "gate"), (dict(gate=P, G=16), "gate"),
    (dict(x=0), "NULL"), (dict(pre=0), "NULL"), (dict(rh=0), "NULL"), (dict(codes=1), "checkpoint"), (dict(x=P + 8), "16-byte"), (dict(gate=P + 2, G=1), "16-byte")])
def test_pair_forward_refuses(case, says):
    refused("lh_rmsnorm_pair_fwd", *pair_fwd(**case), says=says)


@pytest.mark.parametrize("case,says", [
    (dict(n=130), "128"), (dict(n=8320), "8192"), (dict(dtype=7), "dtype"), (dict(codes=-1), "codes"), (dict(gate=P, G=5, dgate=P), "gate"),
    (dict(gate=P, G=1), "NULL"), (dict(dpost=0), "NULL"), (dict(dy=0), "NULL"), (dict(codes=1), "scales"), (dict(dh=P + 4), "16-byte"), (dict(nbytes=64), "scratch"), (dict(scratch=0), "NULL")])
def test_pair_backward_refuses(case, says):
    refused("lh_rmsnorm_pair_bwd", *pair_bwd(**case), says=says)


def test_pair_without_rows_needs_no_pointers():
    lib = _lib.load()
    assert lib.lh_rmsnorm_pair_fwd(*pair_fwd(x=0, o=0, h=0, y=0, M=0), None) == 0
    assert _lib.scratch_bytes("rmsnorm_pair_bwd", 0, 256) == 0
    assert _lib.scratch_bytes("rmsnorm_pair_bwd", 1 << 20, 256) > 0


@pytest.mark.parametrize("args,says", [
    ((P, 0, BF16, F32, 1, 8, 200, P, P, P), "128"), ((P, 0, BF16, F32, 0, 8, 256, P, P, P), "codes"), ((P, 0, RAW, F32, 1, 8, 256, P, P, P), "dtype"),
    ((P, P, BF16, F16, 1, 8, 256, P, P, P), "weights"), ((0, 0, BF16, F32, 1, 8, 256, P, P, P), "NULL"), ((P + 8, 0, BF16, F32, 1, 8, 256, P, P, P), "16-byte"),
    ((P, 0, BF16, F32, 1, 1 << 31, 128, P, P, P), "too many rows"), ((P, 0, BF16, F32, 2, -1, 128, P, P, P), "128")])
def test_silu_checkpoint_forward_refuses(args, says):
    refused("lh_silu_checkpoint_fwd", *args, says=says)


@pytest.mark.parametrize("args,says", [
    ((P, P, P, 0, BF16, F32, 1, 8, 100, P, 0), "128"), ((P, P, P, P, BF16, F32, 1, 8, 128, P, 0), "NULL"), ((P, P, P, 0, BF16, F32, 3, 8, 128, P, 0), "codes"),
    ((P, P + 8, P, 0, BF16, F32, 1, 8, 128, P, 0), "16-byte")])
def test_silu_checkpoint_backward_refuses(args, says):
    refused("lh_silu_checkpoint_bwd", *args, says=says)


@pytest.mark.parametrize("args,says", [
    ((P, 0, BF16, 8, 24, P, P), "16"), ((P, 0, RAW, 8, 32, P, P), "dtype"), ((P, 0, F32, -2, 32, P, P), "M=-2"), ((P, 0, F32, 8, 32, 0, P), "NULL"),
    ((P, P + 4, F32, 8, 32, P, P), "16-byte"), ((P, 0, F32, 8, 0, P, P), "16")])
def test_token_quant_refuses(args, says):
    refused("lh_token_quant_int8", *args, says=says)


@pytest.mark.parametrize("args,says", [
    ((P, P, P, P, P, 8, 8, 24, BF16), "16"), ((P, P, P, P, P, 8, 8, 131072, BF16), "131056"), ((P, P, P, P, P, 8, 0, 32, BF16), "N > 0"),
    ((P, P, P, P, P, -1, 8, 32, BF16), "M=-1"), ((P, P, P, P, P, 8, 8, 32, RAW), "out dtype"), ((P, P, 0, P, P, 8, 8, 32, BF16), "NULL"),
    ((P, P + 8, P, P, P, 8, 8, 32, BF16), "16-byte"), ((P, P, P, P, P + 8, 8, 8, 32, BF16), "16-byte"), ((P, P, P, P, P, 1 << 31, 8, 32, BF16), "range")])
def test_int8_gemm_refuses(args, says):
    refused("lh_int8_gemm", *args, says=says)


@pytest.mark.parametrize("args,says", [
    ((P, 0, BF16, P, P, P, P, P, 8, 8, 24, BF16), "16"), ((P, 0, RAW, P, P, P, P, P, 8, 8, 32, BF16), "dtype"), ((P, 0, BF16, 0, P, P, P, P, 8, 8, 32, BF16), "NULL"),
    ((P, 0, BF16, P, P, 0, P, P, 8, 8, 32, BF16), "NULL"), ((P, 0, BF16, P, P, P, P, P + 4, 8, 8, 32, BF16), "16-byte"), ((P, 0, BF16, P, P, P, P, P, 8, 8, 32, 9), "out dtype")])
def test_int8_linear_refuses(args, says):
    refused("lh_int8_linear", *args, says=says)


@pytest.mark.parametrize("with_host_module", [True, False])
def test_no_cpu_path(monkeypatch, with_host_module):
    """Tensors on the host are refused, with the C++ argument handling and without it."""
    from linghe_b200.gemm.int8_gemm import int8_gemm, int8_linear
    from linghe_b200.quant.token import token_quant_int8
    from linghe_b200.utils.norm import rms_norm_pair_backward, rms_norm_pair_forward
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    if not with_host_module:
        monkeypatch.setattr(_lib, "_host", None)
        monkeypatch.setattr(_lib, "_fn_cache", {})
    x, w, r = torch.zeros((4, 256)), torch.ones(256), torch.ones(4)
    q, s = torch.zeros((4, 256), dtype=torch.int8), torch.ones((4, 2))
    for call in (lambda: rms_norm_pair_forward(x, x, w, w), lambda: rms_norm_pair_backward(x, None, x, x, w, w, r, r),
                 lambda: silu_and_checkpoint_forward(x), lambda: silu_and_checkpoint_backward(x[:, :128].contiguous(), q, s),
                 lambda: token_quant_int8(x), lambda: int8_gemm(q, q, r, r), lambda: int8_linear(x, q, r)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_bound_signatures_take_pointers_first():
    assert _lib.SIGNATURES["lh_int8_linear"][1][0] is ctypes.c_void_p
    assert _lib.CHECKPOINTS == {None: 0, torch.int8: 1, torch.float8_e4m3fn: 2}
