"""Matrix product in 8-bit integers with one scale per token and one per output channel.

Codes and scales of either operand come from `linghe_b200.quant.token.token_quant_int8`.  The sums are 32-bit
integers and exact, so a result does not depend on how many rows a call gets."""

from __future__ import annotations

import torch

from linghe_b200 import _lib


def _no_gradient(*tensors):
    """A gradient that would be lost without a word is refused."""
    assert not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)), (
        "the int8 product has no backward pass: call it under torch.no_grad() or on detached tensors")


def int8_gemm(a, b, a_s, b_s, out_dtype=torch.bfloat16):
    """c [..., N] = (a @ b.T) * a_s[:, None] * b_s for int8 `a` [..., K] and `b` [N, K], float32 `a_s` (one per row of
    a) and `b_s` [N].  K is a multiple of 16, at most 131056; out_dtype bf16, fp16 or fp32.
    There is no backward pass: scales that require a gradient are refused unless the call is under torch.no_grad()."""
    host = _lib.host()
    if host is not None:   # the same steps in C++ (host/lh_host.cpp)
        return host.int8_gemm(a, b, a_s, b_s, out_dtype)
    _no_gradient(a_s, b_s)
    assert out_dtype in _lib._DTYPES, f"unsupported out_dtype {out_dtype}"
    N, K = b.shape
    assert a.dim() >= 1 and a.shape[-1] == K, f"a has {a.shape[-1]} columns, b has {K}"
    assert K > 0 and K % 16 == 0
    M = a.numel() // K
    _lib.check_same(a, torch.int8, None, a=a, b=b)
    _lib.check_same(a, torch.float32, (M,), a_s=a_s)
    _lib.check_same(a, torch.float32, (N,), b_s=b_s)
    (c,) = _lib.empties(a, ((*a.shape[:-1], N), out_dtype))
    _lib.call("lh_int8_gemm", a, _lib.ptr(a), _lib.ptr(b), _lib.ptr(a_s), _lib.ptr(b_s), _lib.ptr(c), M, N, K, _lib._DTYPES[out_dtype])
    return c


def int8_linear(x, w, w_s, smooth_scale=None, out_dtype=None):
    """x @ dequant(w).T for `x` [..., K] (bf16, fp16 or fp32), quantised per token on the way, and int8 weights `w`
    [N, K] with one float32 scale `w_s` [N] per output channel: `token_quant_int8` and `int8_gemm` in one call.

    `smooth_scale` (float32 [K], at a 16-byte boundary like x): x is divided by it before it is quantised; the
    weights hold the product with it.
    The result has `out_dtype`, that of x by default.  There is no backward pass: an x, w_s or smooth_scale that requires a
    gradient is refused unless the call is under torch.no_grad()."""
    host = _lib.host()
    if host is not None:
        return host.int8_linear(x, w, w_s, smooth_scale, out_dtype)
    if out_dtype is None:
        out_dtype = x.dtype
    _no_gradient(x, w_s, smooth_scale)
    assert out_dtype in _lib._DTYPES, f"unsupported out_dtype {out_dtype}"
    N, K = w.shape
    assert x.dim() >= 1 and x.shape[-1] == K, f"x has {x.shape[-1]} columns, w has {K}"
    assert K > 0 and K % 16 == 0
    M = x.numel() // K
    code = _lib.dtype_code(x)
    _lib.check_same(x, x.dtype, None, x=x)
    _lib.check_same(x, torch.int8, None, w=w)
    _lib.check_same(x, torch.float32, (N,), w_s=w_s)
    _lib.check_same(x, torch.float32, (K,), smooth_scale=smooth_scale)
    c, q, s = _lib.empties(x, ((*x.shape[:-1], N), out_dtype), ((M, K), torch.int8), ((M,), torch.float32))
    _lib.call("lh_int8_linear", x, _lib.ptr(x), _lib.ptr(smooth_scale), code, _lib.ptr(w), _lib.ptr(w_s), _lib.ptr(q), _lib.ptr(s),
              _lib.ptr(c), M, N, K, _lib._DTYPES[out_dtype])
    return c
