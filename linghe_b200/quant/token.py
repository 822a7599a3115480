"""Token-wise int8 quantiser: one scale per row, the input of `linghe_b200.gemm.int8_gemm`."""

from __future__ import annotations

import torch

from linghe_b200 import _lib


def token_quant_int8(x, smooth_scale=None, out=None, scale=None):
    """One float32 scale per row and int8 codes of `x` [..., K] (bf16, fp16 or fp32; K % 16 == 0).

    With `smooth_scale` (float32 [K], at a 16-byte boundary like x) the row is divided by max(smooth_scale, 1e-30)
    first, as in the smooth quantisers of this package.  scale = max(amax / 127, 1e-30), code = nearest(x / scale), ties to even; a row
    with a NaN or an infinity gets a NaN scale.  Weights [N, K] take the same call: one scale per output channel.
    Returns (out int8 like x, scale float32 [rows])."""
    host = _lib.host()
    if host is not None:   # the same steps in C++ (host/lh_host.cpp)
        return host.token_quant_int8(x, smooth_scale, out, scale)
    K = x.shape[-1]
    assert x.dim() >= 1 and K > 0 and K % 16 == 0
    rows = x.numel() // K
    code = _lib.dtype_code(x)
    _lib.check_same(x, x.dtype, None, x=x)
    _lib.check_same(x, torch.float32, (K,), smooth_scale=smooth_scale)
    if out is None and scale is None:
        out, scale = _lib.empties(x, (tuple(x.shape), torch.int8), ((rows,), torch.float32))
    elif out is None:
        out = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    elif scale is None:
        scale = torch.empty((rows,), dtype=torch.float32, device=x.device)
    _lib.check_same(x, torch.int8, x.shape, out=out)
    _lib.check_same(x, torch.float32, (rows,), scale=scale)
    _lib.call("lh_token_quant_int8", x, _lib.ptr(x), _lib.ptr(smooth_scale), code, rows, K, _lib.ptr(out), _lib.ptr(scale))
    return out, scale
