"""The int8 product has no backward pass: where autograd would record the call it is refused instead of losing the gradient."""

import pytest
import torch

from linghe_b200 import _lib


@pytest.mark.parametrize("with_host_module", [True, False])
@pytest.mark.parametrize("which", ["x", "w_s", "smooth_scale"])
def test_an_input_that_wants_a_gradient(which, with_host_module, monkeypatch):
    from linghe_b200.gemm.int8_gemm import int8_linear
    if not with_host_module:
        monkeypatch.setattr(_lib, "_host", None)
    t = {"x": torch.zeros((4, 256)), "w_s": torch.ones(4), "smooth_scale": torch.ones(256)}
    w = torch.zeros((4, 256), dtype=torch.int8)
    t[which].requires_grad_()
    with pytest.raises(AssertionError, match="no backward pass"):
        int8_linear(t["x"], w, t["w_s"], t["smooth_scale"])
    # recorded nowhere: refused for being on the host only
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        int8_linear(t["x"], w, t["w_s"], t["smooth_scale"])
    with pytest.raises(RuntimeError, match="CUDA"):
        int8_linear(*(v.detach() if v is not w else w for v in (t["x"], w, t["w_s"], t["smooth_scale"])))


@pytest.mark.parametrize("with_host_module", [True, False])
@pytest.mark.parametrize("which", [0, 1])
def test_scales_that_want_a_gradient(which, with_host_module, monkeypatch):
    from linghe_b200.gemm.int8_gemm import int8_gemm
    if not with_host_module:
        monkeypatch.setattr(_lib, "_host", None)
    a, scales = torch.zeros((4, 256), dtype=torch.int8), [torch.ones(4), torch.ones(4)]
    scales[which].requires_grad_()
    with pytest.raises(AssertionError, match="no backward pass"):
        int8_gemm(a, a, *scales)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        int8_gemm(a, a, *scales)
