"""Gradients as autograd hands them over: pieces of larger tensors that begin at any element."""

import pytest
import torch

from tests.test_gpu_eight_bits import DEV, name, ok, pair_inputs, rand, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [None, torch.int8], ids=name)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=name)
def test_pair_gradients_at_any_offset(dtype, kind):
    """h and y in one flat tensor behind an odd number of elements: the pieces of its gradient begin where no kernel reads."""
    from linghe_b200.facade.norm import rms_norm_pair
    x, o, post, pre, g, _ = [t.to(DEV).requires_grad_() for t in pair_inputs((9, 3), 384, dtype, "channel")[:5]] + [None]
    leaves = [x, o, post, pre, g]
    h, y = rms_norm_pair(*leaves[:4], gate=g, checkpoint=kind)
    gh, gy = [rand(s, *x.shape).to(dtype).to(DEV) for s in (7, 8)]
    want = torch.autograd.grad([h, y], leaves, [gh, gy])
    for odd in (1, 3):
        h, y = rms_norm_pair(*leaves[:4], gate=g, checkpoint=kind)
        flat = torch.cat([torch.zeros(odd, dtype=dtype, device=DEV), y.flatten(), torch.zeros(2, dtype=dtype, device=DEV), h.flatten()])
        grad = torch.cat([torch.ones(odd, dtype=dtype, device=DEV), gy.flatten(), torch.ones(2, dtype=dtype, device=DEV), gh.flatten()])
        for a, b in zip(torch.autograd.grad(flat, leaves, grad), want):
            same(a, b.cpu(), f"{odd} elements in front")
    ok()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=name)
def test_checkpointed_silu_gradient_at_any_offset(dtype):
    from linghe_b200.facade.silu import checkpointed_silu
    x, w = rand(1, 21, 768).to(dtype).to(DEV).requires_grad_(), torch.rand(21, device=DEV).requires_grad_()
    g = rand(2, 21, 384).to(dtype).to(DEV)
    want = torch.autograd.grad(checkpointed_silu(x, w), [x, w], g)
    for odd in (1, 3):
        flat = torch.cat([torch.zeros(odd, dtype=dtype, device=DEV), checkpointed_silu(x, w).flatten()])
        grad = torch.cat([torch.ones(odd, dtype=dtype, device=DEV), g.flatten()])
        for a, b in zip(torch.autograd.grad(flat, [x, w], grad), want):
            same(a, b.cpu(), f"{odd} elements in front")
    ok()
