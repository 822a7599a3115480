"""What must not meet: a row's NaN and the rows beside it, calls of several host threads, a first call and the capture it comes in."""

import os
import subprocess
import sys
import threading

import pytest
import torch

from tests.test_gpu_eight_bits import DEV, KINDS, gemm_inputs, name, ok, pair_inputs, rand, same

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
VALUES = [float("nan"), float("inf"), 3e38]


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("gate", ["none", "sample", "token"])
@pytest.mark.parametrize("kind", [None, *KINDS], ids=name)
@pytest.mark.parametrize("lead,n", [((40, 5), 256), ((400, 3), 1408), ((200, 2), 4224), ((160, 2), 8192)])
def test_pair_rows(lead, n, kind, gate, value):
    """Rows with such a value in one tensor each; every other row has the bits of the call without them."""
    from linghe_b200.utils.norm import rms_norm_pair_backward, rms_norm_pair_forward
    x, o, post, pre, g, _ = [None if t is None else t.to(DEV) for t in pair_inputs(lead, n, torch.float32, gate)]
    dy, dh = rand(8, *x.shape).to(DEV), rand(9, *x.shape).to(DEV)

    def run(x, o, dy, dh):
        h, y, rp, rh, kept = rms_norm_pair_forward(x, o, post, pre, g, checkpoint=kind)
        back = (dy, dh, o, h) if kept is None else (dy, dh, kept[0], kept[2])
        scales = {} if kept is None else dict(o_scale=kept[1], h_scale=kept[3])
        dx, do, *_ = rms_norm_pair_backward(*back, post, pre, rp, rh, g, **scales)
        rows = [t.view(-1, n) for t in (h, y, dx, do)] + [t.view(-1, 1) for t in (rp, rh)]
        if kept is not None:
            rows += [kept[0].view(-1, n).view(torch.uint8), kept[1], kept[2].view(-1, n).view(torch.uint8), kept[3]]
        return rows

    want = run(x, o, dy, dh)
    M = x.numel() // n
    hit = [1, M // 3, M // 2, M - 2]
    tensors = [t.clone() for t in (x, o, dy, dh)]
    for t, r in zip(tensors, hit):
        t.view(-1, n)[r, n - 7] = value
    rest = torch.ones(M, dtype=torch.bool, device=DEV)
    rest[hit] = False
    for i, (a, b) in enumerate(zip(run(*tensors), want)):
        same(a[rest], b[rest].cpu(), f"output {i}")
    ok()


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("M,N,K", [(8, 272, 528), (40, 515, 496), (300, 1027, 528), (900, 4100, 1040)])
def test_linear_rows(M, N, K, value):
    from linghe_b200.gemm.int8_gemm import int8_linear
    x = rand(1, M, K).to(DEV)
    _, w, _, ws = [t.to(DEV) for t in gemm_inputs(1, N, K)]
    want = int8_linear(x, w, ws / K)
    other = x.clone()
    other[M // 2, K - 3] = value
    got = int8_linear(other, w, ws / K)
    rest = torch.arange(M, device=DEV) != M // 2
    same(got[rest], want[rest].cpu(), "other rows")
    ok()


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("M,n", [(33, 128), (70, 1408), (5000, 384)])
def test_silu_rows(M, n, value):
    from linghe_b200.utils.silu import silu_and_checkpoint_backward, silu_and_checkpoint_forward
    x, g, w = rand(1, M, 2 * n).to(DEV), rand(2, M, n).to(DEV), torch.rand(M, device=DEV)
    run = lambda x, g: (lambda y, q, s: (y, q, s, *silu_and_checkpoint_backward(g, q, s, w)))(*silu_and_checkpoint_forward(x, w))  # noqa: E731
    want = run(x, g)
    other, og = x.clone(), g.clone()
    other[M // 2, 3], og[M // 3, n - 1] = value, value
    rest = (torch.arange(M, device=DEV) != M // 2) & (torch.arange(M, device=DEV) != M // 3)
    for a, b in zip(run(other, og), want):
        same(a[rest], b[rest].cpu(), "other rows")
    ok()


def test_threads():
    """Eight host threads, each on its own stream with its own widths, repeat a step and get the same bits every time."""
    from linghe_b200.facade.norm import rms_norm_pair
    from linghe_b200.facade.silu import checkpointed_silu
    from linghe_b200.gemm.int8_gemm import int8_linear
    wrong = []

    def work(i, n):
        try:
            gen = torch.Generator(device=DEV).manual_seed(i)
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                x, o, u = [torch.randn((100 + i, c), device=DEV, generator=gen).bfloat16().requires_grad_() for c in (n, n, 2 * n)]
                w, codes = torch.ones(n, device=DEV).bfloat16(), torch.randint(-127, 128, (n, n), device=DEV, dtype=torch.int8)
                scales, first = torch.rand(n, device=DEV), None
                for _ in range(20):
                    h, y = rms_norm_pair(x, o, w, w, checkpoint=torch.int8 if i % 2 else None)
                    grads = torch.autograd.grad([h, y], [x, o], [torch.ones_like(h), h.detach()])
                    products = [int8_linear(y.detach()[:m], codes, scales) for m in (1, 5, 40, 100)]
                    act = checkpointed_silu(u)
                    out = [h.detach(), y.detach(), *grads, *products, act.detach(), *torch.autograd.grad(act, u, torch.ones_like(act))]
                    stream.synchronize()
                    first = first or [t.clone() for t in out]
                    wrong.extend((i, j) for j, (a, b) in enumerate(zip(out, first)) if not torch.equal(a, b))
        except BaseException as e:       # a thread's exception would go unseen
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=a) for a in enumerate([512, 1408, 4224, 5120, 8192, 256, 2048, 7168])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:10]
    ok()


def test_first_call_in_a_capture():
    """In a process that has launched none of the kernels yet every operator's first call is captured."""
    code = """
import torch
from tests.test_gpu_eight_bits_use import calls
fns, t = calls()
torch.cuda.synchronize()
graphs = []
for which, fn in fns.items():
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        graphs.append((which, fn, graph, fn(t)))
for which, fn, graph, out in graphs:
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, fn(t)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), which
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), (r.returncode, r.stderr[-2000:])
