"""Buffers that a kernel adds to with atomics are cleared by a kernel in front of it, in captured graphs too: every replay, with eager
work of the same sizes between, gives what the eager call gives.

Tolerance.  The sums are the same up to the order of n additions: at most n u sum |t| of them (u = 2^-24), with sum |t| about 0.64 n
for products of normal numbers and a largest sum of about 4.5 sqrt(n): 0.14 n^1.5 u of the largest, for n <= 16 * 256 (the reduction
of the convs, the pixels of the weight gradients) 2.2e-3, and the Winograd form's transforms may double it.  A buffer that was not
cleared is off by as much as the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('what', ['K split over the grid', 'Winograd-domain weight gradient'])
def test_replays_start_from_cleared_buffers(what):
    from advmix_amd import ops
    from advmix_amd._lib import lib
    B, C, H, W, R, stride = (2, 256, 8, 8, 3, 1) if what.startswith('K') else (32, 64, 24, 20, 4, 2)
    assert not what.startswith('K') or lib.advmix_conv_direct_config(0, B, H, W, C, C, R, R, stride) == 4
    g = torch.Generator().manual_seed(0)
    cl = lambda *s: torch.randn(*s, generator=g).cuda().contiguous(memory_format=torch.channels_last)          # noqa: E731
    w = torch.nn.Parameter(cl(C, C, R, R))
    x, dy = cl(B, C, H, W).requires_grad_(), cl(B, C, H // stride, W // stride)
    n0 = ops.COUNTERS.get('w4_wgrad', 0)

    def step(x):
        y = ops.conv2d(x, w, stride=stride, pad=1)
        y.backward(dy)
        return y.detach()
    eager = x.detach().clone().requires_grad_()
    want = [step(eager), eager.grad.clone(), w.grad.clone()]
    assert what.startswith('K') or ops.COUNTERS.get('w4_wgrad', 0) == n0 + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    x.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(x)
    for k in range(4):
        w.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, x.grad, w.grad), want):
            assert float((a - b).abs().max()) <= 5e-3 * float(b.abs().max()), k
        step(x.detach().clone().requires_grad_())
