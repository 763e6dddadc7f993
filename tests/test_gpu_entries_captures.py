"""What of autograd may be captured in a graph: work on streams that take part in the capture, and nothing that leads to a graph recorded outside."""
import pytest
import torch

from tests.test_gpu_dropout import check
from vet_amd import torch_ops

pytestmark = pytest.mark.gpu


def test_a_capture_on_two_streams():
    """x's part of the graph is recorded on a stream that the captured one has forked."""
    x = torch.randn(5000, device="cuda", requires_grad=True)
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            z = 2 * x
        main.wait_stream(side)
        y = torch_ops.dropout(z, 0.3, seed=4, step=2)
        (g,) = torch.autograd.grad(y, z, torch.ones_like(y))
        main.wait_stream(side)
        y, g = y.detach(), g.detach()
    for _ in range(3):
        y.zero_(), g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(y, 2 * x.detach(), 0.3, 4, 2)
        check(g, torch.ones_like(x), 0.3, 4, 2)
        torch.randn(100_000, device="cuda").sort()
