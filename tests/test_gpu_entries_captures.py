"""What of autograd may be captured in a graph: work on streams that take part in the capture, and nothing that leads to a graph recorded outside."""
import pytest
import torch

from tests.test_gpu_dropout import check
from tests.test_gpu_point_dropout import leaves, shim, with_mask
from vet_amd import synthetic, torch_ops

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


@pytest.mark.parametrize("between", [False, True])
def test_a_render_beside_a_living_graph_of_the_same_leaf_is_refused(between, rasterizer):
    """Where its backward pass would come to that graph's stream. The gradients of other leaves are given."""
    scene = synthetic.tiny_scene(num_points=700, K=8, seed=9)
    inputs = leaves(scene)
    count = torch.full((1,), 3, dtype=torch.int64, device="cuda")
    texture, confidence = inputs[0], inputs[5]
    living = (texture * texture).sum()
    kw = dict(dropout=0.25, dropout_seed=5, dropout_device_step=count, allow_distortion=1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        sum(o.sum() for o in shim(scene, [texture.detach(), *inputs[1:]], **kw)).backward()
    torch.cuda.current_stream().wait_stream(stream)
    confidence.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = shim(scene, [1.0 * texture if between else texture, *inputs[1:]], **kw)
        with pytest.raises(RuntimeError, match="still lives"):
            sum(o.sum() for o in outs).backward()
        outs = shim(scene, inputs, **kw)
        (g,) = torch.autograd.grad(sum(o.sum() for o in outs), confidence)
    want, grads = with_mask(rasterizer, scene, 0.25, 5, 3)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(g.view(-1), grads["confidence"])
        torch.randn(100_000, device="cuda").sort()
    living.backward()
    assert torch.equal(texture.grad, 2 * texture.detach()) and confidence.grad is None
