"""A backward pass with a side stream, captured into a HIP graph, for stacks whose weight gradients never
reach the side stream (normalisations above a layer whose gradient stays on the caller's stream): the
capture ends cleanly and its replays give the eager gradients, bit for bit."""
import pytest
import torch

from agents_amd import ops
from agents_amd.networks import layers as L
from agents_amd.networks import sequential
from agents_amd.specs import tensor_spec

pytestmark = pytest.mark.gpu

STACKS = {
    "small dense, norm": ((12,), lambda: [L.Dense(8, "tanh"), L.LayerNormalization()], False),
    "conv, norm": ((9, 9, 4), lambda: [L.Conv2D(16, 3, 2, "tanh"), L.LayerNormalization()], False),
    "conv, norm, head": ((9, 9, 4), lambda: [L.Conv2D(16, 3, 2, "relu"), L.LayerNormalization(),
                                             L.Flatten(), L.Dense(4)], False),
    "conv, norm, head done": ((9, 9, 4), lambda: [L.Conv2D(16, 3, 2, "relu"), L.LayerNormalization(),
                                                  L.Flatten(), L.Dense(4)], True),
    "conv, norm, dense, head": ((9, 9, 4), lambda: [L.Conv2D(16, 3, 2, "relu"), L.LayerNormalization(),
                                                    L.Flatten(), L.Dense(70, "relu"), L.Dense(4)],
                                False),
}


@pytest.mark.parametrize("name", list(STACKS))
def test_captured_backward_replays_the_eager_gradients(dev, name):
    shape, make, head_done = STACKS[name]
    net = sequential.Sequential(make(), input_spec=tensor_spec.TensorSpec(shape, torch.float32), seed=2)
    net.create_variables(device=dev)
    B = 9
    gen = torch.Generator(device=dev).manual_seed(1)
    xs = [torch.randn(B, *shape, generator=gen, device=dev) for _ in range(2)]
    x = xs[0].clone()
    dout = torch.randn(net.forward(x, slot="t", need_grad=True).shape, generator=gen, device=dev)
    side = ops.new_side_stream(dev)
    # what a loss launch that has run the head's backward leaves behind
    top = net._slots[("t", B)].dxs[-1]
    head = torch.randn(top.shape, generator=gen, device=dev) if head_done else None

    def step():
        net.forward(x, slot="t", need_grad=True)
        if head_done:
            top.copy_(head)
        net.backward(dout, slot="t", side_stream=side, head_done=head_done)

    want = []
    for src in xs:
        x.copy_(src)
        step()
        want.append(net.flat_grads.clone())
    assert not torch.equal(*want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):
        x.copy_(xs[i % 2])
        graph.replay()
        got = net.flat_grads.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want[i % 2]), i
        net.flat_grads.zero_()
        step()                                     # eager work between the replays
        assert torch.equal(net.flat_grads, want[i % 2])
