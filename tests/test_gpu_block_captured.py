"""The autograd forms captured into a graph, forward and backward, and replayed with other inputs."""

from __future__ import annotations

import pytest
import torch

from gpu_util import requires_gpu
from test_gpu_block_kernels import Chain, _randn

pytestmark = requires_gpu


@pytest.mark.parametrize("keep", [False, True])
def test_a_captured_step_replays_with_new_inputs(keep) -> None:
    chain = Chain(rows=300, dim=512, ffn=256)
    inputs = [(chain.x.clone(), chain.grad.clone()),
              (2 * _randn(300, 512, dtype=torch.bfloat16, seed=77), _randn(300, 512, dtype=torch.bfloat16, seed=78))]
    eager = []
    for x, grad in inputs:
        chain.x.copy_(x)
        chain.grad.copy_(grad)
        out, grads = chain.autograd(keep)
        eager.append((out.detach().clone(), [g.clone() for g in grads]))
        del out, grads
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain.autograd(keep)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, gots = chain.autograd(keep)
    for turn in range(4):
        x, grad = inputs[turn % 2]
        chain.x.copy_(x)
        chain.grad.copy_(grad)
        graph.replay()
        Chain(rows=40).calls(keep)  # the program's own work in between
        torch.cuda.synchronize()
        out, grads = eager[turn % 2]
        assert torch.equal(got, out) and all(torch.equal(g, w) for g, w in zip(gots, grads))
