"""GPU: a selective block's cache stays the tensors that captured steps read."""
from __future__ import annotations

import pytest
import torch

from pathtile_b200.selective import SelectiveBlock

pytestmark = pytest.mark.gpu


def test_a_prompt_with_gradients_recorded_reaches_captured_steps(cuda_device):
    torch.manual_seed(12)
    block = SelectiveBlock(32, 16).to(cuda_device)
    cache = block.make_cache(2)
    x = torch.randn(2, 11, 32, device=cuda_device)
    token = torch.randn(2, 32, device=cuda_device)
    side = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(side):
        block.step(token, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = block.step(token, cache)
    for grad in (False, True):
        cache.window.zero_()
        cache.state.zero_()
        tensors = (cache.window, cache.state)
        with torch.set_grad_enabled(grad):
            block(x, cache=cache)
        assert cache.window is tensors[0] and cache.state is tensors[1]
        other = block.make_cache(2)
        with torch.no_grad():
            block(x, cache=other)
        want, _ = block.step(token, other)
        graph.replay()
        torch.testing.assert_close(y, want, rtol=1e-6, atol=1e-6)
        assert torch.equal(cache.window, other.window) and torch.equal(cache.state, other.state)


def test_gradients_through_two_prompts_into_one_cache(cuda_device):
    """What the first piece's backward pass has saved is not the cache that the second one moves on."""
    torch.manual_seed(13)
    block = SelectiveBlock(16, 8).to(cuda_device)
    x = torch.randn(2, 12, 16, device=cuda_device)

    def grads(pieces):
        cache = block.make_cache(2)
        outs = [block(piece, cache=cache)[0] for piece in pieces]
        return torch.autograd.grad(sum(o.square().sum() for o in outs), list(block.parameters()))

    first = grads([x[:, :5], x[:, 5:]])
    # The same two pieces, each on a cache of its own that starts where the piece does.
    one, two = block.make_cache(2), block.make_cache(2)
    with torch.no_grad():
        block(x[:, :5], cache=two)
    outs = [block(x[:, :5], cache=one)[0], block(x[:, 5:], cache=two)[0]]
    want = torch.autograd.grad(sum(o.square().sum() for o in outs), list(block.parameters()))
    for got, w in zip(first, want, strict=True):
        torch.testing.assert_close(got, w, rtol=1e-5, atol=1e-5 * float(w.abs().max()))
