"""GPU: the selective state space block -- the sequence operators one behind the
other, as a model calls them -- against the same block in plain float64 torch
operations, whose gradients come from autograd; and its single-token form
against its prompt form.

Tolerances: a block's output passes five matrix products and four operators in
fp32.  Measured against the largest value of a tensor, each operator adds at
most some hundred rounding steps (2^-24 each) at these lengths and the products
about as many as they sum terms, and a norm divides by a root mean square not
far below one: 2^-24 x 2000 = 1.2e-4 covers two blocks and their gradients.
"""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from pathtile_b200 import s4conv
from pathtile_b200.selective import SelectiveBlock

pytestmark = pytest.mark.gpu

TOL = 2000 * 2.0 ** -24


def near(got, want, what=""):
    scale = float(want.abs().max()) + 1e-30
    off = float((got.detach().double() - want).abs().max()) / scale
    assert off <= TOL, f"{what}: {off:.3g} of the largest value"


def plain_norm(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def plain_block(p, block, x, residual):
    """The block in float64, from its parameters p."""
    residual = x if residual is None else residual + x
    u, z = (plain_norm(residual, p["norm_weight"], block.eps) @ p["in_proj.weight"].t()).chunk(2, -1)
    length = u.shape[1]
    rows = F.pad(u, (0, 0, block.taps - 1, 0))
    u = F.silu(sum(rows[:, j:j + length] * p["conv_weight"][:, j] for j in range(block.taps)) + p["conv_bias"])
    dt, B, C = (u @ p["x_proj.weight"].t()).split((block.dt_rank, block.states, block.states), -1)
    delta = F.softplus(dt @ p["dt_proj.weight"].t() + p["dt_bias"])
    a = torch.exp(delta[..., None] * -torch.exp(p["log_A"]))
    h, ys = 0.0, []
    for t in range(length):
        h = a[:, t] * h + (delta[:, t] * u[:, t])[..., None] * B[:, t, None]
        ys.append((h * C[:, t, None]).sum(-1))
    y = torch.stack(ys, 1) + p["D"] * u
    return plain_norm(y * F.silu(z), p["out_norm_weight"], block.eps) @ p["out_proj.weight"].t(), residual


@pytest.mark.parametrize("b,length,hidden,states", [(3, 37, 32, 16), (2, 130, 24, 8), (1, 1, 16, 5)])
def test_two_blocks_against_plain_float64(cuda_device, b, length, hidden, states):
    torch.manual_seed(3)
    blocks = [SelectiveBlock(hidden, states).to(cuda_device) for _ in range(2)]
    x = torch.randn(b, length, hidden, device=cuda_device, requires_grad=True)
    gy, gr = torch.randn(2, b, length, hidden, device=cuda_device)
    y, residual = x, None
    for block in blocks:
        y, residual = block(y, residual)
    params = [p for block in blocks for p in block.parameters()]
    grads = torch.autograd.grad([y, residual], [x, *params], [gy, gr])
    x64 = x.detach().double().requires_grad_()
    p64 = [{n: p.detach().double().requires_grad_() for n, p in block.named_parameters()} for block in blocks]
    want, stream = x64, None
    for p, block in zip(p64, blocks):
        want, stream = plain_block(p, block, want, stream)
    near(y, want.detach(), "branch")
    near(residual, stream.detach(), "stream")
    names = ["x", *(f"{i}.{n}" for i, p in enumerate(p64) for n in p)]
    wants = torch.autograd.grad([want, stream], [x64, *(t for p in p64 for t in p.values())], [gy.double(), gr.double()])
    for name, grad, w in zip(names, grads, wants):
        near(grad, w, name)


def test_prompts_then_tokens_through_a_cache(cuda_device):
    torch.manual_seed(4)
    block = SelectiveBlock(48, 16).to(cuda_device)
    b, length, extra = 4, 21, 5
    x = torch.randn(b, length + extra, 48, device=cuda_device)
    with torch.no_grad():
        whole, _ = block(x)
        # The prompt in two pieces through one cache, then token by token.
        cache = block.make_cache(b)
        first, _ = block(x[:, :9], cache=cache)
        second, _ = block(x[:, 9:length], cache=cache)
        near(torch.cat((first, second), 1), whole[:, :length].double(), "prompt")
        big = block.make_cache(9)
        slots = torch.tensor([7, 0, 3, 8], dtype=torch.int32, device=cuda_device)
        big.window[slots.long()], big.state[slots.long()] = cache.window, cache.state
        for t in range(length, length + extra):
            y, _ = block.step(x[:, t], big, slots=slots)
            near(y, whole[:, t].double(), f"token {t}")
        assert not big.state[[1, 2, 4, 5, 6]].any() and not big.window[[1, 2, 4, 5, 6]].any()


def test_training_in_pieces_through_a_cache(cuda_device):
    """The second piece starts from the first one's end; its gradients stay within it."""
    torch.manual_seed(8)
    block = SelectiveBlock(16, 8).to(cuda_device)
    x = torch.randn(2, 12, 16, device=cuda_device)
    cache = block.make_cache(2)
    first, _ = block(x[:, :5], cache=cache)
    second, _ = block(x[:, 5:], cache=cache)
    (first.square().sum() + second.square().sum()).backward()
    assert all(torch.isfinite(p.grad).all() for p in block.parameters() if p.grad is not None)
    with torch.no_grad():
        whole, _ = block(x)
    near(torch.cat((first, second), 1), whole.double(), "two pieces")


def test_a_padded_batch_of_prompts(cuda_device):
    torch.manual_seed(5)
    block = SelectiveBlock(32, 16).to(cuda_device)
    lengths = torch.tensor([13, 1, 0, 7], dtype=torch.int32, device=cuda_device)
    x = torch.randn(4, 13, 32, device=cuda_device)
    with torch.no_grad():
        cache = block.make_cache(4)
        y, _ = block(x, lengths=lengths, cache=cache)
        for i, n in enumerate(lengths.tolist()):
            one = block.make_cache(1)
            if n:
                alone, _ = block(x[i:i + 1, :n], cache=one)
                near(y[i, :n], alone[0].double(), f"row {i}")
            near(cache.state[i], one.state[0].double(), f"state {i}")
            near(cache.window[i], one.window[0].double(), f"window {i}")


def test_a_block_in_bfloat16_and_under_autocast(cuda_device):
    """Two bfloat16 products of 32 and 64 terms, two more on what they made and six roundings between: 2^-8 each of
    about the largest value, twelve of them 0.047."""
    torch.manual_seed(7)
    block = SelectiveBlock(32, 16).to(cuda_device)
    x = torch.randn(2, 19, 32, device=cuda_device)
    with torch.no_grad():
        whole, _ = block(x)
        runs = {}
        with torch.autocast("cuda", dtype=torch.bfloat16):
            cache = block.make_cache(2, dtype=torch.bfloat16)
            y, _ = block(x[:, :18], cache=cache)
            token, _ = block.step(x[:, 18], cache)
            runs["autocast"] = torch.cat((y, token[:, None]), 1)
    half = SelectiveBlock(32, 16).to(cuda_device)
    half.load_state_dict(block.state_dict())
    half.bfloat16()
    y, _ = half(x.bfloat16())
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == torch.bfloat16 and p.grad.isfinite().all() for p in half.parameters())
    with torch.no_grad():
        cache = half.make_cache(2)
        first, _ = half(x[:, :18].bfloat16(), cache=cache)
        token, _ = half.step(x[:, 18].bfloat16(), cache)
        runs["bfloat16"] = torch.cat((first, token[:, None]), 1)
    runs["bfloat16, whole"] = y.detach()
    for name, got in runs.items():
        off = float((got.float() - whole).abs().max() / whole.abs().max())
        assert got.dtype == torch.bfloat16 and off <= 12 * 2.0 ** -8, f"{name}: {off:.3g}"


def test_the_model_trains_with_selective_blocks(cuda_device):
    torch.manual_seed(6)
    model = s4conv.Model(state_dim=16, hidden_dim=64, num_blocks=2, block="selective").to(cuda_device)
    x, target = s4conv.synthetic_batch(256, device=cuda_device, seed=1)
    before = [p.detach().clone() for p in model.parameters()]
    loss = s4conv.train_step(model, s4conv.make_optimizer(model), x, target)
    assert torch.isfinite(loss)
    moved = [not torch.equal(p, q) for p, q in zip(before, model.parameters())]
    assert all(torch.isfinite(p).all() for p in model.parameters()) and sum(moved) > len(moved) // 2
