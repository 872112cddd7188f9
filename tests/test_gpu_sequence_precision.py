"""GPU: the elementary functions inside the sequence operators in fp32, over their whole range.

Errors are counted in half steps, 2^-24 of the value.  The hardware's 2^x is right to
2^-22 (four half steps), the correction behind it costs a fifth; its reciprocal is right
to a step (two), a product or sum to a half step:

* sigmoid = 1 / (1 + e): 5 + 1 + 2 = 8; silu 9; a product more where one follows;
* softplus = 2 artanh(s) for s = e / (2 + e): e 5, 2 + e 1, reciprocal 2, product 1, times
  1.08 at most (the slope of log artanh against log s at s = 1/3) is 9.8; the series' end
  0.4, its last product 1 and the smaller ones before it 0.5, the final sum 1: 13;
* silu' = s (1 + v (1 - s)), against its terms' sizes, s (1 + |v| (1 + s)): s 8; of
  v (1 - s) at most 4 from s and 1 from the difference; products and sum 3: 16.
"""
from __future__ import annotations

import pytest
import torch

import pathtile_b200 as pt

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24


def values(device):
    """-80 to 80, dense around zero, the tails (e^-80 is still a normal number) and where steps in time start."""
    grid = torch.cat([torch.linspace(-80, 80, 30011), torch.linspace(-9, 9, 30011), torch.linspace(-0.01, 0.01, 2003)])
    return grid.to(torch.float32).to(device)


def within(got, want, size, halves, what):
    off = (got.double() - want).abs() / (size * HALF)
    worst = int(off.argmax())
    assert float(off.max()) <= halves, f"{what}: {float(off.max()):.3g} half steps at {worst} ({float(want.flatten()[worst]):.4g})"


def silu64(v):
    v = v.double()
    s = torch.sigmoid(v)
    return v * s, s * (1 + v * (1 - s)), s * (1 + v.abs() * (1 + s))


def test_softplus(cuda_device):
    """A scan of one step from nothing with B = C = x = 1 gives the step's duration; its gradient the sigmoid."""
    v = values(cuda_device)
    d = v.numel()
    one = torch.ones(1, 1, d, device=cuda_device)
    A, B = torch.zeros(d, 1, device=cuda_device), torch.ones(1, 1, 1, device=cuda_device)
    want = torch.nn.functional.softplus(v.double(), threshold=1e9)
    dt = v.view(1, 1, d).clone().requires_grad_()
    y = pt.selective_scan(one, dt, A, B, B, dt_softplus=True)
    within(y.detach().view(-1), want, want, 13, "softplus")
    grad, = torch.autograd.grad(y, dt, one)
    sig = torch.sigmoid(v.double())
    within(grad.view(-1), sig, sig, 8, "its slope")
    y = pt.selective_scan_step(torch.zeros(1, d, 1, device=cuda_device), one[:, 0], v.view(1, d), A, B[:, 0], B[:, 0],
                               dt_softplus=True)
    within(y.view(-1), want, want, 13, "softplus of a step")


def test_silu_in_the_scan(cuda_device):
    v = values(cuda_device)
    d = v.numel()
    one, zero = torch.ones(1, 1, d, device=cuda_device), torch.zeros(1, 1, 1, device=cuda_device)
    A, D = torch.zeros(d, 1, device=cuda_device), torch.ones(d, device=cuda_device)
    y64, slope, size = silu64(v)
    z = v.view(1, 1, d).clone().requires_grad_()
    y = pt.selective_scan(one, one, A, zero, zero, D, z)
    within(y.detach().view(-1), y64, y64.abs() + 1e-300, 9, "silu")
    grad, = torch.autograd.grad(y, z, one)
    within(grad.view(-1), slope, size, 16, "its slope")
    y = pt.selective_scan_step(torch.zeros(1, d, 1, device=cuda_device), one[:, 0], one[:, 0], A, zero[:, 0], zero[:, 0], D,
                               v.view(1, d))
    within(y.view(-1), y64, y64.abs() + 1e-300, 9, "silu of a step")


def test_silu_in_the_convolution(cuda_device):
    v = values(cuda_device)
    d = v.numel()
    w = torch.ones(d, 1, device=cuda_device)
    y64, slope, size = silu64(v)
    x = v.view(1, 1, d).clone().requires_grad_()
    y = pt.causal_conv(x, w, silu=True)
    within(y.detach().view(-1), y64, y64.abs() + 1e-300, 9, "silu")
    grad, = torch.autograd.grad(y, x, torch.ones_like(y))
    within(grad.view(-1), slope, size, 16, "its slope")
    y = pt.causal_conv_step(torch.zeros(1, 0, d, device=cuda_device), v.view(1, d), w, silu=True)
    within(y.view(-1), y64, y64.abs() + 1e-300, 9, "silu of a step")


@pytest.mark.parametrize("width", [512, 509])
def test_silu_in_the_norm(cuda_device, width):
    """On top of a stream of zeros the stream that goes on is the gated input."""
    v = values(cuda_device)
    v = v[:v.numel() // width * width].view(-1, width)
    y64, slope, size = silu64(v)
    gate = v.clone().requires_grad_()
    one = torch.ones_like(v)
    y, r = pt.fused_norm(one, one[0], gate=gate, residual=torch.zeros_like(v))
    within(r.detach(), y64, y64.abs() + 1e-300, 9, "silu")
    grad, = torch.autograd.grad([y, r], gate, [torch.zeros_like(v), one])
    within(grad, slope, size, 16, "its slope")


def test_far_out_and_not_a_number(cuda_device):
    """Beyond what the exponential can hold the functions are 0, their argument, or what 64 bits give."""
    big = torch.finfo(torch.float32).max
    v = torch.tensor([-big, -1e30, -1000.0, -104.0, 104.0, 1000.0, 1e30, big, float("inf"), float("nan")], device=cuda_device)
    d = v.numel()
    x = v.view(1, 1, d).clone().requires_grad_()
    y = pt.causal_conv(x, torch.ones(d, 1, device=cuda_device), silu=True)
    grad, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert y.flatten()[:4].abs().max() <= 1e-30 and torch.equal(y.flatten()[4:9], v[4:9]) and y.flatten()[9].isnan()
    assert grad.flatten()[:4].abs().max() <= 1e-30 and torch.equal(grad.flatten()[4:8], torch.ones_like(v[4:8]))
    assert grad.flatten()[9].isnan()
    B = torch.ones(1, 1, 1, device=cuda_device)
    v = torch.cat((v, torch.tensor([-float("inf")], device=cuda_device)))
    one, dt = torch.ones(1, 1, d + 1, device=cuda_device), v.view(1, 1, d + 1)
    y = pt.selective_scan(one, dt, -torch.ones(d + 1, 1, device=cuda_device), B, B, dt_softplus=True).flatten()
    assert y[:4].abs().max() <= 1e-30 and torch.equal(y[4:9], v[4:9]) and y[9].isnan() and y[10] == 0
