"""GPU: states that grow over a row whose length is cut into pieces.

A piece acts on the state before it as h -> exp(A sum delta) h + its own.  Where that
factor is past the largest float, a state of zero stays zero and a small one becomes what
the steps one by one make of it.  Tolerances as in test_gpu_sequence.py: errors grow with
the states, so relative to those they are a chain's.
"""
from __future__ import annotations

import pytest
import torch

import pathtile_b200 as pt
from oracle import sequence as ref
from test_gpu_sequence import Maker, close

pytestmark = pytest.mark.gpu


def inputs(device, rate, l=4000, last=30, d=16, n=16):
    """64 steps a piece (4000 steps of 16 channels are cut into 63).  Half the channels grow by e^rate a step, and
    nothing comes in before the last steps."""
    m = Maker(device, 111)
    x = torch.zeros(1, l, d, device=device)
    x[:, l - last:] = m(1, last, d)
    A = torch.full((d, n), -1.0, device=device)
    A[::2] = rate
    return dict(x=x, dt=torch.ones(1, l, d, device=device), A=A, B=m(1, l, n), C=m(1, l, n))


@pytest.mark.parametrize("rate", [1.0, 2.0, 2.5])
def test_nothing_grows_out_of_a_state_of_zero(cuda_device, rate):
    v = inputs(cuda_device, rate)
    y, last = pt.selective_scan(**v, return_final_state=True)
    one, size = (ref.scan(**v, absolute=a) for a in (False, True))
    close(y, one["y"], size["y"], 4 * 30 + 48, "y")
    close(last, one["state"], size["state"], 4 * 30 + 48, "state")
    # A step's own factor has to be a float, below e^88.7: e^100 times a state of zero is not a number in fp32.
    still = {**v, "x": torch.zeros_like(v["x"]), "A": v["A"] * 35}
    y, last = pt.selective_scan(**still, return_final_state=True)
    assert not y.any() and not last.any()


def test_a_small_state_grows(cuda_device):
    """65 steps are cut into 48 and 17; 48 steps of e^2.5 are e^120, and the state ends at e^82."""
    m = Maker(cuda_device, 112)
    l, d, n = 65, 16, 16
    v = dict(x=torch.zeros(1, l, d, device=cuda_device), dt=torch.ones(1, l, d, device=cuda_device),
             A=torch.full((d, n), 2.5, device=cuda_device), B=m(1, l, n), C=m(1, l, n))
    state = m(1, d, n) * 1.8e-35
    y, last = pt.selective_scan(**v, initial_state=state, return_final_state=True)
    one, size = (ref.scan(**v, state=state, absolute=a) for a in (False, True))
    close(y, one["y"], size["y"], 4 * l + 48, "y")
    close(last, one["state"], size["state"], 4 * l + 48, "state")


def test_gradients_of_growing_states(cuda_device):
    """Backward the pieces hand gradients on in the same way: here the last steps have none."""
    v = {k: t.requires_grad_() for k, t in inputs(cuda_device, 2.0).items()}
    y, last = pt.selective_scan(**v, return_final_state=True)
    dy = torch.zeros_like(y)
    dy[:, :20] = 1.0
    grads = torch.autograd.grad([y, last], list(v.values()), [dy, torch.zeros_like(last)])
    one, size = (ref.scan(**{k: t.detach() for k, t in v.items()}, dy=dy, absolute=a) for a in (False, True))
    for name, grad in zip(v, grads):
        close(grad, one["d" + name], size["d" + name], 2 * (4 * 20 + 48) + 4000 / 8, "d" + name)
