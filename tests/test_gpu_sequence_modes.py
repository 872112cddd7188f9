"""GPU: the sequence operators under torch's tracers, dispatch modes and forward mode.

A traced call is the operator, not the memory that it allocates; a tangent, which
no operator carries on, is refused whether or not a gradient is asked for.
"""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import pathtile_b200 as pt
from test_gpu_sequence import BF16, F32, Maker, scan_inputs

pytestmark = pytest.mark.gpu


def conv_inputs(device, seed, b=2, l=23, d=24):
    m = Maker(device, seed)
    return dict(x=m(b, l, d), weight=m(d, 4), bias=m(d), initial_state=m(b, 3, d))


def scan_operands(device, seed, b=2, l=23, d=24, n=8):
    return scan_inputs(Maker(device, seed), b, l, d, n, 2, F32, True, True, True, True, False)


def norm_inputs(device, seed, shape=(3, 5, 48)):
    m = Maker(device, seed)
    return dict(x=m(*shape), weight=m(shape[-1]), gate=m(*shape), residual=m(*shape), scale=m(shape[-1]))


CALLS = {
    "conv": (conv_inputs, lambda v: pt.causal_conv(**v, silu=True, return_final_state=True)),
    "scan": (scan_operands, lambda v: pt.selective_scan(**v, dt_softplus=True, return_final_state=True)),
    "norm": (norm_inputs, lambda v: pt.fused_norm(**v, groups=3)),
}


def step_inputs(device, seed, b=3, d=24, n=8):
    m = Maker(device, seed)
    scan = scan_inputs(m, b, 1, d, n, 1, F32, True, True, True, False, False)
    now = {k: t[:, 0] if k in ("x", "dt", "B", "C", "z") else t for k, t in scan.items() if t is not None}
    return dict(window=m(b, 3, d), weight=m(d, 4), state=m(b, d, n), **now)


def both_steps(v):
    v = dict(v)
    u = pt.causal_conv_step(v.pop("window"), v.pop("x"), v.pop("weight"), silu=True)
    return pt.selective_scan_step(v.pop("state"), u, **v, dt_softplus=True)


def trace(how, fn, args):
    if how == "jit":
        return torch.jit.trace(fn, tuple(args), check_trace=False)
    return make_fx(fn, tracing_mode=how)(*args)


@pytest.mark.parametrize("how", ["jit", "real", "fake"])
@pytest.mark.parametrize("name", CALLS)
def test_a_traced_call_is_the_call(cuda_device, name, how):
    make, call = CALLS[name]
    v = make(cuda_device, 1)
    names = list(v)
    traced = trace(how, lambda *a: tuple(call(dict(zip(names, a)))), v.values())
    for seed in (1, 2):
        fresh = make(cuda_device, seed)
        for got, want in zip(traced(*fresh.values()), call(fresh), strict=True):
            assert torch.equal(got, want)


@pytest.mark.parametrize("name", CALLS)
def test_a_traced_gradient_is_the_gradient(cuda_device, name):
    make, call = CALLS[name]
    v = make(cuda_device, 3)
    names = list(v)

    def grads(*a):
        leaves = [t.detach().requires_grad_() for t in a]
        outs = call(dict(zip(names, leaves)))
        return torch.autograd.grad([t.sin().sum() for t in outs], leaves)

    traced = make_fx(grads)(*v.values())
    fresh = make(cuda_device, 4)
    for got, want in zip(traced(*fresh.values()), grads(*fresh.values()), strict=True):
        assert torch.equal(got, want)


@pytest.mark.parametrize("how", ["jit", "real"])
def test_a_traced_step_moves_the_cache_that_it_is_given(cuda_device, how):
    v = step_inputs(cuda_device, 5)
    names = list(v)
    traced = trace(how, lambda *a: both_steps(dict(zip(names, a))), [t.clone() for t in v.values()])
    for seed in (5, 6):
        one = step_inputs(cuda_device, seed)
        two = {k: t.clone() for k, t in one.items()}
        assert torch.equal(traced(*two.values()), both_steps(one))
        assert torch.equal(one["window"], two["window"]) and torch.equal(one["state"], two["state"])


def test_under_a_dispatch_mode_the_results_are_the_same(cuda_device):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for make, call in CALLS.values():
        v = make(cuda_device, 7)
        seen = []
        with Log():
            got = call(v)
        assert any("pathtile_b200" in s for s in seen)
        assert all(torch.equal(p, q) for p, q in zip(got, call(v), strict=True))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(cuda_device, name, grad):
    make, call = CALLS[name]
    v = make(cuda_device, 8)
    for k, t in v.items():
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
            with pytest.raises(ValueError, match="forward mode"):
                call({**v, k: dual})
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(v["x"], torch.ones_like(v["x"]))
        with pytest.raises(ValueError, match="forward mode"):
            call({**v, "x": dual})
    call(v)


def test_a_tangent_of_an_outputs_gradient_is_refused(cuda_device):
    for make, call in CALLS.values():
        v = {k: t.requires_grad_() for k, t in make(cuda_device, 9).items()}
        outs = call(v)
        with forward_ad.dual_level():
            given = [forward_ad.make_dual(torch.ones_like(t), torch.ones_like(t)) for t in outs]
            with pytest.raises(ValueError, match="forward mode"):
                torch.autograd.grad(outs, list(v.values()), given)


def test_a_tangent_is_refused_by_the_steps(cuda_device):
    v = step_inputs(cuda_device, 10)
    for k, t in v.items():
        with forward_ad.dual_level(), torch.no_grad():
            dual = forward_ad.make_dual(t.clone(), torch.ones_like(t))
            with pytest.raises(ValueError, match="forward mode"):
                both_steps({**v, k: dual})


def test_transforms_that_have_no_rule_for_the_operators_say_so(cuda_device):
    for make, call in CALLS.values():
        v = make(cuda_device, 11)
        rest = {k: t for k, t in v.items() if k != "x"}
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.vmap(lambda x: call({**rest, "x": x})[0])(torch.stack((v["x"], v["x"])))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.grad(lambda x: call({**rest, "x": x})[0].sum())(v["x"])
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(lambda x: call({**rest, "x": x})[0], (v["x"],), (v["x"],))


def test_in_inference_mode_a_step_counts_as_a_change_of_its_cache(cuda_device):
    m = Maker(cuda_device, 12)
    state, x, w = m(2, 3, 8, dtype=BF16), m(2, 8, dtype=BF16), m(8, 4)
    before = state._version
    with torch.inference_mode():
        y = pt.causal_conv_step(state, x, w)
        assert y.is_inference()
    assert state._version > before
