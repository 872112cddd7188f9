"""CPU: the sequence operators as operators of torch's dispatcher.  On meta tensors
and on stand-ins for CUDA tensors shapes are checked and traced, nothing is launched."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import pathtile_b200 as pt
from pathtile_b200 import sequence

B, L, D, N, K = 2, 37, 24, 8, 4


@pytest.fixture(autouse=True)
def operators(native_lib):
    sequence._load()


def f(*shape, dtype=torch.float32, device="meta"):
    return torch.empty(*shape, dtype=dtype, device=device)


def conv_inputs(device="meta"):
    return dict(x=f(B, L, D, device=device), weight=f(D, K, device=device), bias=f(D, device=device),
                initial_state=f(B, K - 1, D, device=device))


def scan_inputs(device="meta"):
    rows = {k: f(B, L, D, dtype=torch.bfloat16, device=device) for k in ("x", "dt", "z")}
    shared = {k: f(B, L, 2, N, dtype=torch.bfloat16, device=device) for k in ("B", "C")}
    return dict(**rows, **shared, A=f(D, N, device=device), D=f(D, device=device), dt_bias=f(D, device=device),
                initial_state=f(B, D, N, device=device))


def norm_inputs(device="meta"):
    return dict(x=f(B, L, D, dtype=torch.float16, device=device), weight=f(D, device=device),
                gate=f(B, L, D, dtype=torch.float16, device=device), residual=f(B, L, D, device=device),
                scale=f(D, device=device))


CALLS = {
    "causal_conv": (conv_inputs, lambda v: pt.causal_conv(**v, silu=True, return_final_state=True)),
    "selective_scan": (scan_inputs, lambda v: pt.selective_scan(**v, return_final_state=True)),
    "fused_norm": (norm_inputs, lambda v: pt.fused_norm(**v, groups=3)),
}


def step_inputs(device="meta"):
    conv = dict(state=f(5, K - 1, D, device=device), x=f(B, D, device=device), weight=f(D, K, device=device))
    rows = {k: f(B, D, device=device) for k in ("x", "dt", "z")}
    scan = dict(state=f(5, D, N, device=device), **rows, A=f(D, N, device=device), B=f(B, N, device=device),
                C=f(B, N, device=device))
    return conv, scan, torch.zeros(B, dtype=torch.int32, device=device)


def steps(device="meta"):
    conv, scan, slots = step_inputs(device)
    return ((conv, lambda v: pt.causal_conv_step(**v, slots=slots)), (scan, lambda v: pt.selective_scan_step(**v, slots=slots)))


def in_order(make, call):
    names = list(make())
    return lambda *a: tuple(call(dict(zip(names, a))))


@pytest.mark.parametrize("name", CALLS)
def test_shapes_and_types_without_data(name):
    make, call = CALLS[name]
    v = {k: t.requires_grad_() for k, t in make().items()}
    outs = call(v)
    x = v["x"]
    last = {"causal_conv": "initial_state", "selective_scan": "initial_state", "fused_norm": "residual"}[name]
    for got, like in zip(outs, (x, v[last]), strict=True):
        assert got.is_meta and got.shape == like.shape and got.dtype == like.dtype and got.is_contiguous()
    grads = torch.autograd.grad(outs, list(v.values()), [torch.empty_like(t) for t in outs])
    assert all(g.shape == t.shape and g.dtype == t.dtype for g, t in zip(grads, v.values(), strict=True))
    only, = torch.autograd.grad(call(v)[1].sum(), v[last])
    assert only.shape == v[last].shape
    with torch.no_grad():
        assert not call(v)[0].requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(call(v)[0].sum(), x, create_graph=True)[0].sum().backward()


def test_shapes_of_steps_and_their_caches():
    for v, call in steps():
        before = v["state"]._version
        y = call(v)
        assert y.is_meta and y.shape == v["x"].shape and v["state"]._version > before
        with pytest.raises(ValueError, match="no_grad"):
            call({**v, "x": v["x"].clone().requires_grad_()})


@pytest.mark.parametrize("name", CALLS)
def test_make_fx_records_the_operators(name):
    make, call = CALLS[name]
    with FakeTensorMode() as mode:
        args, fn = list(make("cuda").values()), in_order(make, call)

        def grads(*a):
            leaves = [t.detach().requires_grad_() for t in a]
            outs = fn(*leaves)
            return torch.autograd.grad([t.sum() for t in outs], leaves)

        graph = make_fx(fn)(*args)
        both = make_fx(grads)(*make().values())  # the autograd engine asks for a real GPU even of stand-ins
        got = graph(*args)
    op, back = f"pathtile_b200.{name}.default", f"pathtile_b200.{name}_backward.default"
    assert [str(n.target) for n in graph.graph.nodes].count(op) == 1
    assert not any("empty" in str(n.target) for g in (graph, both) for n in g.graph.nodes)
    assert all([str(n.target) for n in both.graph.nodes].count(o) == 1 for o in (op, back))
    assert all(t.device.type == "cuda" and t.fake_mode is mode for t in got)


def test_make_fx_records_the_steps():
    with FakeTensorMode():
        for v, call in steps("cuda"):
            graph = make_fx(lambda *a: call(dict(zip(v, a))))(*v.values())
            assert sum("pathtile_b200" in str(n.target) for n in graph.graph.nodes) == 1
            graph.graph.eliminate_dead_code()
            assert sum("pathtile_b200" in str(n.target) for n in graph.graph.nodes) == 1


@pytest.mark.parametrize("name", CALLS)
def test_jit_trace_records_the_operators(name):
    make, call = CALLS[name]
    traced = torch.jit.trace(in_order(make, call), tuple(make().values()), check_trace=False)
    kinds = [n.kind() for n in traced.graph.nodes()]
    assert kinds.count(f"pathtile_b200::{name}") == 1 and "aten::empty" not in kinds


@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(grad):
    calls = [(make(), call) for make, call in CALLS.values()]
    for v, call in calls if grad else [*calls, *steps()]:
        for k, t in v.items():
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                dual = forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
                with pytest.raises(ValueError, match="forward mode"):
                    call({**v, k: dual})
        call(v)


def test_a_tangent_of_an_outputs_gradient_is_refused():
    for make, call in CALLS.values():
        v = {k: t.requires_grad_() for k, t in make().items()}
        outs = call(v)
        with forward_ad.dual_level():
            given = [forward_ad.make_dual(torch.empty_like(t), torch.empty_like(t)) for t in outs]
            with pytest.raises(ValueError, match="forward mode"):
                torch.autograd.grad(outs, list(v.values()), given)


def test_transforms_without_a_rule_say_so():
    for v, call in [(make(), call) for make, call in CALLS.values()] + list(steps()):
        one = lambda x: call({**v, "x": x})[0]
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.vmap(one)(torch.stack((v["x"], v["x"])))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.grad(lambda x: one(x).sum())(v["x"])
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(one, (v["x"],), (v["x"],))


def test_a_backward_operator_called_by_name_asks_for_no_gradient_of_its_own_accord():
    """As a traced gradient calls it: with plain tensors its results are plain too."""
    v = conv_inputs()
    args = [f(B, L, D), None, v["x"], v["weight"], None, None, None, True, [True, True, False, False]]
    assert not any(t.requires_grad for t in torch.ops.pathtile_b200.causal_conv_backward(*args))
    args[3] = args[3].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.ops.pathtile_b200.causal_conv_backward(*args)[0].sum().backward()


def test_operators_called_by_name_check_their_arguments():
    ops = torch.ops.pathtile_b200
    conv, scan, norm = conv_inputs(), scan_inputs(), norm_inputs()
    with pytest.raises(ValueError):
        ops.causal_conv(conv["x"], conv["weight"][:3], None, False, None, False, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv(torch.zeros(2, 3, 4), torch.zeros(4, 4), None, False, None, False, None)
    good = [f(B, L, D), None, conv["x"], conv["weight"], None, None, None, True, [True, True, False, False]]
    assert [t.shape for t in ops.causal_conv_backward(*good)] == [(B, L, D), (D, K)]
    for i, bad in ((0, f(B, L - 1, D)), (0, f(B, L, D).half()), (1, f(B, K, D)), (5, f(B, K, D)), (3, f(D - 1, K))):
        with pytest.raises(ValueError):
            ops.causal_conv_backward(*[bad if j == i else a for j, a in enumerate(good)])
    states = 3 * B * D * N  # 37 steps: three tiles of 16
    good = [scan["x"], None, scan["x"], scan["dt"], scan["A"], scan["B"], scan["C"], None, None, None, None, None, f(states),
            True, [True] * 5 + [False] * 4]
    assert [t.shape for t in ops.selective_scan_backward(*good)] == [t.shape for t in good[2:7]]
    for i, bad in ((0, f(B, L, D)), (1, f(B, D, N + 1)), (12, f(states - 1)), (12, f(states).half()), (4, f(D, N).double())):
        with pytest.raises(ValueError):
            ops.selective_scan_backward(*[bad if j == i else a for j, a in enumerate(good)])
    good = [norm["x"], norm["residual"], norm["x"], norm["weight"], None, None, norm["residual"], 1, 1e-5,
            [True, True, False, True, False]]
    assert len(ops.fused_norm_backward(*good)) == 3
    for i, bad in ((0, norm["residual"]), (1, norm["x"]), (6, None), (3, f(D + 1)), (7, 5)):
        with pytest.raises(ValueError):
            ops.fused_norm_backward(*[bad if j == i else a for j, a in enumerate(good)])
