"""GPU: the forms of the sequence operators' kernels that only large calls choose,
and the backward passes under graphs and on streams.

Which form a call takes follows from its sizes on 148 SMs; each case names the
one it is there for.  Tolerances as in test_gpu_sequence.py.
"""
from __future__ import annotations

import pytest
import torch

import pathtile_b200 as pt
from oracle import sequence as ref
from pathtile_b200 import ops, s4conv
from test_gpu_sequence import BF16, F16, F32, Maker, close, lengths_of, scan_inputs, spoil

pytestmark = pytest.mark.gpu


# A backward block walks several rows where batch > 8 * 148 / (blocks of channels * pieces of the length).
@pytest.mark.parametrize("b,l,d,n,g,dtype,ragged", [
    (600, 20, 256, 16, 1, F32, False),  # 4 blocks of channels: 296 walkers for 600 rows
    (601, 19, 260, 16, 1, BF16, True),
    (700, 17, 200, 5, 2, F32, True),
    (500, 18, 160, 24, 1, F16, True),
    (300, 33, 96, 64, 2, F32, True),
])
def test_backward_blocks_that_walk_several_rows(cuda_device, b, l, d, n, g, dtype, ragged):
    m = Maker(cuda_device, 81)
    v = scan_inputs(m, b, l, d, n, g, dtype, True, True, True, True, False)
    dy, dlast = m(b, l, d, dtype=dtype), m(b, d, n)
    lengths = lengths_of(cuda_device, b, l) if ragged else None
    if ragged:
        v.update((k, spoil(v[k], lengths)) for k in ("x", "dt", "z", "B", "C"))
        dy = spoil(dy, lengths)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
    y, last = pt.selective_scan(**leaves, dt_softplus=True, lengths=lengths, return_final_state=True)
    grads = torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])
    clean = {k if k != "initial_state" else "state": t.nan_to_num(0, 0, 0) for k, t in v.items()}
    one, size = (ref.scan(**clean, softplus=True, lengths=lengths, dy=dy.nan_to_num(0, 0, 0), dlast=dlast, absolute=a)
                 for a in (False, True))
    links = 4 * l + n + 32
    close(y.detach(), one["y"], size["y"], links, "y")
    close(last.detach(), one["state"], size["state"], links, "state")
    for name, grad in zip(leaves, grads):
        name = "dstate" if name == "initial_state" else "d" + name
        over = {"dA": b * l / 8, "dD": b * l / 8, "ddt_bias": b * l / 8, "dB": d / g / 8, "dC": d / g / 8}.get(name, 0)
        close(grad, one[name], size[name], 2 * links + over, name)


@pytest.mark.parametrize("b,l,d,n,dtype", [(2, 300, 96, 64, F32), (1, 520, 40, 64, BF16), (3, 150, 33, 61, F32)])
def test_many_states_backward_over_long_rows(cuda_device, b, l, d, n, dtype):
    m = Maker(cuda_device, 82)
    v = scan_inputs(m, b, l, d, n, 1, dtype, True, False, True, True, False)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    dy, dlast = m(b, l, d, dtype=dtype), m(b, d, n)
    y, last = pt.selective_scan(**leaves, dt_softplus=True, return_final_state=True)
    grads = torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])
    plain = {k if k != "initial_state" else "state": t for k, t in v.items()}
    one, size = (ref.scan(**plain, softplus=True, dy=dy, dlast=dlast, absolute=a) for a in (False, True))
    links = 4 * l + n + 32
    close(y.detach(), one["y"], size["y"], links, "y")
    for name, grad in zip(leaves, grads):
        name = "dstate" if name == "initial_state" else "d" + name
        over = {"dA": b * l / 8, "dD": b * l / 8, "ddt_bias": b * l / 8, "dB": d / 8, "dC": d / 8}.get(name, 0)
        close(grad, one[name], size[name], 2 * links + over, name)


def test_the_model_with_its_own_number_of_states(cuda_device):
    """64 states, the model's default, in every block: a training step's gradients are finite and reach every block."""
    torch.manual_seed(9)
    model = s4conv.Model(hidden_dim=32, num_blocks=2, block="selective").to(cuda_device)
    x, target = s4conv.synthetic_batch(16, device=cuda_device, seed=2)
    assert torch.isfinite(s4conv.train_step(model, s4conv.make_optimizer(model), x, target))
    assert all(p.grad.isfinite().all() and p.grad.any() for p in model.blocks[0].parameters())


# ---------------------------------------------------------------- single tokens
# A step runs blocks of four warps where lanes * batch >= 512 * 148.
@pytest.mark.parametrize("b,d,n,g,dtype", [(256, 2048, 16, 1, BF16), (300, 1030, 16, 2, F32), (257, 640, 24, 1, F16),
                                           (310, 900, 5, 3, F32), (270, 1025, 8, 1, BF16), (129, 513, 64, 1, F32)])
def test_steps_of_many_rows(cuda_device, b, d, n, g, dtype):
    m = Maker(cuda_device, 83)
    v = scan_inputs(m, b, 1, d, n, g, dtype, True, True, True, True, False)
    rows = b + 17
    gen = torch.Generator().manual_seed(4)
    slots = torch.randperm(rows, generator=gen)[:b].to(torch.int32).to(cuda_device)
    cache = m(rows, d, n)
    cache[slots.long()] = v["initial_state"]
    before = cache.clone()
    now = {k: v[k][:, 0] for k in ("x", "dt", "B", "C", "z")}
    y = pt.selective_scan_step(cache, **now, A=v["A"], D=v["D"], dt_bias=v["dt_bias"], dt_softplus=True, slots=slots)
    plain = {k if k != "initial_state" else "state": t for k, t in v.items()}
    one, size = (ref.scan(**plain, softplus=True, absolute=a) for a in (False, True))
    close(y, one["y"][:, 0], size["y"][:, 0], 4 + n + 32, "y")
    close(cache[slots.long()], one["state"], size["state"], 4 + n + 32, "state")
    rest = torch.ones(rows, dtype=torch.bool, device=cuda_device)
    rest[slots.long()] = False
    assert torch.equal(cache[rest], before[rest])
    assert ops.device_error() == 0


@pytest.mark.parametrize("b,d", [(400, 24), (520, 1100)])
def test_a_slot_named_far_apart(cuda_device, b, d):
    """The second row of a pair is refused, whatever warp or trip of the search meets the first."""
    m = Maker(cuda_device, 84)
    slots = torch.arange(b, dtype=torch.int32)
    pairs = [(0, 1), (2, 2 + 31), (3, 3 + 32), (4, 4 + 127), (5, 5 + 128), (6, 6 + 129), (40, 40 + 256), (90, 90 + 300),
             (10, b - 1), (b - 3, b - 2)]
    refused = set()
    for first, second in pairs:
        slots[second] = slots[first]
        refused.add(second)
    slots[7] = -1
    keep = torch.tensor([i not in refused and i != 7 for i in range(b)], device=cuda_device)
    at = slots.to(cuda_device)[keep].long()
    x, w, window = m(b, d, dtype=BF16), m(d, 4), m(b, 3, d, dtype=BF16)
    after = window.clone()
    y = pt.causal_conv_step(after, x, w, slots=slots.to(cuda_device))
    alone = window[at].clone()
    assert torch.equal(y[keep], pt.causal_conv_step(alone, x[keep], w)) and not y[~keep].any()
    assert torch.equal(after[at], alone)
    v = scan_inputs(m, b, 1, d, 16, 1, BF16, True, True, True, True, False)
    cache = v.pop("initial_state")
    now = {k: t[:, 0] if k in ("x", "dt", "B", "C", "z") else t for k, t in v.items()}
    after = cache.clone()
    y = pt.selective_scan_step(after, **now, dt_softplus=True, slots=slots.to(cuda_device))
    alone = cache[at].clone()
    mine = {k: t[keep] if k in ("x", "dt", "B", "C", "z") else t for k, t in now.items()}
    assert torch.equal(y[keep], pt.selective_scan_step(alone, **mine, dt_softplus=True)) and not y[~keep].any()
    assert torch.equal(after[at], alone)
    untouched = torch.ones(b, dtype=torch.bool, device=cuda_device)
    untouched[at] = False
    assert torch.equal(after[untouched], cache[untouched])
    assert ops.device_error(clear=True) == 256


# ---------------------------------------------------------------- norms in single elements, 2049 to 4096 wide
@pytest.mark.parametrize("rows,d,groups,dtype,rdtype,gate,scale", [
    (5, 2051, 1, BF16, None, True, False), (7, 4095, 1, F32, F32, False, True), (3, 3001, 1, F16, F32, True, True),
    (4, 2 * 2049, 2, BF16, None, False, False), (400, 2051, 1, BF16, F32, False, False), (2, 4097, 1, F32, None, True, False),
    (2, 5120, 1, BF16, None, True, False), (300, 8192, 1, BF16, None, True, False), (2, 16384, 1, F16, F16, False, True),
])
def test_wide_norms(cuda_device, rows, d, groups, dtype, rdtype, gate, scale):
    m = Maker(cuda_device, 85)
    v = dict(x=m(rows, d, dtype=dtype), weight=m(d, mean=1.0), gate=m(rows, d, dtype=dtype) if gate else None,
             residual=m(rows, d, dtype=rdtype, std=2.0) if rdtype else None, scale=m(d) if scale else None)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    got = pt.fused_norm(**leaves, groups=groups)
    outs = got if rdtype else (got,)
    given = [m(rows, d, dtype=dtype)] + ([m(rows, d, dtype=rdtype)] if rdtype else [])
    grads = torch.autograd.grad(outs, list(leaves.values()), given)
    kw = dict(groups=groups, eps=1e-5, dy=given[0], dr=given[1] if rdtype else None, r=outs[1].detach() if rdtype else None)
    one, size = (ref.norm(**v, **kw, absolute=a) for a in (False, True))
    close(outs[0].detach(), one["y"], size["y"], 40, "y")
    for name, grad in zip(leaves, grads):
        over = rows / 8 if name in ("weight", "scale") else 0
        close(grad, one["d" + name], size["d" + name], 80 + over, "d" + name)


# ---------------------------------------------------------------- streams and graphs
def _conv_set(device, seed, b=3, l=500, d=96):
    m = Maker(device, seed)
    v = dict(x=m(b, l, d, dtype=BF16), weight=m(d, 4), bias=m(d), initial_state=m(b, 3, d, dtype=BF16))
    return {k: t.requires_grad_() for k, t in v.items()}, [m(b, l, d, dtype=BF16), m(b, 3, d, dtype=BF16)]


def _conv_pass(v, given):
    outs = pt.causal_conv(**v, silu=True, return_final_state=True)
    return [*(t.detach() for t in outs), *torch.autograd.grad(outs, list(v.values()), given)]


def _norm_set(device, seed, rows=700, d=264):
    m = Maker(device, seed)
    v = dict(x=m(rows, d, dtype=BF16), weight=m(d), gate=m(rows, d, dtype=BF16), residual=m(rows, d), scale=m(d))
    return {k: t.requires_grad_() for k, t in v.items()}, [m(rows, d, dtype=BF16), m(rows, d)]


def _norm_pass(v, given):
    outs = pt.fused_norm(**v)
    return [*(t.detach() for t in outs), *torch.autograd.grad(outs, list(v.values()), given)]


KINDS = {"conv": (_conv_set, _conv_pass), "norm": (_norm_set, _norm_pass)}


@pytest.mark.parametrize("kind", KINDS)
def test_training_passes_on_two_streams_at_once(cuda_device, kind):
    make, run = KINDS[kind]
    sets = [make(cuda_device, s) for s in (91, 92)]
    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream(cuda_device) for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(run(*s))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(outs, want[i % 2], strict=True))


@pytest.mark.parametrize("kind", KINDS)
def test_training_passes_in_two_captured_graphs(cuda_device, kind):
    """Replayed at the same time on new inputs: each has a workspace of its own."""
    make, run = KINDS[kind]
    sets = [make(cuda_device, s) for s in (93, 94)]
    side = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(side):
        for s in sets:
            run(*s)
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run(*s)
        graphs.append((g, outs))
    fresh = [make(cuda_device, s) for s in (95, 96)]
    with torch.no_grad():
        for (v, given), (nv, ngiven) in zip(sets, fresh):
            for old, new in zip([*v.values(), *given], [*nv.values(), *ngiven]):
                old.copy_(new)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in graphs]
    for _ in range(3):
        for (g, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for (_, outs), s in zip(graphs, fresh):
        assert all(torch.equal(p, q) for p, q in zip(outs, run(*s), strict=True))
