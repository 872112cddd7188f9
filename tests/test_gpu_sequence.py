"""GPU: the sequence operators against their FP64 definitions (oracle/sequence.py).

Tolerances.  An output of a type with machine epsilon e is rounded once: off by
e/2 of its value (fp16 below its normal range: 2^-25).  Before that, everything
is computed in fp32 from products and sums; an error is measured against the
same sums with every term's absolute value (``absolute=True``).  An elementary
operation adds 2^-24, the exponentials, quotients and square roots a few of
those: 2^-22 covers each.  The longest chain of operations that an output depends
on gives the factor: a scan step costs three operations (decay, product, sum)
whose errors the later steps carry on, and decays of exp(-8) or more count, so a
chain over L steps and N states has 4 L + N + 32 links; gradients run through it
twice; sums over rows and steps (fp32, up to one link per 8 terms: they are
added in blocks) come on top.
"""
from __future__ import annotations

import pytest
import torch

import pathtile_b200 as pt
from oracle import sequence as ref
from pathtile_b200 import ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = 2.0 ** -22


def close(got, want, size, links, what=""):
    """|got - want| within one rounding of got's type and `links` fp32 operations on terms of total size `size`."""
    assert got.shape == want.shape, what
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    tiny = 2.0 ** -25 if got.dtype == F16 else 1e-37
    room = half * want.abs() + (1 + half) * links * UNIT * size.abs() + tiny
    off = (got.double() - want).abs()
    bad = ~(off <= room)  # NaN is bad
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by "
                           f"{float((off / room).nan_to_num(nan=9e9).max()):.3g} times the room")


class Maker:
    def __init__(self, device, seed):
        self.device, self.gen = device, torch.Generator(device=device).manual_seed(seed)

    def __call__(self, *shape, dtype=F32, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=self.gen, device=self.device) * std + mean).to(dtype)

    def strided(self, *shape, dtype=F32, pad=3):
        """A slice of something wider: rows that are not one behind the other (and not aligned)."""
        wide = self(*shape[:-1], shape[-1] + 2 * pad, dtype=dtype)
        return wide[..., pad:pad + shape[-1]]


def lengths_of(device, b, length):
    """Full, empty, negative (as empty), past the end (as full) and partial rows."""
    n = [length, 0, -3, length + 5, max(1, length // 2), 1, max(0, length - 1)]
    return torch.tensor([n[i % len(n)] for i in range(b)], dtype=torch.int32, device=device)


def spoil(t, lengths):
    """NaN and infinities behind every row's end."""
    t = t.clone()
    for i, n in enumerate(lengths.tolist()):
        n = max(0, n)
        t[i, n:] = float("nan")
        t[i, n + 1:] = float("inf")
    return t


# ---------------------------------------------------------------- causal convolution
CONV = [
    # b, l, d, taps, dtype, parameters' dtype, bias, silu, state, ragged, strided
    (2, 37, 64, 4, BF16, F32, True, True, True, False, False),
    (1, 1, 1, 1, F32, F32, False, False, False, False, False),
    (1, 1, 8, 4, F32, F32, True, True, False, False, False),
    (7, 19, 33, 3, F16, F16, True, True, True, True, False),
    (7, 5, 130, 8, BF16, BF16, True, False, True, True, True),
    (3, 2, 16, 4, F32, F32, False, True, True, False, True),
    (2, 300, 258, 2, F16, F32, True, True, False, True, False),
    (5, 64, 48, 5, F32, F32, True, True, False, True, False),
    (1, 1000, 24, 6, BF16, F32, True, True, True, False, False),
    (300, 4, 12, 7, F32, F32, True, False, True, False, False),
    (2, 0, 8, 4, F32, F32, True, True, True, False, False),
    (0, 5, 8, 4, F32, F32, True, True, True, False, False),
]


@pytest.mark.parametrize("b,l,d,k,dtype,pdtype,bias,silu,state,ragged,strided", CONV)
def test_causal_conv(cuda_device, b, l, d, k, dtype, pdtype, bias, silu, state, ragged, strided):
    m = Maker(cuda_device, 11)
    x = m.strided(b, l, d, dtype=dtype) if strided else m(b, l, d, dtype=dtype)
    w = m(d, k, dtype=pdtype, std=k ** -0.5)
    bias = m(d, dtype=pdtype) if bias else None
    state = m(b, k - 1, d, dtype=dtype) if state else None
    lengths = lengths_of(cuda_device, b, l) if ragged else None
    x = spoil(x, lengths) if ragged and not strided else x
    dy = m.strided(b, l, d, dtype=dtype) if strided else m(b, l, d, dtype=dtype)
    dlast = m(b, k - 1, d, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, bias, state) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, bias, state)]
    kw = dict(silu=silu, lengths=lengths, return_final_state=True)
    y, last = pt.causal_conv(args[0], args[1], args[2], initial_state=args[3], **kw)
    grads = torch.autograd.grad([y, last], leaves, [dy, dlast])
    with torch.no_grad():
        y2, last2 = pt.causal_conv(x, w, bias, initial_state=state, **kw)
    assert torch.equal(y2, y) and torch.equal(last2, last)
    if b == 0:
        assert y.shape == x.shape and all(not g.any() for g in grads)
        return
    clean = x.nan_to_num(0, 0, 0) if ragged else x
    one, size = (ref.conv(clean, w, bias, silu, state, lengths, dy, dlast, absolute=a) for a in (False, True))
    close(y.detach(), one["y"], size["y"], k + 16, "y")
    assert torch.equal(last.double(), one["state"])
    names = [n for n, t in zip(("dx", "dweight", "dbias", "dstate"), (x, w, bias, state)) if t is not None]
    for name, grad in zip(names, grads):
        close(grad, one[name], size[name], 2 * k + 32 + (b * l / 8 if name in ("dweight", "dbias") else 0), name)


@pytest.mark.parametrize("b,d,k,dtype,silu", [(1, 64, 4, BF16, True), (5, 33, 3, F32, True), (9, 2050, 4, F16, False),
                                              (3, 8, 1, F32, True), (4, 1024, 8, BF16, True)])
def test_causal_conv_step_continues_a_prompt(cuda_device, b, d, k, dtype, silu):
    m = Maker(cuda_device, 12)
    x, w, bias = m(b, 9, d, dtype=dtype), m(d, k), m(d)
    whole, end = pt.causal_conv(x, w, bias, silu=silu, return_final_state=True)
    _, state = pt.causal_conv(x[:, :4], w, bias, silu=silu, return_final_state=True)
    for t in range(4, 9):
        y = pt.causal_conv_step(state, x[:, t], w, bias, silu=silu)
        assert torch.equal(y, whole[:, t])
    assert torch.equal(state, end)


# ---------------------------------------------------------------- selective scan
SCAN = [
    # b, l, d, n, g, dtype, D, z, bias, softplus, state, ragged, strided
    (2, 33, 64, 16, 1, BF16, True, True, True, True, False, False, False),
    (1, 1, 1, 1, 1, F32, False, False, False, False, False, False, False),
    (1, 1, 64, 16, 1, F32, True, True, True, True, True, False, False),
    (7, 17, 130, 16, 1, F32, True, True, True, True, True, True, False),
    (7, 16, 66, 3, 2, F16, True, True, True, True, True, True, True),
    (2, 15, 40, 8, 4, F32, True, False, False, True, True, False, True),
    (3, 47, 33, 9, 1, BF16, False, True, True, True, False, True, True),
    (2, 200, 96, 24, 3, F32, True, True, True, True, True, True, False),  # several segments
    (1, 333, 70, 16, 1, BF16, True, True, False, True, True, False, False),
    (1, 130, 64, 64, 2, F32, True, True, True, True, True, False, False),
    (2, 80, 20, 33, 1, F32, False, True, True, True, False, False, True),
    (4, 70, 7, 5, 7, F16, True, False, True, True, True, True, False),
    (70, 20, 64, 16, 1, F32, True, True, True, True, False, False, False),  # many rows: blocks that walk several
    (2, 0, 8, 4, 1, F32, True, True, True, True, True, False, False),
    (0, 4, 8, 4, 1, F32, True, True, True, True, True, False, False),
]


def scan_inputs(m, b, l, d, n, g, dtype, D, z, bias, state, strided):
    make = (lambda *s: m.strided(*s, dtype=dtype)) if strided else (lambda *s: m(*s, dtype=dtype))
    v = dict(x=make(b, l, d), dt=make(b, l, d), A=-torch.exp(m(d, n, std=0.7)), B=make(b, l, g, n), C=make(b, l, g, n))
    v["D"] = m(d) if D else None
    v["z"] = make(b, l, d) if z else None
    v["dt_bias"] = m(d, std=0.5, mean=-1.0) if bias else None
    v["initial_state"] = m(b, d, n) if state else None
    return v


@pytest.mark.parametrize("b,l,d,n,g,dtype,D,z,bias,softplus,state,ragged,strided", SCAN)
def test_selective_scan(cuda_device, b, l, d, n, g, dtype, D, z, bias, softplus, state, ragged, strided):
    m = Maker(cuda_device, 21)
    v = scan_inputs(m, b, l, d, n, g, dtype, D, z, bias, state, strided)
    lengths = lengths_of(cuda_device, b, l) if ragged else None
    if ragged:
        for k in ("x", "dt", "z", "B", "C"):
            v[k] = spoil(v[k], lengths) if v[k] is not None else None
    if not softplus:
        v["dt"] = v["dt"].abs() * 0.2
    dy, dlast = m(b, l, d, dtype=dtype), m(b, d, n)
    if ragged:
        dy = spoil(dy, lengths)
    v = {k: t.detach().requires_grad_() if t is not None else None for k, t in v.items()}
    kw = dict(dt_softplus=softplus, lengths=lengths, return_final_state=True)
    y, last = pt.selective_scan(**v, **kw)
    leaves = {k: t for k, t in v.items() if t is not None}
    grads = torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])
    with torch.no_grad():
        y2, last2 = pt.selective_scan(**v, **kw)
    assert torch.equal(y2, y) and torch.equal(last2, last)
    if b == 0:
        assert y.shape == v["x"].shape and all(not t.any() for t in grads)
        return
    v["state"] = v.pop("initial_state")
    clean = {k: t.detach().nan_to_num(0, 0, 0) if t is not None else None for k, t in v.items()}
    one, size = (ref.scan(**clean, softplus=softplus, lengths=lengths, dy=dy.nan_to_num(0, 0, 0), dlast=dlast, absolute=a)
                 for a in (False, True))
    links = 4 * l + n + 32
    close(y.detach(), one["y"], size["y"], links, "y")
    close(last.detach(), one["state"], size["state"], links, "state")
    for name, grad in zip(leaves, grads):
        name = "dstate" if name == "initial_state" else "d" + name
        over = {"dA": b * l / 8, "dD": b * l / 8, "ddt_bias": b * l / 8, "dB": d / g / 8, "dC": d / g / 8}.get(name, 0)
        close(grad, one[name], size[name], 2 * links + over, name)


def test_selective_scan_takes_operands_without_groups_and_any_layout(cuda_device):
    m = Maker(cuda_device, 22)
    v = scan_inputs(m, 2, 40, 32, 16, 1, F32, True, True, True, False, False)
    want = pt.selective_scan(**v, dt_softplus=True)
    v["B"], v["C"] = v["B"][:, :, 0], v["C"][:, :, 0]
    assert torch.equal(pt.selective_scan(**v, dt_softplus=True), want)
    # Channels that are not contiguous are copied; a batch stride of 0 is read as it is.
    v["x"] = v["x"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(pt.selective_scan(**v, dt_softplus=True), want)
    row = v["z"][:1]
    same = pt.selective_scan(**{**v, "z": row.expand(2, -1, -1)}, dt_softplus=True)
    assert torch.equal(same, pt.selective_scan(**{**v, "z": row.repeat(2, 1, 1)}, dt_softplus=True))


def test_gradients_of_a_broadcast_input_and_of_one_output(cuda_device):
    m = Maker(cuda_device, 23)
    v = scan_inputs(m, 3, 20, 16, 8, 1, F32, True, True, True, False, False)
    x = v["x"][:1].clone().requires_grad_()
    dy = m(3, 20, 16)
    y = pt.selective_scan(**{**v, "x": x.expand(3, -1, -1)}, dt_softplus=True)
    grad, = torch.autograd.grad(y, x, dy)
    full = v["x"][:1].repeat(3, 1, 1).requires_grad_()
    each, = torch.autograd.grad(pt.selective_scan(**{**v, "x": full}, dt_softplus=True), full, dy)
    torch.testing.assert_close(grad, each.sum(0, keepdim=True))
    # Only the final state is used; only one operand needs a gradient; the gradient of a sum has strides of 0.
    B = v["B"].clone().requires_grad_()
    _, last = pt.selective_scan(**{**v, "B": B}, dt_softplus=True, return_final_state=True)
    only, = torch.autograd.grad(last.sum(), B)
    clean = {k: t for k, t in v.items() if k != "initial_state"}
    one, size = (ref.scan(**clean, softplus=True, dy=torch.zeros_like(dy), dlast=torch.ones_like(last), absolute=a)
                 for a in (False, True))
    close(only, one["dB"], size["dB"], 2 * (80 + 8 + 32) + 2, "dB")
    total, = torch.autograd.grad(pt.selective_scan(**{**v, "B": B}, dt_softplus=True).sum(), B)
    one, size = (ref.scan(**clean, softplus=True, dy=torch.ones_like(dy), absolute=a) for a in (False, True))
    close(total, one["dB"], size["dB"], 2 * (80 + 8 + 32) + 2, "dB of a sum")


def test_backward_is_the_same_twice_and_once_differentiable(cuda_device):
    m = Maker(cuda_device, 24)
    v = scan_inputs(m, 4, 150, 96, 16, 1, BF16, True, True, True, False, False)
    v = {k: t.requires_grad_() for k, t in v.items() if t is not None}
    dy = m(4, 150, 96, dtype=BF16)
    first, second = (torch.autograd.grad(pt.selective_scan(**v, dt_softplus=True), list(v.values()), dy) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    y = pt.selective_scan(**v, dt_softplus=True)
    grad, = torch.autograd.grad(y, v["x"], dy, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("b,d,n,g,dtype", [(1, 64, 16, 1, BF16), (5, 33, 3, 3, F32), (9, 130, 24, 2, F16), (3, 8, 64, 1, F32),
                                           (2, 7, 1, 1, F32), (4, 2048, 16, 1, BF16)])
def test_selective_scan_step_continues_a_prompt(cuda_device, b, d, n, g, dtype):
    m = Maker(cuda_device, 25)
    v = scan_inputs(m, b, 6, d, n, g, dtype, True, True, True, True, False)
    one, size = (ref.scan(**{k if k != "initial_state" else "state": t for k, t in v.items()}, softplus=True, absolute=a)
                 for a in (False, True))
    _, state = pt.selective_scan(**{k: t[:, :2] if k in ("x", "dt", "B", "C", "z") else t for k, t in v.items()},
                                 dt_softplus=True, return_final_state=True)
    for t in range(2, 6):
        now = {k: v[k][:, t] for k in ("x", "dt", "B", "C", "z")}
        y = pt.selective_scan_step(state, **now, A=v["A"], D=v["D"], dt_bias=v["dt_bias"], dt_softplus=True)
        close(y, one["y"][:, t], size["y"][:, t], 4 * t + n + 32, f"y at {t}")
    close(state, one["state"], size["state"], 4 * 6 + n + 32, "state")


def test_steps_behind_a_rows_end_leave_its_state_as_it_is(cuda_device):
    """Bit for bit, over thousands of them: the state of a padded row is that of the row alone (from zero: a long
    call joins pieces, and adds an initial state in another order), and an empty row's the initial one."""
    m = Maker(cuda_device, 26)
    for length, used in ((4000, 3), (4000, 0), (70, 33), (20, 7), (20, 0)):
        v = scan_inputs(m, 1, length, 16, 16, 1, F32, True, True, True, used == 0, False)
        v["A"][0] = 0.0
        lengths = torch.tensor([used], dtype=torch.int32, device=cuda_device)
        _, padded = pt.selective_scan(**v, dt_softplus=True, return_final_state=True, lengths=lengths)
        short = {k: t[:, :used] if k in ("x", "dt", "B", "C", "z") else t for k, t in v.items()}
        _, alone = pt.selective_scan(**short, dt_softplus=True, return_final_state=True)
        assert torch.equal(padded, alone)
        if used == 0:
            assert torch.equal(padded, v["initial_state"])


# ---------------------------------------------------------------- slots
def _step_both(device, slots, rows, d=40, n=16, k=4):
    """Both step forms with these slots; returns (cache before, cache after, y, row b's y were it alone) for each."""
    m = Maker(device, 31)
    b = len(slots)
    slots = torch.tensor(slots, dtype=torch.int32, device=device)
    got = []
    cache, x, w = m(rows, k - 1, d, dtype=BF16), m(b, d, dtype=BF16), m(d, k)
    after = cache.clone()
    y = pt.causal_conv_step(after, x, w, slots=slots)
    alone = []
    for i, s in enumerate(slots.tolist()):
        one = cache[s:s + 1].clone() if 0 <= s < rows else torch.zeros_like(cache[:1])
        alone.append((pt.causal_conv_step(one, x[i:i + 1], w)[0], one[0]))
    got.append((cache, after, y, alone))
    cache = m(rows, d, n)
    v = scan_inputs(m, b, 1, d, n, 1, F32, True, True, True, False, False)
    v.pop("initial_state")
    now = {key: t[:, 0] if key in ("x", "dt", "B", "C", "z") else t for key, t in v.items()}
    after = cache.clone()
    y = pt.selective_scan_step(after, **now, dt_softplus=True, slots=slots)
    alone = []
    for i, s in enumerate(slots.tolist()):
        one = cache[s:s + 1].clone() if 0 <= s < rows else torch.zeros_like(cache[:1])
        mine = {key: t[i:i + 1] if key in ("x", "dt", "B", "C", "z") else t for key, t in now.items()}
        alone.append((pt.selective_scan_step(one, **mine, dt_softplus=True)[0], one[0]))
    got.append((cache, after, y, alone))
    return got


def test_slots_padding_rows_and_rows_left_alone(cuda_device):
    slots = [5, -1, 0, 7, -9, 2]
    for cache, after, y, alone in _step_both(cuda_device, slots, 9):
        for i, s in enumerate(slots):
            if s < 0:
                assert not y[i].any()
            else:
                assert torch.equal(y[i], alone[i][0]) and torch.equal(after[s], alone[i][1])
        for s in set(range(9)) - set(slots):
            assert torch.equal(after[s], cache[s])
    assert ops.device_error() == 0


@pytest.mark.parametrize("slots,bit", [([3, 9, 1], 128), ([3, 1, 3, 0, 3], 256), ([2 ** 31 - 1, 1], 128)])
def test_slots_past_the_cache_and_named_twice_are_refused(cuda_device, slots, bit):
    for cache, after, y, alone in _step_both(cuda_device, slots, 9):
        seen = set()
        for i, s in enumerate(slots):
            if s >= 9 or s in seen:
                assert not y[i].any()
            else:
                assert torch.equal(y[i], alone[i][0]) and torch.equal(after[s], alone[i][1])
            seen.add(s)
        for s in set(range(9)) - seen:
            assert torch.equal(after[s], cache[s])
    assert ops.device_error(clear=True) == bit


def test_a_step_counts_as_a_change_of_its_cache(cuda_device):
    """Autograd sees that a saved cache was changed, and a cache that asks for a gradient is refused."""
    m = Maker(cuda_device, 34)
    state, x, w = m(2, 3, 8), m(2, 8), m(8, 4)
    leaf = m(2, 3, 8).requires_grad_()
    product = (leaf * state).sum()  # saves state
    pt.causal_conv_step(state, x, w)
    with pytest.raises(RuntimeError, match="inplace"):
        product.backward()
    with pytest.raises(ValueError, match="no_grad"):
        pt.causal_conv_step(state.requires_grad_(), x, w)


def test_offsets_past_32_bits(cuda_device):
    """A cache whose last rows lie more than 2^32 bytes and 2^31 elements in, and one layer's rows of it."""
    d, n, rows = 1024, 64, 33000
    cache = torch.empty(rows, 1, d, n, device=cuda_device)[:, 0]
    m = Maker(cuda_device, 33)
    v = scan_inputs(m, 2, 1, d, n, 1, F32, True, True, True, False, False)
    v.pop("initial_state")
    now = {key: t[:, 0] if key in ("x", "dt", "B", "C", "z") else t for key, t in v.items()}
    small = m(2, d, n)
    slots = torch.tensor([rows - 1, 0], dtype=torch.int32, device=cuda_device)
    cache[rows - 1], cache[0] = small[0], small[1]
    y = pt.selective_scan_step(cache, **now, dt_softplus=True, slots=slots)
    want = pt.selective_scan_step(small, **now, dt_softplus=True)
    assert torch.equal(y, want) and torch.equal(cache[rows - 1], small[0]) and torch.equal(cache[0], small[1])


def test_tensors_of_more_than_two_billion_elements(cuda_device):
    """The far end of operands past 2^31 elements, forward and backward: what a short call on the last steps gives
    (the scan forgets the earlier ones: 100 steps of decay e^-2 leave e^-200)."""
    l, d, n, end = 530_000, 4096, 4, 200
    m = Maker(cuda_device, 35)

    def big(*shape):
        return torch.randn(*shape, generator=m.gen, device=cuda_device, dtype=BF16)

    x, w, bias = big(1, l, d), m(d, 4), m(d)
    assert x.numel() > 2 ** 31
    leaf = x.requires_grad_()
    y = pt.causal_conv(leaf, w, bias, silu=True)
    dy = big(1, l, d)
    dx, = torch.autograd.grad(y, leaf, dy)
    tail = x[:, -end:].detach().clone().requires_grad_()
    want = pt.causal_conv(tail, w, bias, silu=True)
    dtail, = torch.autograd.grad(want, tail, dy[:, -end:])
    assert torch.equal(y[:, -end + 3:], want[:, 3:]) and torch.equal(dx[:, -end + 3:], dtail[:, 3:])
    del y, dx
    torch.cuda.empty_cache()

    rows = x.detach().view(l, d)
    gain = m(d).requires_grad_()
    y = pt.fused_norm(rows, gain, gate=dy.view(l, d))
    assert torch.equal(y[-9:], pt.fused_norm(rows[-9:].clone(), gain, gate=dy.view(l, d)[-9:].clone()))
    del y
    torch.cuda.empty_cache()

    A = torch.full((d, n), -2.0, device=cuda_device)
    B, C = m(1, l, n, dtype=BF16), m(1, l, n, dtype=BF16)
    dt = torch.ones((), dtype=BF16, device=cuda_device).expand(1, l, d)
    y, last = pt.selective_scan(leaf, dt, A, B, C, return_final_state=True)
    dx, = torch.autograd.grad(y, leaf, dy)
    part = [t[:, -end:] for t in (dt, B, C)]
    want, state = pt.selective_scan(tail, part[0], A, part[1], part[2], return_final_state=True)
    dtail, = torch.autograd.grad(want, tail, dy[:, -end:])
    # Both sides are rounded once to bf16: 2^-8 of the value each.
    for got, w in ((y[:, -100:], want[:, -100:]), (last, state), (dx[:, -100:], dtail[:, -100:])):
        torch.testing.assert_close(got, w, rtol=2.0 ** -7, atol=2.0 ** -7)


# ---------------------------------------------------------------- norm
NORM = [
    # shape, groups, dtype, residual's dtype, gate, scale, parameters' dtype
    ((5, 64), 1, F32, None, False, False, F32),
    ((1, 1), 1, F32, F32, True, True, F32),
    ((37, 1027), 1, BF16, F32, False, True, F32),
    ((9, 4096), 8, BF16, None, True, False, F32),
    ((3, 5, 96), 3, F16, F16, True, True, F16),
    ((600, 48), 1, BF16, BF16, False, False, BF16),
    ((2, 8192), 1, BF16, F32, False, False, F32),
    ((3, 20000), 1, F16, None, True, True, F32),
    ((2, 32768), 1, F32, F32, True, True, F32),
    ((2, 32768), 1, BF16, F32, True, True, F32),
    ((2, 10003), 1, F32, None, True, False, F32),
    ((3000, 256), 2, BF16, F32, True, True, F32),
    ((0, 64), 1, F32, F32, False, True, F32),
]


@pytest.mark.parametrize("shape,groups,dtype,rdtype,gate,scale,pdtype", NORM)
def test_fused_norm(cuda_device, shape, groups, dtype, rdtype, gate, scale, pdtype):
    m = Maker(cuda_device, 41)
    d = shape[-1]
    v = dict(x=m(*shape, dtype=dtype), weight=m(d, dtype=pdtype, mean=1.0), gate=m(*shape, dtype=dtype) if gate else None,
             residual=m(*shape, dtype=rdtype, std=2.0) if rdtype else None, scale=m(d, dtype=pdtype) if scale else None)
    v = {k: t.requires_grad_() if t is not None else None for k, t in v.items()}
    leaves = {k: t for k, t in v.items() if t is not None}
    got = pt.fused_norm(**v, groups=groups, eps=1e-4)
    y, r = got if rdtype else (got, None)
    assert y.dtype == dtype and y.shape == shape and (r is None or r.dtype == rdtype)
    dy, dr = m(*shape, dtype=dtype), m(*shape, dtype=rdtype) if rdtype else None
    grads = torch.autograd.grad([y, r] if rdtype else [y], list(leaves.values()), [dy, dr] if rdtype else [dy])
    with torch.no_grad():
        plain = pt.fused_norm(**v, groups=groups, eps=1e-4)
    for p, q in zip(plain if rdtype else (plain,), got if rdtype else (got,)):
        assert torch.equal(p, q)
    rows = y.numel() // d
    if rows == 0:
        assert all(not t.any() for t in grads)
        return
    flat = {k: t.detach().reshape(rows, d) if t is not None and k in ("x", "gate", "residual") else t for k, t in v.items()}
    kw = dict(groups=groups, eps=1e-4, dy=dy.view(rows, d), dr=dr.view(rows, d) if rdtype else None)
    first, fsize = (ref.norm(**flat, **kw, absolute=a) for a in (False, True))
    if rdtype:
        close(r.detach().view(rows, d), first["r"], fsize["r"], 8, "r")
    one, size = (ref.norm(**flat, **kw, r=r.detach().view(rows, d) if rdtype else None, absolute=a) for a in (False, True))
    links = 40  # sums over a row are trees; a row's statistics add a few operations to every element
    close(y.detach().view(rows, d), one["y"], size["y"], links, "y")
    for name, grad in zip(leaves, grads):
        over = rows / 8 if name in ("weight", "scale") else 0
        close(grad.view(-1, d) if name in ("x", "gate", "residual") else grad, one["d" + name], size["d" + name],
              2 * links + over, "d" + name)


def test_fused_norm_on_strided_rows(cuda_device):
    m = Maker(cuda_device, 42)
    both = m(6, 10, 2 * 65, dtype=BF16)
    x, gate = both[..., :65], both[..., 65:]  # halves of one projection, rows of odd width
    w = m(65, mean=1.0)
    assert torch.equal(pt.fused_norm(x, w, gate=gate), pt.fused_norm(x.contiguous(), w, gate=gate.contiguous()))
    cols = m(65, 12, dtype=BF16).t()
    assert torch.equal(pt.fused_norm(cols, w), pt.fused_norm(cols.contiguous(), w))
    leaf = m(1, 65).requires_grad_()
    grad, = torch.autograd.grad(pt.fused_norm(leaf.expand(8, 65), w).sum(), leaf)
    one = ref.norm(leaf, w, dy=torch.ones(1, 65, device=cuda_device))
    size = ref.norm(leaf, w, dy=torch.ones(1, 65, device=cuda_device), absolute=True)
    close(grad, 8 * one["dx"], 8 * size["dx"], 100, "dx")


# ---------------------------------------------------------------- alignment
def shifted(t):
    """The same values, contiguous, from the second element of a buffer on."""
    if t is None or t.dtype == torch.int32:
        return t
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = buf[1:].view(t.shape)
    out.copy_(t)
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_tensors_that_begin_at_an_odd_element(cuda_device, dtype):
    m = Maker(cuda_device, 45)
    b, l, d, n = 3, 21, 64, 16
    x, w, bias, state = m(b, l, d, dtype=dtype), m(d, 4), m(d), m(b, 3, d, dtype=dtype)
    dy, dlast = m(b, l, d, dtype=dtype), m(b, 3, d, dtype=dtype)

    def conv(args, grads):
        leaves = [t.detach().requires_grad_() for t in args]
        y, last = pt.causal_conv(*leaves[:3], silu=True, initial_state=leaves[3], return_final_state=True)
        return [y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, grads)]

    plain = conv((x, w, bias, state), (dy, dlast))
    every = (x, w, bias, state, dy, dlast)
    for i in range(len(every)):  # one at a time: one alone decides the width for all
        args = [shifted(t) if j == i else t for j, t in enumerate(every)]
        for p, q in zip(conv(args[:4], args[4:]), plain):
            torch.testing.assert_close(p, q, rtol=1e-5 if dtype == F32 else 1e-2, atol=1e-5 if dtype == F32 else 1e-2)
    one, two = state.clone(), shifted(state)
    assert torch.equal(pt.causal_conv_step(one, x[:, 0], w, bias), pt.causal_conv_step(two, shifted(x[:, 0]), shifted(w), shifted(bias)))
    assert torch.equal(one, two)

    v = scan_inputs(m, b, l, d, n, 1, dtype, True, True, True, True, False)
    gy, gl = m(b, l, d, dtype=dtype), m(b, d, n)

    def scan(v, grads):
        v = {k: t.detach().requires_grad_() for k, t in v.items()}
        y, last = pt.selective_scan(**v, dt_softplus=True, return_final_state=True)
        return [y.detach(), last.detach(), *torch.autograd.grad([y, last], list(v.values()), grads)]

    for p, q in zip(scan({k: shifted(t) for k, t in v.items()}, (shifted(gy), shifted(gl))), scan(v, (gy, gl))):
        assert torch.equal(p, q)
    now = {k: v[k][:, 0].contiguous() for k in ("x", "dt", "B", "C", "z")} | {k: v[k] for k in ("A", "D", "dt_bias")}
    one, two = v["initial_state"].clone(), shifted(v["initial_state"])
    assert torch.equal(pt.selective_scan_step(one, **now, dt_softplus=True),
                       pt.selective_scan_step(two, **{k: shifted(t) for k, t in now.items()}, dt_softplus=True))
    assert torch.equal(one, two)

    parts = dict(x=m(9, d, dtype=dtype), weight=m(d), gate=m(9, d, dtype=dtype), residual=m(9, d), scale=m(d))
    gy, gr = m(9, d, dtype=dtype), m(9, d)

    def norm(v, grads):
        v = {k: t.detach().requires_grad_() for k, t in v.items()}
        outs = pt.fused_norm(**v)
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, list(v.values()), grads)]

    plain = norm(parts, (gy, gr))
    for p, q in zip(norm({k: shifted(t) for k, t in parts.items()}, (shifted(gy), shifted(gr))), plain):
        torch.testing.assert_close(p, q, rtol=1e-5 if p.dtype == F32 else 1e-2, atol=1e-4 if p.dtype == F32 else 1e-2)


# ---------------------------------------------------------------- infinities and NaN
def test_infinities_and_nans_stay_in_their_channel(cuda_device):
    m = Maker(cuda_device, 51)
    for n in (16, 5):
        v = scan_inputs(m, 2, 24, 12, n, 1, F32, True, True, True, False, False)
        v["C"], v["B"] = v["C"].abs() + 0.1, v["B"].abs() + 0.1
        want = pt.selective_scan(**v, dt_softplus=True)
        x = v["x"].clone()
        x[0, 10, 3], x[1, 5, 7] = float("inf"), float("nan")
        got = pt.selective_scan(**{**v, "x": x}, dt_softplus=True)
        exact = ref.scan(**{k: t for k, t in {**v, "x": x}.items() if k != "initial_state"}, softplus=True)["y"]
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[0, 10:, 3], touched[1, 5:, 7] = True, True
        assert torch.equal(got[~touched], want[~touched])
        assert got[1, 5:, 7].isnan().all()
        assert torch.equal(got[0, 10:, 3].isinf(), exact[0, 10:, 3].isinf())
        assert torch.equal(got[0, 10:, 3].sign(), exact[0, 10:, 3].sign().float())
    x = m(2, 12, 8)
    w = m(8, 4)
    want = pt.causal_conv(x, w, silu=True)
    x[0, 3, 2] = float("inf")
    got = pt.causal_conv(x, w, silu=True)
    touched = torch.zeros_like(got, dtype=torch.bool)
    touched[0, 3:7, 2] = True
    assert torch.equal(got[~touched], want[~touched])
    rows = m(4, 64)
    want = pt.fused_norm(rows, torch.ones(64, device=cuda_device))
    rows[1, 5] = float("nan")
    got = pt.fused_norm(rows, torch.ones(64, device=cuda_device))
    assert got[1].isnan().all() and torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])


@pytest.mark.parametrize("l,n", [(20, 16), (50, 6), (300, 24)])
def test_an_empty_rows_state_reaches_no_sum(cuda_device, l, n):
    """What a row without valid steps carries from its initial to its final state, finite or not, is in no other
    row's gradient and in none that sums over rows."""
    m = Maker(cuda_device, 53)
    v = scan_inputs(m, 3, l, 24, n, 1, F32, True, True, True, True, False)
    w, window = m(24, 4), m(3, 3, 24)
    dy, dlast, dwindow = m(3, l, 24), m(3, 24, n), m(3, 3, 24)
    lengths = torch.tensor([l, 0, l // 3], dtype=torch.int32, device=cuda_device)

    def grads(state, dlast, window, dwindow):
        leaves = [t.detach().requires_grad_() for t in {**v, "initial_state": state}.values()]
        y, last = pt.selective_scan(**dict(zip(v, leaves)), dt_softplus=True, lengths=lengths, return_final_state=True)
        out = [y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, [dy, dlast])]
        leaves = [t.detach().requires_grad_() for t in (v["x"], w, window)]
        y, last = pt.causal_conv(*leaves[:2], initial_state=leaves[2], lengths=lengths, return_final_state=True)
        return [*out, y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, [dy, dwindow])]

    want = grads(v["initial_state"], dlast, window, dwindow)
    odd = [t.clone() for t in (v["initial_state"], dlast, window, dwindow)]
    for t in odd:
        t[1, ::2], t[1, 1::2] = float("nan"), float("inf")
    for i, (got, one) in enumerate(zip(grads(*odd), want, strict=True)):
        if got.shape[0] == 3 and not torch.isfinite(got).all():  # a state, or its gradient: as it came
            assert torch.equal(got[1].isnan(), odd[0 if got.shape == odd[0].shape else 2][1].isnan()), i
            got, one = got[[0, 2]], one[[0, 2]]
        assert torch.equal(got, one), i


def test_far_decays_and_large_steps(cuda_device):
    """Steps that forget everything, steps of no duration, and rates of zero."""
    m = Maker(cuda_device, 52)
    v = scan_inputs(m, 1, 40, 8, 16, 1, F32, False, False, False, True, False)
    v = {k: t for k, t in v.items() if t is not None}
    v["dt"] = torch.where(torch.arange(40, device=cuda_device)[:, None] % 3 == 0, 300.0, -90.0).expand(1, 40, 8).contiguous()
    v["A"][0] = 0.0
    y, last = pt.selective_scan(**v, dt_softplus=True, return_final_state=True)
    v["state"] = v.pop("initial_state")
    one, size = (ref.scan(**v, softplus=True, absolute=a) for a in (False, True))
    close(y, one["y"], size["y"], 4 * 40 + 16 + 32, "y")
    close(last, one["state"], size["state"], 4 * 40 + 16 + 32, "state")


# ---------------------------------------------------------------- streams, graphs
def _train_once(v, dy):
    y = pt.selective_scan(**v, dt_softplus=True)
    return [y.detach(), *torch.autograd.grad(y, [t for t in v.values() if t.requires_grad], dy)]


def _train_inputs(device, seed, d=64, l=150):
    m = Maker(device, seed)
    v = scan_inputs(m, 2, l, d, 16, 1, BF16, True, True, True, False, False)
    return {k: t.requires_grad_() for k, t in v.items() if t is not None}, m(2, l, d, dtype=BF16)


def test_calls_on_two_streams_at_once(cuda_device):
    sets = [_train_inputs(cuda_device, s) for s in (61, 62)]
    want = [_train_once(*s) for s in sets]
    streams = [torch.cuda.Stream(cuda_device) for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(_train_once(*s))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(outs, want[i % 2]))


def test_two_captured_graphs_have_their_own_workspaces(cuda_device):
    """Forward and backward in graphs, replayed at the same time on new inputs."""
    sets = [_train_inputs(cuda_device, s) for s in (63, 64)]
    side = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(side):
        for s in sets:
            _train_once(*s)
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = _train_once(*s)
        graphs.append((g, outs))
    fresh = [_train_inputs(cuda_device, s) for s in (65, 66)]
    with torch.no_grad():
        for (v, dy), (nv, ndy) in zip(sets, fresh):
            dy.copy_(ndy)
            for k in v:
                v[k].copy_(nv[k])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in graphs]
    for _ in range(3):
        for (g, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for (_, outs), s in zip(graphs, fresh):
        assert all(torch.equal(p, q) for p, q in zip(outs, _train_once(*s)))


def test_captured_steps_and_a_cache_that_moves_on(cuda_device):
    m = Maker(cuda_device, 67)
    v = scan_inputs(m, 3, 1, 64, 16, 1, BF16, True, True, True, False, False)
    v.pop("initial_state")
    now = {k: t[:, 0].contiguous() if k in ("x", "dt", "B", "C", "z") else t for k, t in v.items()}
    slots = torch.tensor([4, 0, -1], dtype=torch.int32, device=cuda_device)
    w, bias = m(64, 4), m(64)
    first, window = m(6, 64, 16), m(6, 3, 64, dtype=BF16)

    def step(cache, win):
        with torch.no_grad():
            x = pt.causal_conv_step(win, now["x"], w, bias, silu=True, slots=slots)
            return pt.selective_scan_step(cache, **{**now, "x": x}, dt_softplus=True, slots=slots)

    cache, win = first.clone(), window.clone()
    want = [step(cache, win).clone() for _ in range(3)]
    c2, w2 = first.clone(), window.clone()
    step(c2, w2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step(c2, w2)
    c2.copy_(first)
    w2.copy_(window)
    for i in range(3):
        g.replay()
        assert torch.equal(y, want[i])
    assert torch.equal(c2, cache) and torch.equal(w2, win)


# ---------------------------------------------------------------- refusals
def test_refusals(cuda_device):
    m = Maker(cuda_device, 71)
    v = scan_inputs(m, 2, 5, 8, 4, 2, F32, True, True, True, True, False)
    good = dict(v)
    pt.selective_scan(**good)
    for name, bad in [("x", v["x"].double()), ("x", v["x"][0]), ("dt", v["dt"].half()), ("dt", v["dt"][:, :4]),
                      ("A", v["A"].double()), ("A", v["A"][:4]), ("A", m(8, 65)), ("A", m(8, 0)), ("B", v["B"].bfloat16()),
                      ("B", v["B"][:, :, :1]), ("B", m(2, 5, 3, 4)), ("C", v["C"][..., :3]), ("C", v["C"].cpu()),
                      ("D", v["D"].half()), ("D", v["D"][:4]), ("z", v["z"][:1]), ("dt_bias", v["dt_bias"].cpu()),
                      ("initial_state", v["initial_state"].bfloat16()), ("initial_state", v["initial_state"][:1]),
                      ("lengths", torch.zeros(2, dtype=torch.int64, device=cuda_device)),
                      ("lengths", torch.zeros(3, dtype=torch.int32, device=cuda_device)),
                      ("lengths", torch.zeros(2, dtype=torch.int32))]:
        with pytest.raises(ValueError):
            pt.selective_scan(**{**good, name: bad})
    x, w = m(2, 5, 8), m(8, 4)
    for args, kw in [((x, m(8, 9)), {}), ((x, m(7, 4)), {}), ((x, w.half()), {}), ((x, w, m(7)), {}),
                     ((x, w, m(8).half()), {}), ((x, w), dict(initial_state=m(2, 4, 8))), ((x[0], w), {}),
                     ((x, w), dict(initial_state=m(2, 3, 8).half())), ((x, w.cpu()), {})]:
        with pytest.raises(ValueError):
            pt.causal_conv(*args, **kw)
    state = m(4, 3, 8)
    for cache, kw in [(state, {}), (state.half(), {}), (state.transpose(1, 2), {}), (state[:1].expand(2, 3, 8), {}),
                      (state, dict(slots=torch.zeros(2, dtype=torch.int64, device=cuda_device))),
                      (state, dict(slots=torch.zeros(3, dtype=torch.int32, device=cuda_device)))]:
        with pytest.raises(ValueError):
            pt.causal_conv_step(cache, x[:, 0], w, **kw)
    with pytest.raises(ValueError, match="no_grad"):
        pt.causal_conv_step(state[:2].clone(), x[:, 0], w.requires_grad_())
    rows, one = m(3, 12), m(12)
    for args, kw in [((rows, one[:6]), {}), ((rows, one.half()), {}), ((rows, one), dict(gate=rows.half())),
                     ((rows, one), dict(residual=rows[:2])), ((rows, one), dict(residual=rows.half())),
                     ((rows, one), dict(scale=one.half())), ((rows, one), dict(groups=5)), ((rows, one), dict(groups=0)),
                     ((m(1, 32769), m(32769)), {}), ((rows, one.cpu()), {}), ((rows.double(), one.double()), {})]:
        with pytest.raises(ValueError):
            pt.fused_norm(*args, **kw)
