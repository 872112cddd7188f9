"""Sequence operators of a selective state space block, on the native kernels.

* :func:`causal_conv` -- causal depthwise convolution of 1 to 8 taps with bias
  and silu; :func:`causal_conv_step` for one token.
* :func:`selective_scan` -- the input-dependent diagonal state space (up to 64
  states per channel); :func:`selective_scan_step` for one token.
* :func:`fused_norm` -- root-mean-square norm with the gate, residual add and
  residual scale around it.

Activations are ``[batch, length, channels]`` in float32, bfloat16 or float16,
channels contiguous (another layout is copied first), with any batch and step
strides, so halves and slices of a projection's output go in as they are.
Sums, states and statistics are float32.  ``lengths`` (int32 ``[batch]``) gives
each row of a padded batch its valid steps, clamped to 0..length: what lies
behind them is never read, outputs and gradients there are 0, and states pass
them unchanged.  The prompt forms are differentiable (once); the step forms
are not, and say so.  Work runs on the tensors' device and the current stream
of that device; calls allocate their outputs and scratch from the current
stream's allocator, so they may be captured into CUDA graphs.  (As with every
differentiable operation, a backward pass is captured only while no eager graph
of the same leaves is alive: autograd would synchronise with that graph's
stream, which ends the capture.)  There is no counterpart in the reference, and
no fallback.
"""
from __future__ import annotations

import ctypes
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import PT_CONV_MAX_TAPS, PT_NORM_MAX_WIDTH, PT_SCAN_MAX_STATE, ConvArgs, NormArgs, ScanArgs

Tensor = torch.Tensor

_TYPES = {torch.float32: _lib.PT_F32, torch.bfloat16: _lib.PT_BF16, torch.float16: _lib.PT_F16}
_F32 = torch.float32


# ---------------------------------------------------------------- arguments
def _activation(t: Tensor, name: str, ndim: int) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name}: only float32, bfloat16 and float16 are supported, got {t.dtype}")
    if t.ndim != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got shape {tuple(t.shape)}")


def _like(t: Tensor | None, name: str, shape: tuple[int, ...], dtype: torch.dtype, device: torch.device) -> None:
    if t is None:
        return
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")


def _rows(t: Tensor | None) -> Tensor | None:
    """t with contiguous channels: itself where they are."""
    if t is None or t.stride(-1) == 1 or t.shape[-1] == 1:
        return t
    return t.contiguous()


def _dense(t: Tensor | None) -> Tensor | None:
    return None if t is None else t.contiguous()


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _wants_grad(*tensors: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_grad(what: str, *tensors: Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no backward pass: call it under torch.no_grad()")


def _cache(t: Tensor, name: str, tail: tuple[int, int], dtype: torch.dtype, device: torch.device) -> tuple[int, int]:
    """Check a cache [rows, *tail] that a step updates in place; returns (rows, elements between rows)."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.ndim != 3 or tuple(t.shape[1:]) != tail:
        raise ValueError(f"{name} must have shape (rows, {tail[0]}, {tail[1]}), got {tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    rows, size = t.shape[0], tail[0] * tail[1]
    row = t.stride(0)
    if size and rows:
        if (tail[1] > 1 and t.stride(2) != 1) or (tail[0] > 1 and t.stride(1) != tail[1]) or (rows > 1 and row < size):
            raise ValueError(f"{name} is updated in place: each of its rows must be contiguous and none may overlap")
    return rows, row


def _slots(slots: Tensor | None, batch: int, rows: int, name: str, device: torch.device) -> Tensor | None:
    if slots is None:
        if rows != batch:
            raise ValueError(f"{name} has {rows} rows for a batch of {batch}: pass slots to choose among them")
        return None
    _like(slots, "slots", (batch,), torch.int32, device)
    return slots.contiguous()


class _on:
    """Makes a tensor's device current where it is not; ``stream`` is its current stream."""

    __slots__ = ("guard", "stream")

    def __init__(self, device: torch.device) -> None:
        index = device.index
        self.guard = None if torch.cuda.current_device() == index else torch.cuda.device(index)
        self.stream = torch.cuda.current_stream(index).cuda_stream

    def __enter__(self) -> "_on":
        if self.guard is not None:
            self.guard.__enter__()
        return self

    def __exit__(self, *exc: Any) -> None:
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _workspace(nbytes: int, device: torch.device) -> Tensor | None:
    """Scratch of one call, from the allocator of the current stream: calls on other
    streams, and captured graphs, have their own."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _launch(name: str, args: ctypes.Structure, device: torch.device, workspace: str | None = None) -> None:
    lib = _lib.load()
    p = ctypes.byref(args)
    with _on(device) as on:
        if workspace is None:
            st = getattr(lib, name)(p, on.stream)
        else:
            need = int(getattr(lib, workspace)(p))
            ws = _workspace(need, device)
            st = getattr(lib, name)(p, _ptr(ws), need, on.stream)
    if st:
        _lib.check(st, name)


# ---------------------------------------------------------------- causal convolution
def _conv_check(x: Tensor, weight: Tensor, bias: Tensor | None, ndim: int) -> None:
    _activation(x, "x", ndim)
    if not isinstance(weight, Tensor):
        raise TypeError("weight must be a torch.Tensor")
    if weight.ndim != 2 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"weight must have shape ({x.shape[-1]}, taps), got {tuple(weight.shape)}")
    if x.shape[-1] < 1 or not 1 <= weight.shape[1] <= PT_CONV_MAX_TAPS:
        raise ValueError(f"the convolution needs channels and 1 to {PT_CONV_MAX_TAPS} taps, got {tuple(weight.shape)}")
    if weight.dtype != _F32 and weight.dtype != x.dtype:
        raise ValueError(f"weight must be float32 or {x.dtype}, got {weight.dtype}")
    if weight.device != x.device:
        raise ValueError(f"weight must be on {x.device}, got {weight.device}")
    if bias is not None:
        _like(bias, "bias", (x.shape[-1],), weight.dtype, x.device)


def _conv_args(x: Tensor, weight: Tensor, bias: Tensor | None, silu: bool, state: Tensor | None,
               lengths: Tensor | None) -> ConvArgs:
    b, length, d = x.shape
    a = ConvArgs(_TYPES[x.dtype], weight.dtype == _F32, b, length, d, weight.shape[1], bool(silu), 0,
                 x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), _ptr(bias), _ptr(state))
    a.lengths = _ptr(lengths)
    return a


def _conv_forward(x: Tensor, weight: Tensor, bias: Tensor | None, state: Tensor | None, lengths: Tensor | None,
                  silu: bool, final: bool) -> tuple[Tensor, Tensor | None]:
    b, length, d = x.shape
    y = torch.empty((b, length, d), dtype=x.dtype, device=x.device)
    last = torch.empty((b, weight.shape[1] - 1, d), dtype=x.dtype, device=x.device) if final else None
    a = _conv_args(x, weight, bias, silu, state, lengths)
    a.y, a.state_out = y.data_ptr(), _ptr(last)
    _launch("pt_causal_conv", a, x.device)
    return y, last


class CausalConv(torch.autograd.Function):
    """:func:`causal_conv` with its backward pass (one kernel and a sum of its partial dW)."""

    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor, bias: Tensor | None, state: Tensor | None,
                lengths: Tensor | None, silu: bool, final: bool):
        ctx.set_materialize_grads(False)
        y, last = _conv_forward(x, weight, bias, state, lengths, silu, final)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        return (y, last) if final else y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor | None, dlast: Tensor | None = None):
        x, weight, bias, state, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else _rows(dy)
        dlast = _dense(dlast)
        make = torch.empty if x.shape[0] else torch.zeros  # an empty batch launches nothing
        dx, dw, db, ds = (make(t.shape, dtype=t.dtype, device=t.device) if n else None
                          for t, n in zip((x, weight, bias, state), need))
        a = _conv_args(x, weight, bias, ctx.silu, state, lengths)
        a.dy, a.dy_batch, a.dy_step = dy.data_ptr(), dy.stride(0), dy.stride(1)
        a.dstate_out = _ptr(dlast)
        a.dx, a.dw, a.dbias, a.dstate_in = _ptr(dx), _ptr(dw), _ptr(db), _ptr(ds)
        _launch("pt_causal_conv_bwd", a, x.device, "pt_causal_conv_bwd_workspace_bytes")
        return dx, dw, db, ds, None, None, None


def causal_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, silu: bool = False,
                initial_state: Tensor | None = None, return_final_state: bool = False,
                lengths: Tensor | None = None):
    """Causal depthwise convolution over ``x[batch, length, channels]``:

    ``y[b,t,d] = act(bias[d] + sum_j weight[d,j] x[b, t - taps + 1 + j, d])``,
    act being silu or nothing.  ``weight`` is ``[channels, taps]``, 1 to 8 taps,
    in float32 or x's type, ``bias`` ``[channels]`` of weight's type.

    ``initial_state`` ``[batch, taps - 1, channels]`` (x's type) holds the inputs
    before step 0 (zeros without it); with ``return_final_state`` the result is
    ``(y, state)``, the state holding each row's last ``taps - 1`` inputs: what
    the next call, or :func:`causal_conv_step`, starts from.  Differentiable in
    x, weight, bias and initial_state, through y and the final state.
    """
    _conv_check(x, weight, bias, 3)
    b, _, d = x.shape
    _like(initial_state, "initial_state", (b, weight.shape[1] - 1, d), x.dtype, x.device)
    _like(lengths, "lengths", (b,), torch.int32, x.device)
    args = (_rows(x), weight.contiguous(), _dense(bias), _dense(initial_state), _dense(lengths))
    if _wants_grad(x, weight, bias, initial_state):
        return CausalConv.apply(*args, bool(silu), bool(return_final_state))
    y, last = _conv_forward(*args, silu, return_final_state)
    return (y, last) if return_final_state else y


def causal_conv_step(state: Tensor, x: Tensor, weight: Tensor, bias: Tensor | None = None, *, silu: bool = False,
                     slots: Tensor | None = None) -> Tensor:
    """One token of :func:`causal_conv`: ``x[batch, channels]`` gives ``y[batch, channels]``.

    ``state`` ``[rows, taps - 1, channels]`` (x's type) is a cache of windows,
    shifted in place.  Row b of the batch uses window ``slots[b]`` (int32), or
    window b without ``slots``.  A negative slot marks a padding row: its output
    is 0 and no window is touched.  So is a row whose slot is past the cache, or
    was named by an earlier row of the batch; bits 7 and 8 of
    :func:`pathtile_b200.ops.device_error` report that.
    """
    _refuse_grad("causal_conv_step", x, weight, bias)
    _conv_check(x, weight, bias, 2)
    b, d = x.shape
    taps = weight.shape[1]
    device = x.device
    rows, row = _cache(state, "state", (taps - 1, d), x.dtype, device)
    slots = _slots(slots, b, rows, "state", device)
    x, weight, bias = _rows(x), weight.contiguous(), _dense(bias)
    y = torch.empty((b, d), dtype=x.dtype, device=device)
    a = ConvArgs(_TYPES[x.dtype], weight.dtype == _F32, b, 1, d, taps, bool(silu), rows,
                 x.data_ptr(), x.stride(0), 0, weight.data_ptr(), _ptr(bias), None, state.data_ptr(), row,
                 None, _ptr(slots), y.data_ptr())
    _launch("pt_causal_conv_step", a, device)
    return y


# ---------------------------------------------------------------- selective scan
def _scan_check(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None, z: Tensor | None,
                dt_bias: Tensor | None, ndim: int) -> tuple[Tensor, Tensor]:
    """Check the operands; returns B and C with their dimension of groups."""
    _activation(x, "x", ndim)
    shape, device, d = x.shape, x.device, x.shape[-1]
    _like(dt, "dt", shape, x.dtype, device)
    _like(z, "z", shape, x.dtype, device)
    if not isinstance(A, Tensor):
        raise TypeError("A must be a torch.Tensor")
    if A.ndim != 2 or A.shape[0] != d:
        raise ValueError(f"A must have shape ({d}, states), got {tuple(A.shape)}")
    n = A.shape[1]
    if d < 1 or not 1 <= n <= PT_SCAN_MAX_STATE:
        raise ValueError(f"the scan needs channels and 1 to {PT_SCAN_MAX_STATE} states, got A {tuple(A.shape)}")
    if A.dtype != _F32 or A.device != device:
        raise ValueError(f"A must be float32 on {device}, got {A.dtype} on {A.device}")
    _like(D, "D", (d,), _F32, device)
    _like(dt_bias, "dt_bias", (d,), _F32, device)
    both = []
    for t, name in ((B, "B"), (C, "C")):
        if not isinstance(t, Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.ndim == ndim:
            t = t.unsqueeze(-2)
        if t.ndim != ndim + 1 or t.shape[:-2] != shape[:-1] or t.shape[-1] != n:
            raise ValueError(f"{name} must have shape {tuple(shape[:-1])} + ({n},) or + (groups, {n}), "
                             f"got {tuple(t.shape)}")
        if t.dtype != x.dtype or t.device != device:
            raise ValueError(f"{name} must be {x.dtype} on {device}, got {t.dtype} on {t.device}")
        both.append(t)
    groups = both[0].shape[-2]
    if both[1].shape[-2] != groups or groups < 1 or d % groups:
        raise ValueError(f"B and C must have one number of groups that divides {d} channels, got "
                         f"{groups} and {both[1].shape[-2]}")
    return both[0], both[1]


def _scan_args(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None, z: Tensor | None,
               dt_bias: Tensor | None, state: Tensor | None, lengths: Tensor | None, softplus: bool) -> ScanArgs:
    b, length, d = x.shape
    zb, zs = (z.stride(0), z.stride(1)) if z is not None else (0, 0)
    a = ScanArgs(_TYPES[x.dtype], b, length, d, A.shape[1], B.shape[2], bool(softplus), 0,
                 x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), C.data_ptr(),
                 x.stride(0), x.stride(1), dt.stride(0), dt.stride(1), zb, zs,
                 B.stride(0), B.stride(1), B.stride(2), C.stride(0), C.stride(1), C.stride(2),
                 A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(state))
    a.lengths = _ptr(lengths)
    return a


def _scan_forward(args: tuple, softplus: bool, final: bool, train: bool):
    x, A = args[0], args[2]
    b, length, d = x.shape
    a = _scan_args(*args, softplus)
    y = torch.empty((b, length, d), dtype=x.dtype, device=x.device)
    last = torch.empty((b, d, A.shape[1]), dtype=_F32, device=x.device) if final else None
    a.y, a.hlast = y.data_ptr(), _ptr(last)
    checkpoints = None
    if train:
        size = int(_lib.load().pt_scan_checkpoint_bytes(ctypes.byref(a)))
        checkpoints = torch.empty(size // 4, dtype=_F32, device=x.device)
        a.checkpoints = checkpoints.data_ptr()
    _launch("pt_scan", a, x.device, "pt_scan_workspace_bytes")
    return y, last, checkpoints


class SelectiveScan(torch.autograd.Function):
    """:func:`selective_scan` with its backward pass.  The forward pass keeps the
    states at every 16th step for it (float32)."""

    @staticmethod
    def forward(ctx: Any, x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus: bool, final: bool):
        ctx.set_materialize_grads(False)
        args = (x, dt, A, B, C, D, z, dt_bias, state, lengths)
        y, last, checkpoints = _scan_forward(args, softplus, final, True)
        ctx.save_for_backward(*args, checkpoints)
        ctx.softplus = softplus
        return (y, last) if final else y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor | None, dlast: Tensor | None = None):
        *args, checkpoints = ctx.saved_tensors
        x = args[0]
        need = ctx.needs_input_grad
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else _rows(dy)
        dlast = _dense(dlast)
        make = torch.empty if x.shape[0] else torch.zeros  # an empty batch launches nothing
        grads = [make(t.shape, dtype=t.dtype, device=t.device) if n and t is not None else None
                 for t, n in zip(args[:9], need)]
        a = _scan_args(*args, ctx.softplus)
        a.checkpoints = checkpoints.data_ptr()
        a.dy, a.dy_batch, a.dy_step = dy.data_ptr(), dy.stride(0), dy.stride(1)
        a.dhlast = _ptr(dlast)
        a.dx, a.ddt, a.dA, a.dB, a.dC, a.dD, a.dz, a.ddt_bias, a.dh0 = map(_ptr, grads)
        _launch("pt_scan_bwd", a, x.device, "pt_scan_bwd_workspace_bytes")
        return (*grads, None, None, None)


def selective_scan(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None,
                   z: Tensor | None = None, dt_bias: Tensor | None = None, *, dt_softplus: bool = False,
                   initial_state: Tensor | None = None, return_final_state: bool = False,
                   lengths: Tensor | None = None):
    """Selective diagonal state space over ``x[batch, length, channels]``:

    ``delta = dt + dt_bias`` (softplus of it with ``dt_softplus``),
    ``h_t[n] = exp(delta A[d,n]) h_{t-1}[n] + delta x B_t[n]``,
    ``y_t = sum_n C_t[n] h_t[n] + D[d] x``, times ``silu(z)`` where z is given.

    ``dt`` and ``z`` are shaped and typed like x; ``A`` is ``[channels, states]``
    (1 to 64 states), ``D`` and ``dt_bias`` ``[channels]``, all float32; ``B``
    and ``C`` are ``[batch, length, states]``, or ``[batch, length, groups,
    states]`` where each group serves channels / groups neighbouring channels,
    in x's type.  ``initial_state`` is ``[batch, channels, states]`` float32
    (zeros without it); with ``return_final_state`` the result is ``(y, state)``.
    Differentiable in all tensors but lengths, through y and the final state.
    """
    B4, C4 = _scan_check(x, dt, A, B, C, D, z, dt_bias, 3)
    b, _, d = x.shape
    _like(initial_state, "initial_state", (b, d, A.shape[1]), _F32, x.device)
    _like(lengths, "lengths", (b,), torch.int32, x.device)
    args = (_rows(x), _rows(dt), A.contiguous(), _rows(B4), _rows(C4), _dense(D), _rows(z), _dense(dt_bias),
            _dense(initial_state), _dense(lengths))
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, initial_state):
        return SelectiveScan.apply(*args, bool(dt_softplus), bool(return_final_state))
    y, last, _ = _scan_forward(args, dt_softplus, return_final_state, False)
    return (y, last) if return_final_state else y


def selective_scan_step(state: Tensor, x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor,
                        D: Tensor | None = None, z: Tensor | None = None, dt_bias: Tensor | None = None, *,
                        dt_softplus: bool = False, slots: Tensor | None = None) -> Tensor:
    """One token of :func:`selective_scan`: x, dt, z ``[batch, channels]``, B and C
    ``[batch, states]`` or ``[batch, groups, states]``; returns ``y[batch, channels]``.

    ``state`` ``[rows, channels, states]`` (float32) is a cache of states, updated
    in place; ``slots`` as in :func:`causal_conv_step`.
    """
    _refuse_grad("selective_scan_step", x, dt, A, B, C, D, z, dt_bias)
    B, C = _scan_check(x, dt, A, B, C, D, z, dt_bias, 2)
    b, d = x.shape
    n = A.shape[1]
    device = x.device
    rows, row = _cache(state, "state", (d, n), _F32, device)
    slots = _slots(slots, b, rows, "state", device)
    x, dt, z, A, B, C = _rows(x), _rows(dt), _rows(z), A.contiguous(), _rows(B), _rows(C)
    D, dt_bias = _dense(D), _dense(dt_bias)
    y = torch.empty((b, d), dtype=x.dtype, device=device)
    a = ScanArgs(_TYPES[x.dtype], b, 1, d, n, B.shape[1], bool(dt_softplus), rows,
                 x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), C.data_ptr(),
                 x.stride(0), 0, dt.stride(0), 0, z.stride(0) if z is not None else 0, 0,
                 B.stride(0), 0, B.stride(1), C.stride(0), 0, C.stride(1),
                 A.data_ptr(), _ptr(D), _ptr(dt_bias), None, state.data_ptr(), row, None, _ptr(slots), y.data_ptr())
    _launch("pt_scan_step", a, device)
    return y


# ---------------------------------------------------------------- norm
def _flat(t: Tensor | None) -> Tensor | None:
    """t as [rows, channels], channels contiguous."""
    return None if t is None else _rows(t if t.ndim == 2 else t.reshape(-1, t.shape[-1]))


def _norm_args(x: Tensor, weight: Tensor, gate: Tensor | None, residual: Tensor | None, scale: Tensor | None,
               groups: int, eps: float) -> NormArgs:
    return NormArgs(_TYPES[x.dtype], weight.dtype == _F32, residual is not None and residual.dtype == _F32, groups,
                    x.shape[0], x.shape[1], eps, x.data_ptr(), _ptr(gate), _ptr(residual),
                    x.stride(0), gate.stride(0) if gate is not None else 0,
                    residual.stride(0) if residual is not None else 0, weight.data_ptr(), _ptr(scale))


def _norm_forward(x, weight, gate, residual, scale, groups: int, eps: float) -> tuple[Tensor, Tensor | None]:
    a = _norm_args(x, weight, gate, residual, scale, groups, eps)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r = torch.empty(x.shape, dtype=residual.dtype, device=x.device) if residual is not None else None
    a.y, a.r = y.data_ptr(), _ptr(r)
    _launch("pt_fused_norm", a, x.device)
    return y, r


class FusedNorm(torch.autograd.Function):
    """:func:`fused_norm` with its backward pass, on [rows, channels]."""

    @staticmethod
    def forward(ctx: Any, x, weight, gate, residual, scale, groups: int, eps: float):
        ctx.set_materialize_grads(False)
        y, r = _norm_forward(x, weight, gate, residual, scale, groups, eps)
        ctx.save_for_backward(x, weight, gate, scale, r)
        ctx.groups, ctx.eps = groups, eps
        return (y, r) if residual is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor | None, dr: Tensor | None = None):
        x, weight, gate, scale, r = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else _rows(dy)
        dr = _rows(dr)
        make = torch.empty if x.shape[0] else torch.zeros  # no rows launch nothing
        dx, dw, dg, dres, ds = (make(t.shape, dtype=t.dtype, device=t.device) if n and t is not None else None
                                for t, n in zip((x, weight, gate, r, scale), need))
        # The kernel needs to know of a residual, and reads its sum r instead.
        a = _norm_args(x, weight, gate, r, scale, ctx.groups, ctx.eps)
        a.r, a.dy, a.dy_row = _ptr(r), dy.data_ptr(), dy.stride(0)
        if dr is not None:
            a.dr, a.dr_row = dr.data_ptr(), dr.stride(0)
        a.dx, a.dgate, a.dresidual, a.dweight, a.dscale = map(_ptr, (dx, dg, dres, dw, ds))
        _launch("pt_fused_norm_bwd", a, x.device, "pt_fused_norm_bwd_workspace_bytes")
        return dx, dw, dg, dres, ds, None, None


def fused_norm(x: Tensor, weight: Tensor, *, gate: Tensor | None = None, residual: Tensor | None = None,
               scale: Tensor | None = None, groups: int = 1, eps: float = 1e-5):
    """Root-mean-square norm over the last dimension, fused with what stands around it:

    ``u = x * silu(gate)``, ``r = residual + scale * u``, ``y = r / sqrt(mean(r^2) +
    eps) * weight``, the mean over each of ``groups`` equal parts of the last
    dimension (up to 32768 wide).  Without gate, scale or residual that part
    falls away.  Before a block: ``fused_norm(branch, w, residual=stream)``;
    behind a scan: ``fused_norm(y, w, gate=z)``.

    ``gate`` and ``residual`` are shaped like x; gate has x's type, residual
    float32 or x's type.  ``weight`` and ``scale`` are ``[channels]``, both
    float32 or both x's type.  Returns y in x's type; with a residual ``(y, r)``,
    r in the residual's type, rounded to it before it is normalised.
    Differentiable in all five.
    """
    if isinstance(x, Tensor) and x.ndim < 1:
        raise ValueError("x must have at least one dimension")
    _activation(x, "x", x.ndim if isinstance(x, Tensor) else 1)
    shape, device, d = x.shape, x.device, x.shape[-1]
    _like(gate, "gate", shape, x.dtype, device)
    if residual is not None:
        wide = isinstance(residual, Tensor) and residual.dtype == _F32
        _like(residual, "residual", shape, _F32 if wide else x.dtype, device)
    if not isinstance(weight, Tensor):
        raise TypeError("weight must be a torch.Tensor")
    _like(weight, "weight", (d,), _F32 if weight.dtype == _F32 else x.dtype, device)
    _like(scale, "scale", (d,), weight.dtype, device)
    groups = int(groups)
    if d < 1 or groups < 1 or d % groups:
        raise ValueError(f"groups must divide the {d} channels, got {groups}")
    if d // groups > PT_NORM_MAX_WIDTH:
        raise ValueError(f"a group may have up to {PT_NORM_MAX_WIDTH} channels, got {d // groups}")
    args = (_flat(x), weight.contiguous(), _flat(gate), _flat(residual), _dense(scale))
    if _wants_grad(x, weight, gate, residual, scale):
        got = FusedNorm.apply(*args, groups, float(eps))
        y, r = got if residual is not None else (got, None)
    else:
        y, r = _norm_forward(*args, groups, float(eps))
    if len(shape) != 2:
        y, r = y.view(shape), None if r is None else r.view(shape)
    return y if r is None else (y, r)


__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "fused_norm",
           "CausalConv", "SelectiveScan", "FusedNorm"]
