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
stream, which ends the capture.)  Each call is an operator of torch's dispatcher
(``torch.ops.pathtile_b200``, there from the first call on), backward passes too: ``torch.jit.trace``,
``make_fx`` and dispatch modes record it as one, and on meta tensors it gives
shapes only.  There are no derivatives in forward mode and no rules for
``torch.func``'s transforms: a tensor with a tangent, and a transform, are refused.
There is no counterpart in the reference, and no fallback.
"""
from __future__ import annotations

from types import ModuleType

import torch

Tensor = torch.Tensor

_native: ModuleType | None = None


def _load() -> ModuleType:
    """The native calls (csrc/binding/sequence.cpp): argument checks, autograd nodes and launches."""
    global _native
    if _native is None:
        try:
            from . import _sequence
        except ImportError as e:
            raise RuntimeError(
                "the native binding pathtile_b200/_sequence.so cannot be loaded; build it with "
                f"`python -m pathtile_b200.build`. There is no fallback. ({e})") from e
        _native = _sequence
    return _native


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
    out = (_native or _load()).causal_conv(x, weight, bias, silu, initial_state, return_final_state, lengths)
    return (out[0], out[1]) if return_final_state else out[0]


def causal_conv_step(state: Tensor, x: Tensor, weight: Tensor, bias: Tensor | None = None, *, silu: bool = False,
                     slots: Tensor | None = None) -> Tensor:
    """One token of :func:`causal_conv`: ``x[batch, channels]`` gives ``y[batch, channels]``.

    ``state`` ``[rows, taps - 1, channels]`` (x's type) is a cache of windows,
    shifted in place.  Row b of the batch uses window ``slots[b]`` (int32), or
    window b without ``slots``.  A negative slot marks a padding row: its output
    is 0 and no window is touched.  So is a row whose slot is past the cache, or
    was named by an earlier row of the batch; bits 7 and 8 of
    :func:`pathtile_b200.ops.device_error` report that.  (Each row looks through
    the slots of all rows before it: a tenth of a step's time at 256 rows, more
    than the step itself at some ten thousand.)
    """
    return (_native or _load()).causal_conv_step(state, x, weight, bias, silu, slots)


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
    A step's ``exp(delta A)`` is a float32: states may grow, by up to e^88 a step.
    For its backward pass a call keeps a quarter of a byte per step, channel and
    state; for the gradients of B and C that pass takes 2 bytes of scratch per step
    and channel with up to 16 states, 8 with up to 32, 32 with more.
    Differentiable in all tensors but lengths, through y and the final state.
    """
    out = (_native or _load()).selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state,
                                              return_final_state, lengths)
    return (out[0], out[1]) if return_final_state else out[0]


def selective_scan_step(state: Tensor, x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor,
                        D: Tensor | None = None, z: Tensor | None = None, dt_bias: Tensor | None = None, *,
                        dt_softplus: bool = False, slots: Tensor | None = None) -> Tensor:
    """One token of :func:`selective_scan`: x, dt, z ``[batch, channels]``, B and C
    ``[batch, states]`` or ``[batch, groups, states]``; returns ``y[batch, channels]``.

    ``state`` ``[rows, channels, states]`` (float32) is a cache of states, updated
    in place; ``slots`` as in :func:`causal_conv_step`.
    """
    return (_native or _load()).selective_scan_step(state, x, dt, A, B, C, D, z, dt_bias, dt_softplus, slots)


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
    out = (_native or _load()).fused_norm(x, weight, gate, residual, scale, groups, eps)
    return (out[0], out[1]) if residual is not None else out[0]


__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "fused_norm"]
