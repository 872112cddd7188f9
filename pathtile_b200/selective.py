"""A selective state space block on the sequence operators.

The S4 block (:mod:`pathtile_b200.s4conv`) convolves with a kernel that is the
same at every step; here the state space depends on the input, so it is
scanned.  One block, on ``[batch, length, hidden]``:

    h, stream = fused_norm(x, residual=stream)        norm in front, residual add fused
    u, z      = in_proj(h)                            two halves, read as they lie
    u         = causal_conv(u, silu)                  a few taps
    dt, B, C  = x_proj(u);  dt = dt_proj(dt)
    y         = selective_scan(u, dt, A, B, C, D)
    y         = fused_norm(y, gate=z)                 norm behind, gate fused
    x         = out_proj(y)

The block returns its branch and the residual stream apart: the next block's
norm adds them.  :meth:`SelectiveBlock.step` does the same for one token on a
:class:`SelectiveCache`, which :meth:`SelectiveBlock.forward` can fill from
prompts, padded or not.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from .sequence import causal_conv, causal_conv_step, fused_norm, selective_scan, selective_scan_step


@dataclass
class SelectiveCache:
    """What one block carries from token to token: the convolution's window
    ``[rows, taps - 1, inner]`` and the scan's states ``[rows, inner, states]``."""

    window: torch.Tensor
    state: torch.Tensor


class SelectiveBlock(nn.Module):
    def __init__(self, hidden_dim: int, state_dim: int = 16, expand: int = 2, taps: int = 4, dt_rank: int | None = None,
                 norm_groups: int = 1, eps: float = 1e-5) -> None:
        super().__init__()
        inner = expand * hidden_dim
        dt_rank = dt_rank or max(1, math.ceil(hidden_dim / 16))
        self.inner, self.states, self.taps, self.dt_rank = inner, state_dim, taps, dt_rank
        self.norm_groups, self.eps = norm_groups, eps
        self.norm_weight = nn.Parameter(torch.ones(hidden_dim))
        self.in_proj = nn.Linear(hidden_dim, 2 * inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(inner, taps).uniform_(-1.0, 1.0) * taps ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.x_proj = nn.Linear(inner, dt_rank + 2 * state_dim, bias=False)
        self.dt_proj = nn.Linear(dt_rank, inner, bias=False)
        # Time steps between 0.001 and 0.1, decay rates 1 to state_dim.
        first = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(0.001))
        self.dt_bias = nn.Parameter(first + torch.log(-torch.expm1(-first)))
        self.log_A = nn.Parameter(torch.log(torch.arange(1, state_dim + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        self.out_norm_weight = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Linear(inner, hidden_dim, bias=False)

    def _enter(self, x: torch.Tensor, residual: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
        """The normalised sum of branch and stream, and the sum."""
        if residual is None:
            return fused_norm(x, self.norm_weight, eps=self.eps), x
        return fused_norm(x, self.norm_weight, residual=residual, eps=self.eps)

    def _operands(self, u: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        dt, B, C = self.x_proj(u).split((self.dt_rank, self.states, self.states), dim=-1)
        return F.linear(dt, self.dt_proj.weight), B, C

    def _scan_params(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """A, D and the bias of dt, which the scan takes in float32 whatever the module's type."""
        return -torch.exp(self.log_A.float()), self.D.float(), self.dt_bias.float()

    def _leave(self, y: torch.Tensor, z: torch.Tensor) -> torch.Tensor:
        return self.out_proj(fused_norm(y, self.out_norm_weight, gate=z, groups=self.norm_groups, eps=self.eps))

    def make_cache(self, rows: int, dtype: torch.dtype | None = None) -> SelectiveCache:
        """An empty cache of ``rows`` sequences, on the block's device.  ``dtype``: the
        type the block computes in, its weights' own unless it runs under autocast."""
        w = self.in_proj.weight
        return SelectiveCache(w.new_zeros(rows, self.taps - 1, self.inner, dtype=dtype),
                              torch.zeros(rows, self.inner, self.states, dtype=torch.float32, device=w.device))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                cache: SelectiveCache | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Branch output and residual stream for ``x[batch, length, hidden]``.

        ``cache`` (one row per batch row) holds what came before and is brought
        up to each row's end, in place, so that captured steps read it; no
        gradient passes through it.  ``lengths`` as in :func:`selective_scan`.
        """
        h, residual = self._enter(x, residual)
        u, z = self.in_proj(h).chunk(2, dim=-1)
        keep = cache is not None
        window = state = None
        if keep:
            window, state = cache.window, cache.state
            if torch.is_grad_enabled():  # what the backward pass saves must stay, and the cache moves on
                window, state = window.detach().clone(), state.detach().clone()
        u = causal_conv(u, self.conv_weight, self.conv_bias, silu=True, initial_state=window,
                        return_final_state=keep, lengths=lengths)
        if keep:
            u, window = u
        dt, B, C = self._operands(u)
        A, D, dt_bias = self._scan_params()
        y = selective_scan(u, dt, A, B, C, D, None, dt_bias, dt_softplus=True,
                           initial_state=state, return_final_state=keep, lengths=lengths)
        if keep:
            y, state = y
            with torch.no_grad():
                cache.window.copy_(window)
                cache.state.copy_(state)
        return self._leave(y, z), residual

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: SelectiveCache, residual: torch.Tensor | None = None,
             slots: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """One token: ``x[batch, hidden]``; the cache moves on in place (``slots``: which of its rows)."""
        h, residual = self._enter(x, residual)
        u, z = self.in_proj(h).chunk(2, dim=-1)
        u = causal_conv_step(cache.window, u, self.conv_weight, self.conv_bias, silu=True, slots=slots)
        dt, B, C = self._operands(u)
        A, D, dt_bias = self._scan_params()
        y = selective_scan_step(cache.state, u, dt, A, B, C, D, None, dt_bias, dt_softplus=True, slots=slots)
        return self._leave(y, z), residual
