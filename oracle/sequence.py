"""FP64 definitions of the sequence operators, with their gradients (test infrastructure only).

Step by step, in float64, straight from the formulas.  With ``absolute=True``
every product enters with its absolute value: the result bounds the sums of
absolute terms that rounding errors are measured against.
"""
from __future__ import annotations

import torch

Tensor = torch.Tensor


def _f(t: Tensor | None, absolute: bool) -> Tensor | None:
    if t is None:
        return None
    t = t.detach().double()
    return t.abs() if absolute else t


def silu_parts(v: Tensor, absolute: bool) -> tuple[Tensor, Tensor]:
    """silu(v) and its derivative (their absolute values)."""
    s = torch.sigmoid(v)
    y, d = v * s, s * (1 + v * (1 - s))
    return (y.abs(), s * (1 + v.abs() * (1 - s))) if absolute else (y, d)


def _ends(lengths: Tensor | None, batch: int, length: int) -> list[int]:
    return [length] * batch if lengths is None else [min(max(int(n), 0), length) for n in lengths]


def conv(x, weight, bias=None, silu=False, state=None, lengths=None, dy=None, dlast=None, absolute=False) -> dict:
    """y and the final state; with dy also dx, dweight, dbias and dstate."""
    pre_x, w = x.detach().double(), weight.detach().double()
    b, length, d = x.shape
    k = w.shape[1]
    out = {n: [] for n in ("y", "state", "dx", "dstate")}
    dw, db = torch.zeros_like(w), w.new_zeros(d)
    for i, end in enumerate(_ends(lengths, b, length)):
        old = pre_x.new_zeros(k - 1, d) if state is None else state[i].double()
        seq = torch.cat((old, pre_x[i, :end]))
        pre = torch.stack([sum((w[:, j] * seq[t + j] for j in range(k)), pre_x.new_zeros(d))
                           for t in range(end)]) if end else pre_x.new_zeros(0, d)
        if bias is not None:
            pre = pre + bias.double()
        y, slope = silu_parts(pre, absolute) if silu else (pre, torch.ones_like(pre))
        if absolute:
            seq, w = seq.abs(), w.abs()
            size = torch.stack([sum((w[:, j] * seq[t + j] for j in range(k)), pre_x.new_zeros(d))
                                for t in range(end)]) if end else pre
            y = size + (bias.double().abs() if bias is not None else 0)
        out["y"].append(torch.cat((y, y.new_zeros(length - end, d))))
        out["state"].append(seq[end:])
        if dy is None:
            continue
        g = _f(dy[i, :end], absolute) * slope
        if absolute and silu:  # an error of pre moves the slope (its derivative stays below 1/2)
            g = g + _f(dy[i, :end], True) * y
        dseq = torch.zeros_like(seq)
        for t in range(end):
            for j in range(k):
                dseq[t + j] += w[:, j] * g[t]
                dw[:, j] += g[t] * seq[t + j]
        if dlast is not None:
            dseq[end:] += _f(dlast[i], absolute)
        db += g.sum(0)
        out["dx"].append(torch.cat((dseq[k - 1:], dseq.new_zeros(length - end, d))))
        out["dstate"].append(dseq[:k - 1])
    got = {n: torch.stack(v) for n, v in out.items() if v}
    if dy is not None:
        got.update(dweight=dw, dbias=db)
    return got


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, state=None, lengths=None, dy=None,
         dlast=None, absolute=False) -> dict:
    """y and the final state; with dy also the gradients of every operand."""
    if B.ndim == 3:
        got = scan(x, dt, A, B[:, :, None], C[:, :, None], D, z, dt_bias, softplus, state, lengths, dy, dlast, absolute)
        for n in ("dB", "dC"):
            if n in got:
                got[n] = got[n][:, :, 0]
        return got
    b, length, d = x.shape
    g, n = B.shape[2:]
    per = d // g
    dev = x.device
    xs, Bs, Cs, Ds = (_f(t, absolute) for t in (x, B, C, D))
    Ds = torch.zeros(d, dtype=torch.float64, device=dev) if Ds is None else Ds
    raw = dt.detach().double() + (0 if dt_bias is None else dt_bias.detach().double())
    delta = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    rates = A.detach().double()
    ends = torch.tensor(_ends(lengths, b, length), device=dev)
    live = torch.arange(length, device=dev) < ends[:, None]
    # What lies behind a row's end is no part of it.
    xs, delta = (torch.where(live[..., None], t, 0.0) for t in (xs, delta))
    Bs, Cs = (torch.where(live[..., None, None], t, 0.0).repeat_interleave(per, 2) for t in (Bs, Cs))
    size = delta.abs() if absolute else delta
    h = x.new_zeros(b, d, n, dtype=torch.float64) if state is None else _f(state, absolute)
    a = torch.exp(delta[..., None] * rates)
    hs = [h]
    for t in range(length):
        h = a[:, t] * h + (size[:, t] * xs[:, t])[..., None] * Bs[:, t]
        hs.append(h)
    inner = torch.stack([(hs[t + 1] * Cs[:, t]).sum(-1) for t in range(length)], 1) if length else xs
    inner = inner + Ds * xs
    if z is not None:
        zs = torch.where(live[..., None], z.detach().double(), 0.0)
        gate, dgate = silu_parts(zs, absolute)
    else:
        gate, dgate = torch.ones_like(inner), torch.zeros_like(inner)
    out = {"y": torch.where(live[..., None], inner * gate, 0.0), "state": h}
    if dy is None:
        return out
    dout = torch.where(live[..., None], _f(dy, absolute), 0.0)
    u = dout * gate
    dh = torch.zeros_like(h) if dlast is None else _f(dlast, absolute)
    dx, ddelta = Ds * u, torch.zeros_like(u)
    dA, dB, dC = torch.zeros_like(rates), torch.zeros_like(Bs), torch.zeros_like(Cs)
    for t in reversed(range(length)):
        dC[:, t] = u[:, t, :, None] * hs[t + 1]
        dh = dh + u[:, t, :, None] * Cs[:, t]
        dB[:, t] = dh * (size[:, t] * xs[:, t])[..., None]
        dhB = (dh * Bs[:, t]).sum(-1)
        dh = a[:, t] * dh
        dlog = dh * hs[t]
        dA += (dlog * size[:, t, :, None]).sum(0)
        ddelta[:, t] = (dlog * (rates.abs() if absolute else rates)).sum(-1) + dhB * xs[:, t]
        dx[:, t] += dhB * size[:, t]
    ddt = torch.where(live[..., None], ddelta * slope, 0.0)
    share = (b, length, g, per, n)
    out.update(dx=torch.where(live[..., None], dx, 0.0), ddt=ddt, dA=dA, dB=dB.view(share).sum(3), dC=dC.view(share).sum(3),
               dD=(u * xs).sum((0, 1)), ddt_bias=ddt.sum((0, 1)), dstate=dh)
    if z is not None:
        out["dz"] = torch.where(live[..., None], dout * inner * dgate, 0.0)
    return out


def norm(x, weight, gate=None, residual=None, scale=None, groups=1, eps=1e-5, dy=None, dr=None, r=None,
         absolute=False) -> dict:
    """y and r; with dy also the gradients.  ``r``: the stream as stored (it is normalised after its rounding)."""
    xs, w = _f(x, absolute), _f(weight, absolute)
    rows, d = xs.shape
    opened, slope = silu_parts(gate.detach().double(), absolute) if gate is not None else (torch.ones_like(xs), None)
    sc = torch.ones(d, dtype=torch.float64, device=x.device) if scale is None else _f(scale, absolute)
    u = xs * opened
    stream = sc * u if residual is None else _f(residual, absolute) + sc * u
    out = {"r": stream}
    used = _f(stream if r is None else r, False).view(rows, groups, -1)
    rstd = torch.rsqrt(used.square().mean(-1, keepdim=True) + eps)
    hat = used * rstd
    if absolute:
        hat = hat.abs()
    flat = hat.reshape(rows, d)
    out["y"] = flat * w
    if dy is None:
        return out
    dys = _f(dy, absolute)
    v = (dys * w).view(rows, groups, -1)
    mean = (v * hat).mean(-1, keepdim=True)
    g = rstd * (v + hat * mean if absolute else v - hat * mean)
    g = g.reshape(rows, d)
    if dr is not None:
        g = g + _f(dr, absolute)
    out.update(dweight=(dys * flat).sum(0), dresidual=g, dscale=(g * u).sum(0), dx=g * sc * opened)
    if gate is not None:
        out["dgate"] = g * sc * xs * slope
    return out
