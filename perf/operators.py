"""The sequence operators' measured cases: the causal convolution, the selective scan and the fused norm.

Each operator in its plain form (elementary torch operations in 32 bits, rounded
once at the end) and as the calls a user makes of the package, with the inputs,
the work and a 64-bit evaluation of every case.  Shapes: activations are
[batch, length, channels], channels contiguous.

* conv:  y[t] = silu(bias + sum_j w[j] x[t-K+1+j]); earlier x come from a state of K-1 rows
* scan:  d = softplus(dt + dt_bias); h[t] = exp(d A) h[t-1] + d x B[t];
         y = (C[t].h[t] + D x) silu(z)
* norm:  r = residual + scale x silu(gate); y = r / sqrt(mean_group(r^2) + eps) weight
"""
import math

import torch
import torch.nn.functional as F

own = False

EPS = 1e-5
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # One stream decoding: every layer makes this call for every token, so its latency counts.
        {"name": "scan step, one stream", "op": "scan", "mode": "step", "b": 1, "l": 1, "d": 2048, "n": 16, "g": 1, "dtype": "bf16",
         "slots": 0, "state": True, "ragged": False},
        # A server's decoding batch over a cache of states, rows addressed through their slots.
        {"name": "scan step, batch", "op": "scan", "mode": "step", "b": 256, "l": 1, "d": 4096, "n": 16, "g": 1, "dtype": "bf16",
         "slots": 320, "state": True, "ragged": False},
        # One long prompt: few rows, so the length has to be split.
        {"name": "scan prompt, long", "op": "scan", "mode": "prompt", "b": 1, "l": 16384, "d": 2048, "n": 16, "g": 1, "dtype": "bf16",
         "slots": 0, "state": False, "ragged": False},
        # A padded batch of prompts that continue earlier ones; odd sizes, B and C shared by two groups of channels.
        {"name": "scan prompt, ragged", "op": "scan", "mode": "prompt", "b": 5, "l": 1021, "d": 1000, "n": 24, "g": 2, "dtype": "fp16",
         "slots": 0, "state": True, "ragged": True},
        # A training step of a language model's layer.
        {"name": "scan train", "op": "scan", "mode": "train", "b": 8, "l": 2048, "d": 2048, "n": 16, "g": 1, "dtype": "bf16",
         "slots": 0, "state": False, "ragged": False},
        # A training step on this repository's windows: 48 steps, hidden size 128 expanded twice, fp32.
        {"name": "scan train, windows", "op": "scan", "mode": "train", "b": 2048, "l": 48, "d": 256, "n": 16, "g": 1, "dtype": "fp32",
         "slots": 0, "state": False, "ragged": False},
        # Decoding: the convolution's window of the last three tokens, by slot.
        {"name": "conv step", "op": "conv", "mode": "step", "b": 64, "l": 1, "d": 4096, "k": 4, "dtype": "bf16",
         "slots": 80, "state": True, "ragged": False},
        # A padded batch of prompts that continue earlier ones.
        {"name": "conv prompt, ragged", "op": "conv", "mode": "prompt", "b": 3, "l": 4099, "d": 2050, "k": 4, "dtype": "fp16",
         "slots": 0, "state": True, "ragged": True},
        # A training step of a language model's layer.
        {"name": "conv train", "op": "conv", "mode": "train", "b": 8, "l": 2048, "d": 4096, "k": 4, "dtype": "bf16",
         "slots": 0, "state": False, "ragged": False},
        # Decoding: the residual add and the norm in front of a block, residual stream in fp32.
        {"name": "norm residual, decode", "op": "norm", "mode": "prompt", "rows": 64, "d": 2048, "g": 1, "dtype": "bf16",
         "gate": False, "residual": "fp32", "scale": False},
        # Training: the norm behind the scan with its gate, in groups of channels.
        {"name": "norm gated, train", "op": "norm", "mode": "train", "rows": 16384, "d": 4096, "g": 8, "dtype": "bf16",
         "gate": True, "residual": "", "scale": False},
        # Training: residual add with its per-channel scale and norm, an odd width.
        {"name": "norm residual, train", "op": "norm", "mode": "train", "rows": 8191, "d": 1027, "g": 1, "dtype": "bf16",
         "gate": False, "residual": "fp32", "scale": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("scan", "scan", "conv", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "norm":
        g = rng.choice((1, 1, 2, 8))
        d = g * _log(rng, 16, 4096 // g)
        gate = rng.random() < 0.5
        residual = rng.choice(("fp32", dtype)) if not gate or rng.random() < 0.3 else ""
        most = 16384 * 4096 // (2 if dtype == "fp32" or (gate and residual) else 1)
        rows = _log(rng, 1, min(32768, most // (2 if dtype == "fp32" and gate and residual else 1) // d))
        return {"op": op, "mode": rng.choice(("prompt", "train")), "rows": rows, "d": d, "g": g, "dtype": dtype,
                "gate": gate, "residual": residual, "scale": bool(residual) and rng.random() < 0.5}
    mode = rng.choice(("step", "prompt", "train"))
    case = {"op": op, "mode": mode, "b": 1, "l": 1, "d": _log(rng, 32, 4096), "dtype": dtype}
    if op == "scan":
        case["g"] = rng.choice((1, 1, 2, 4))
        case["d"] = max(1, case["d"] // case["g"]) * case["g"]
        case["n"] = rng.choice((8, 16, 16, 16, 24, 32, 64))
    else:
        case["k"] = rng.choice((2, 3, 4, 4, 4, 5, 8))
    if mode == "step":
        case["b"] = _log(rng, 1, 256)
        case["slots"] = rng.choice((0, case["b"] + rng.randrange(1, 64)))
    else:
        # As many positions as the largest listed case has room for.
        most = (8 * 2048 * 2048 * 16 // (case["d"] * max(16, case["n"]))) if op == "scan" else 8 * 2048 * 4096 // case["d"]
        most //= 2 if dtype == "fp32" else 1
        case["l"] = _log(rng, 2, min(16384, most))
        case["b"] = _log(rng, 1, max(1, min(2048, most // case["l"])))
        case["slots"] = 0
    case["state"] = mode == "step" or (mode == "prompt" and rng.random() < 0.5)
    case["ragged"] = mode == "prompt" and case["b"] > 1 and rng.random() < 0.5
    return case


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dev = dict(case), torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    act, f32, train = TYPES[c["dtype"]], torch.float32, c["mode"] == "train"

    def normal(*shape, dtype=act, std=1.0, mean=0.0):
        return (torch.randn(*shape, device=dev, generator=gen) * std + mean).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=gen)

    s = {"case": c}
    if c["op"] == "norm":
        rows, d = c["rows"], c["d"]
        s["x"], s["weight"] = normal(rows, d), normal(d, dtype=f32, std=0.1, mean=1.0)
        s["gate"] = normal(rows, d) if c["gate"] else None
        s["residual"] = normal(rows, d, dtype=TYPES[c["residual"]], std=3.0) if c["residual"] else None
        s["scale"] = normal(d, dtype=f32, std=0.1, mean=0.5) if c["scale"] else None
        names = ("x", "weight", "gate", "residual", "scale")
        if train:
            s["dy"] = normal(rows, d)
            s["dr"] = normal(rows, d, dtype=TYPES[c["residual"]]) if c["residual"] else None
    else:
        b, l, d = c["b"], c["l"], c["d"]
        step = c["mode"] == "step"
        row = (b, d) if step else (b, l, d)
        # What is convolved or scanned is one half of a projection's output, the gate the other half.
        both = normal(*row[:-1], 2 * d)
        s["x"] = both[..., :d]
        held = c["slots"] or b
        s["slots"] = torch.randperm(held, device=dev, generator=gen)[:b].to(torch.int32) if c["slots"] else None
        s["lengths"] = None
        if c["ragged"]:
            s["lengths"] = (1 + uniform(b) * l).to(torch.int32).clamp(max=l)
            s["lengths"][:1] = l
        if c["op"] == "conv":
            s["weight"], s["bias"] = normal(d, c["k"], dtype=f32, std=c["k"] ** -0.5), normal(d, dtype=f32, std=0.1)
            s["state"] = normal(held, c["k"] - 1, d) if c["state"] else None
            names = ("x", "weight", "bias")
        else:
            n, g = c["n"], c["g"]
            s["z"] = both[..., d:]
            s["dt"] = normal(*row, std=0.5)
            # Time steps between 0.001 and 0.1, decay rates 1 to n: the usual initialisation of such layers.
            first = torch.exp(uniform(d) * math.log(100.0) + math.log(0.001))
            s["dt_bias"] = first + torch.log(-torch.expm1(-first))
            s["A"] = -torch.arange(1, n + 1, device=dev, dtype=f32) * (0.8 + 0.4 * uniform(d, 1))
            s["D"] = normal(d, dtype=f32, std=0.1, mean=1.0)
            s["B"], s["C"] = normal(*row[:-1], g, 2 * n).split(n, dim=-1)
            s["state"] = normal(held, d, n, dtype=f32) if c["state"] else None
            names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
        if train:
            s["dy"] = normal(*row)
    if train:
        s["wrt"] = [k for k in names if s[k] is not None]
        for k in s["wrt"]:
            s[k] = s[k].detach().requires_grad_()
    return s


# ---------------------------------------------------------------- plain forms
def run(state):
    return _own(state) if own else _plain(state)


@torch.no_grad()
def _plain(s):
    c = s["case"]
    if c["op"] == "norm":
        return _plain_norm(s)
    if c["mode"] == "step":
        return _plain_conv_step(s) if c["op"] == "conv" else _plain_scan_step(s)
    return _plain_conv(s) if c["op"] == "conv" else _plain_scan(s)


def _valid(s):
    """[b, l, 1]: whether a position is before its row's length."""
    t = torch.arange(s["case"]["l"], device=s["x"].device)
    return (t < s["lengths"].long()[:, None])[..., None] if s["lengths"] is not None else (t >= 0)[None, :, None]


def _silu_grad(v):
    sig = torch.sigmoid(v)
    return sig * (1 + v * (1 - sig))


def _plain_norm(s):
    c = s["case"]
    rows, d, g = c["rows"], c["d"], c["g"]
    x, w = s["x"].float(), s["weight"].float()
    gate = s["gate"].float() if c["gate"] else None
    u = x * F.silu(gate) if c["gate"] else x
    su = s["scale"] * u if c["scale"] else u
    r = s["residual"].float() + su if c["residual"] else su
    # The sum that goes on as the residual stream is what is normalised: it is rounded to its type first.
    r = r.to(s["residual"].dtype).float() if c["residual"] else r
    rstd = torch.rsqrt(r.view(rows, g, d // g).square().mean(-1, keepdim=True) + EPS)
    hat = (r.view(rows, g, d // g) * rstd).view(rows, d)
    out = {"y": (hat * w).to(s["x"].dtype)}
    if c["residual"]:
        out["r"] = r.to(s["residual"].dtype)
    if c["mode"] == "train":
        dy = s["dy"].float()
        dhat = dy * w
        mean = (dhat * hat).view(rows, g, d // g).mean(-1, keepdim=True)
        dr = (rstd * (dhat.view(rows, g, d // g) - hat.view(rows, g, d // g) * mean)).view(rows, d)
        if c["residual"]:
            dr = dr + s["dr"].float()
            out["dresidual"] = dr.to(s["residual"].dtype)
        du = dr * s["scale"] if c["scale"] else dr
        if c["scale"]:
            out["dscale"] = (dr * u).sum(0)
        out["dx"] = (du * F.silu(gate) if c["gate"] else du).to(s["x"].dtype)
        if c["gate"]:
            out["dgate"] = (du * x * _silu_grad(gate)).to(s["x"].dtype)
        out["dweight"] = (dy * hat).sum(0)
    return out


def _plain_conv_step(s):
    at = s["slots"].long() if s["slots"] is not None else torch.arange(s["case"]["b"], device=s["x"].device)
    window = torch.cat((s["state"][at], s["x"][:, None]), 1)
    pre = s["bias"] + (window.float() * s["weight"].t()).sum(1)
    s["state"][at] = window[:, 1:]
    return {"y": F.silu(pre).to(s["x"].dtype), "state": s["state"]}


def _plain_conv(s):
    c = s["case"]
    b, l, k = c["b"], c["l"], c["k"]
    x, w, valid = s["x"], s["weight"].float(), _valid(s)
    before = s["state"] if c["state"] else x.new_zeros(b, k - 1, c["d"])
    rows = torch.cat((before, torch.where(valid, x, 0)), 1)
    windows = rows.float().unfold(1, k, 1)
    pre = s["bias"] + (windows * w).sum(-1)
    out = {"y": torch.where(valid, F.silu(pre), 0).to(x.dtype)}
    if c["mode"] == "prompt":
        last = s["lengths"].long() if c["ragged"] else torch.full((b,), l, device=x.device)
        at = last[:, None] + torch.arange(k - 1, device=x.device)
        out["state"] = rows.gather(1, at[..., None].expand(-1, -1, c["d"]))
    else:
        g = s["dy"].float() * _silu_grad(pre)
        out["dx"] = (F.pad(g, (0, 0, 0, k - 1)).unfold(1, k, 1) * w.flip(1)).sum(-1).to(x.dtype)
        out["dweight"] = (g[..., None] * windows).sum((0, 1))
        out["dbias"] = g.sum((0, 1))
    return out


def _plain_scan_step(s):
    c = s["case"]
    g = c["g"]
    b, d, n = c["b"], c["d"], c["n"]
    at = s["slots"].long() if s["slots"] is not None else torch.arange(b, device=s["x"].device)
    x, z = s["x"].float(), s["z"].float()
    delta = F.softplus(s["dt"].float() + s["dt_bias"])
    B, C = (s[m].float()[:, :, None].expand(b, g, d // g, n).reshape(b, d, n) for m in "BC")
    h = torch.exp(delta[..., None] * s["A"]) * s["state"][at] + (delta * x)[..., None] * B
    s["state"][at] = h
    y = ((h * C).sum(-1) + s["D"] * x) * F.silu(z)
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _recur(a, u):
    """h[t] = a[t] h[t-1] + u[t] along dim 1, by doubling: after each round h holds twice as many terms."""
    step = 1
    while step < a.shape[1]:
        u = torch.cat((u[:, :step], torch.addcmul(u[:, step:], a[:, step:], u[:, :-step])), 1)
        if 2 * step < a.shape[1]:
            a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return u


def _plain_scan(s):
    c = s["case"]
    b, l, d, n, g = c["b"], c["l"], c["d"], c["n"], c["g"]
    heads = (b, l, g, d // g)
    valid = _valid(s)
    x = torch.where(valid, s["x"].float(), 0).view(heads)
    raw = s["dt"].float() + s["dt_bias"]
    # A step past a row's end has no duration: the state stays as it is.
    delta = torch.where(valid, F.softplus(raw), 0).view(heads)
    A = s["A"].view(g, d // g, n)
    B, C = s["B"].float()[:, :, :, None], s["C"].float()[:, :, :, None]
    a = torch.exp(delta[..., None] * A)
    u = (delta * x)[..., None] * B
    if c["state"]:
        u[:, 0] += a[:, 0] * s["state"].view(b, g, d // g, n)
    h = _recur(a, u)
    del u
    z = s["z"].float().view(heads)
    y = (h * C).sum(-1) + s["D"].view(g, d // g) * x
    out = {"y": torch.where(valid, (y * F.silu(z)).view(b, l, d), 0).to(s["x"].dtype)}
    if c["mode"] == "prompt":
        out["state"] = h[:, -1].reshape(b, d, n).clone()
        return out
    dout = s["dy"].float().view(heads)
    dy = dout * F.silu(z)
    out["dz"] = (dout * y * _silu_grad(z)).view(b, l, d).to(s["z"].dtype)
    out["dC"] = (dy[..., None] * h).sum(3).to(s["C"].dtype)
    out["dD"] = (dy * x).sum((0, 1)).view(d)
    # Backwards in time, a step's decay is the next step's.
    later = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1).flip(1)
    dh = _recur(later, (dy[..., None] * C).flip(1)).flip(1)
    del later
    h = F.pad(h, (0, 0) * 3 + (1, 0))[:, :-1]
    dlog = a.mul_(h).mul_(dh)
    del h
    ddelta = (dlog * A).sum(-1)
    dA = dlog.mul_(delta[..., None]).sum((0, 1)).view(d, n)
    del dlog, a
    out["dB"] = (dh * (delta * x)[..., None]).sum(3).to(s["B"].dtype)
    dhB = (dh * B).sum(-1)
    ddt = (ddelta + dhB * x).view(b, l, d) * torch.sigmoid(raw)
    out["dx"] = (dhB * delta + s["D"].view(g, d // g) * dy).view(b, l, d).to(s["x"].dtype)
    out["ddt"], out["ddt_bias"], out["dA"] = ddt.to(s["dt"].dtype), ddt.sum((0, 1)), dA
    return out


# ---------------------------------------------------------------- the package's calls
def _own(s):
    import pathtile_b200 as pt

    c = s["case"]
    if c["op"] == "norm":
        got = pt.fused_norm(s["x"], s["weight"], gate=s["gate"], residual=s["residual"], scale=s["scale"],
                            groups=c["g"], eps=EPS)
        y, r = got if c["residual"] else (got, None)
        out = {"y": y.detach()} if r is None else {"y": y.detach(), "r": r.detach()}
        given = [s["dy"], s["dr"]] if c["mode"] == "train" and c["residual"] else [s.get("dy")]
        results = [y, r] if c["residual"] else [y]
    elif c["mode"] == "step":
        if c["op"] == "conv":
            y = pt.causal_conv_step(s["state"], s["x"], s["weight"], s["bias"], silu=True, slots=s["slots"])
        else:
            y = pt.selective_scan_step(s["state"], s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"],
                                       s["dt_bias"], dt_softplus=True, slots=s["slots"])
        return {"y": y, "state": s["state"]}
    else:
        prompt = c["mode"] == "prompt"
        more = {"initial_state": s["state"], "return_final_state": prompt, "lengths": s["lengths"]}
        if c["op"] == "conv":
            got = pt.causal_conv(s["x"], s["weight"], s["bias"], silu=True, **more)
        else:
            got = pt.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"],
                                    dt_softplus=True, **more)
        if prompt:
            return {"y": got[0], "state": got[1]}
        out, results, given = {"y": got.detach()}, [got], [s["dy"]]
    if c["mode"] == "train":
        grads = torch.autograd.grad(results, [s[k] for k in s["wrt"]], given)
        out.update(("d" + k, v) for k, v in zip(s["wrt"], grads))
    return out


# ---------------------------------------------------------------- work
def work(case):
    """What one pass cannot do without: every input read once, every output written once, and the formulas' operations."""
    c = case
    e, train = TYPES[c["dtype"]].itemsize, c["mode"] == "train"
    if c["op"] == "norm":
        n, r = c["rows"] * c["d"], TYPES[c["residual"]].itemsize if c["residual"] else 0
        inputs = e * (2 if c["gate"] else 1) + r
        params = 4 * c["d"] * (2 if c["scale"] else 1)
        moved, flops = n * (inputs + e + r) + params, n * (4 + 5 * c["gate"] + 2 * c["scale"])
        if train:  # dy (and the residual stream's gradient) in, a gradient for every input out
            moved, flops = moved + n * (e + r + inputs) + params, flops + n * (9 + 10 * c["gate"] + 3 * c["scale"])
        return {"bytes": moved, "flops": flops}
    b, l, d = c["b"], c["l"], c["d"]
    tokens = b * l * d
    if c["op"] == "conv":
        params = 4 * d * (c["k"] + 1)
        held = e * b * (c["k"] - 1) * d * (int(c["state"]) + (c["mode"] != "train"))
        moved, flops = 2 * e * tokens + held + params, tokens * (2 * c["k"] + 4)
        if train:
            moved, flops = moved + 2 * e * tokens + params, flops + tokens * (4 * c["k"] + 6)
        return {"bytes": moved, "flops": flops}
    n, g = c["n"], c["g"]
    shared = 2 * e * b * l * g * n
    params = 4 * d * (n + 2)
    held = 4 * b * d * n * (int(c["state"]) + (c["mode"] != "train"))
    moved, flops = 4 * e * tokens + shared + held + params, tokens * (7 * n + 12)
    if train:
        moved, flops = moved + 4 * e * tokens + shared + params, flops + tokens * (16 * n + 24)
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------- 64 bits
@torch.no_grad()
def exact(case, seed):
    """The definitions in 64 bits: the recurrences one step after the other, sums over explicit indices."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    return (_exact_conv if case["op"] == "conv" else _exact_scan)(case, s)


def _sig64(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _exact_norm(c, s):
    f = {k: s[k].detach().double() for k in ("x", "weight", "gate", "residual", "scale", "dy", "dr") if s.get(k) is not None}
    one = torch.ones((), dtype=torch.float64, device=s["x"].device)
    sig = _sig64(f["gate"]) if "gate" in f else one
    opened = f["gate"] * sig if "gate" in f else one
    scale = f.get("scale", one)
    r = scale * f["x"] * opened
    if "residual" in f:
        # The definition normalises the residual stream as it is stored.
        r = (f["residual"] + r).to(s["residual"].dtype).double() if c["residual"] != "fp32" else f["residual"] + r
    width = c["d"] // c["g"]
    group = r.reshape(-1, c["g"], width)
    norm = torch.sqrt((group * group).sum(-1, keepdim=True) / width + EPS)
    out = {"y": (group / norm).reshape(r.shape) * f["weight"]}
    if "residual" in f:
        out["r"] = r
    if c["mode"] == "train":
        v = (f["dy"] * f["weight"]).reshape(group.shape)
        dr = v / norm - group * (v * group).sum(-1, keepdim=True) / (width * norm ** 3)
        dr = dr.reshape(r.shape) + (f["dr"] if "dr" in f else 0.0)
        if "residual" in f:
            out["dresidual"] = dr
        if "scale" in f:
            out["dscale"] = torch.einsum("rd,rd->d", dr, f["x"] * opened)
        out["dx"] = dr * scale * opened
        if "gate" in f:
            out["dgate"] = dr * scale * f["x"] * (sig + f["gate"] * sig * (1.0 - sig))
        out["dweight"] = torch.einsum("rd,rd->d", f["dy"], (group / norm).reshape(r.shape))
    return out


def _exact_conv(c, s):
    step = c["mode"] == "step"
    x = s["x"].detach().double()
    x = x[:, None] if step else x
    w, bias, k = s["weight"].detach().double(), s["bias"].detach().double(), c["k"]
    b, l, d = x.shape
    at = s["slots"].long() if s["slots"] is not None else torch.arange(b, device=x.device)
    old = s["state"].double()[at] if c["state"] else x.new_zeros(b, k - 1, d)
    ends = s["lengths"].tolist() if c["ragged"] else [l] * b
    y, last = torch.zeros_like(x), torch.zeros_like(old)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    for i, end in enumerate(ends):
        seq = torch.cat((old[i], x[i, :end]))
        last[i] = seq[seq.shape[0] - (k - 1):]
        pre = bias.expand(end, d).clone()
        for j in range(k):
            pre += w[:, j] * seq[j:j + end]
        sig = _sig64(pre)
        y[i, :end] = pre * sig
        if c["mode"] == "train":
            grad = s["dy"][i, :end].double() * (sig + pre * sig * (1.0 - sig))
            dseq = torch.zeros_like(seq)
            for j in range(k):
                dseq[j:j + end] += w[:, j] * grad
                dw[:, j] += torch.einsum("td,td->d", grad, seq[j:j + end])
            dx[i, :end], db = dseq[k - 1:], db + grad.sum(0)
    if step:
        whole = s["state"].double()
        whole[at] = last
        return {"y": y[:, 0], "state": whole}
    if c["mode"] == "prompt":
        return {"y": y, "state": last}
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _exact_scan(c, s):
    step, train = c["mode"] == "step", c["mode"] == "train"
    f = {k: s[k].detach().double() for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")}
    if step:
        f.update((k, f[k][:, None]) for k in ("x", "dt", "B", "C", "z"))
    b, l, d = f["x"].shape
    n, g = c["n"], c["g"]
    per = d // g
    at = s["slots"].long() if s["slots"] is not None else torch.arange(b, device=f["x"].device)
    h = s["state"].double()[at] if c["state"] else f["x"].new_zeros(b, d, n)
    end = s["lengths"].long() if c["ragged"] else torch.full((b,), l, device=h.device)
    raw = f["dt"] + f["dt_bias"]
    delta = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    sig = _sig64(f["z"])
    gate = f["z"] * sig
    y = torch.zeros_like(f["x"])
    past = []
    for t in range(l):
        B, C = (f[m][:, t].repeat_interleave(per, 1) for m in "BC")
        new = torch.exp(delta[:, t, :, None] * f["A"]) * h + (delta[:, t] * f["x"][:, t])[..., None] * B
        if train:
            past.append(h)
        if c["ragged"]:
            live = t < end
            h = torch.where(live[:, None, None], new, h)
            y[:, t] = torch.where(live[:, None], torch.einsum("bdn,bdn->bd", h, C) + f["D"] * f["x"][:, t], 0.0)
        else:
            h = new
            y[:, t] = torch.einsum("bdn,bdn->bd", h, C) + f["D"] * f["x"][:, t]
    if step:
        whole = s["state"].double()
        whole[at] = h
        return {"y": (y * gate)[:, 0], "state": whole}
    if not train:
        return {"y": y * gate, "state": h}
    dout = s["dy"].double()
    out = {"y": y * gate, "dz": dout * y * (sig + f["z"] * sig * (1.0 - sig))}
    dy = dout * gate
    dx, ddelta = f["D"] * dy, torch.zeros_like(delta)
    dA, dB, dC = torch.zeros_like(f["A"]), torch.zeros_like(f["B"]), torch.zeros_like(f["C"])
    carried = torch.zeros_like(h)
    for t in reversed(range(l)):
        B, C = (f[m][:, t].repeat_interleave(per, 1) for m in "BC")
        a = torch.exp(delta[:, t, :, None] * f["A"])
        dC[:, t] = torch.einsum("bgk,bgkn->bgn", dy[:, t].reshape(b, g, per), h.reshape(b, g, per, n))
        dh = dy[:, t, :, None] * C + carried
        dB[:, t] = torch.einsum("bgk,bgkn->bgn", (delta[:, t] * f["x"][:, t]).reshape(b, g, per), dh.reshape(b, g, per, n))
        dhB = torch.einsum("bdn,bdn->bd", dh, B)
        carried = a * dh
        h = past.pop()
        dlog = carried * h
        dA += torch.einsum("bd,bdn->dn", delta[:, t], dlog)
        ddelta[:, t] = torch.einsum("bdn,dn->bd", dlog, f["A"]) + dhB * f["x"][:, t]
        dx[:, t] += dhB * delta[:, t]
    ddt = ddelta * _sig64(raw)
    out.update(dx=dx, ddt=ddt, dA=dA, dB=dB, dC=dC, dD=(dy * f["x"]).sum((0, 1)), ddt_bias=ddt.sum((0, 1)))
    return out
