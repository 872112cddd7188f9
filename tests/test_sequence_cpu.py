"""CPU: the sequence operators' refusals (C entry points and Python checks) and the
FP64 definitions that the GPU tests hold the kernels to, against autograd and
differences.  No kernel is launched here."""
from __future__ import annotations

import ctypes

import pytest
import torch

import pathtile_b200 as pt
from oracle import sequence as ref
from pathtile_b200 import _lib

FAKE = 0x10000  # aligned, never dereferenced: checks fail before any CUDA call
NULL = None


def conv_args(**kw):
    a = _lib.ConvArgs(dtype=_lib.PT_BF16, param_f32=1, batch=2, len=4, dim=8, taps=4, cache_rows=2, x=FAKE, w=FAKE,
                      y=FAKE, dy=FAKE, state_out=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def scan_args(**kw):
    a = _lib.ScanArgs(dtype=_lib.PT_BF16, batch=2, len=4, dim=8, state=16, groups=2, cache_rows=2, x=FAKE, dt=FAKE,
                      B=FAKE, C=FAKE, A=FAKE, y=FAKE, dy=FAKE, checkpoints=FAKE, hlast=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def norm_args(**kw):
    a = _lib.NormArgs(dtype=_lib.PT_F32, param_f32=1, groups=2, rows=3, dim=8, eps=1e-5, x=FAKE, weight=FAKE, y=FAKE,
                      dy=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), _lib.PT_ERR_ARGS),
    (dict(batch=-1), _lib.PT_ERR_ARGS),
    (dict(len=-1), _lib.PT_ERR_ARGS),
    (dict(dim=0), _lib.PT_ERR_ARGS),
    (dict(taps=0), _lib.PT_ERR_ARGS),
    (dict(taps=9), _lib.PT_ERR_UNSUPPORTED),
    (dict(x=NULL), _lib.PT_ERR_ARGS),
    (dict(w=NULL), _lib.PT_ERR_ARGS),
    (dict(batch=0, x=NULL, w=NULL, y=NULL, dy=NULL), _lib.PT_OK),
])
def test_conv_argument_checks(native_lib, kw, status):
    assert native_lib.pt_causal_conv(conv_args(**kw), NULL) == status
    assert native_lib.pt_causal_conv_bwd(conv_args(**kw), NULL, 0, NULL) == status
    assert native_lib.pt_causal_conv_step(conv_args(**{"len": 1, **kw}), NULL) == status
    assert native_lib.pt_causal_conv_bwd_workspace_bytes(conv_args(**kw)) == 0


def test_lengths_that_leave_no_room_to_count_past_a_rows_end(native_lib):
    for n in (2 ** 31 - 1, 2 ** 31 - 4096):
        assert native_lib.pt_causal_conv(conv_args(len=n), NULL) == _lib.PT_ERR_UNSUPPORTED
        assert native_lib.pt_causal_conv_bwd(conv_args(len=n), NULL, 0, NULL) == _lib.PT_ERR_UNSUPPORTED
        assert native_lib.pt_scan(scan_args(len=n), NULL, 0, NULL) == _lib.PT_ERR_UNSUPPORTED
        assert native_lib.pt_scan_bwd(scan_args(len=n), NULL, 0, NULL) == _lib.PT_ERR_UNSUPPORTED


def test_step_argument_checks(native_lib):
    assert native_lib.pt_causal_conv(NULL, NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_causal_conv(conv_args(y=NULL), NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_causal_conv_bwd(conv_args(dy=NULL), NULL, 0, NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_causal_conv_step(conv_args(len=2), NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_causal_conv_step(conv_args(len=1, cache_rows=1), NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_causal_conv_step(conv_args(len=1, state_out=NULL), NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_scan_step(scan_args(len=2), NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_scan_step(scan_args(len=1, cache_rows=1), NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_scan_step(scan_args(len=1, hlast=NULL), NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_scan_step(scan_args(len=1, y=NULL), NULL) == _lib.PT_ERR_ARGS


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=-1), _lib.PT_ERR_ARGS),
    (dict(batch=-1), _lib.PT_ERR_ARGS),
    (dict(state=0), _lib.PT_ERR_ARGS),
    (dict(state=65), _lib.PT_ERR_UNSUPPORTED),
    (dict(groups=3), _lib.PT_ERR_ARGS),
    (dict(groups=0), _lib.PT_ERR_ARGS),
    (dict(A=NULL), _lib.PT_ERR_ARGS),
    (dict(dt=NULL), _lib.PT_ERR_ARGS),
    (dict(C=NULL), _lib.PT_ERR_ARGS),
    (dict(batch=0, x=NULL, A=NULL), _lib.PT_OK),
])
def test_scan_argument_checks(native_lib, kw, status):
    assert native_lib.pt_scan(scan_args(**kw), NULL, 0, NULL) == status
    assert native_lib.pt_scan_bwd(scan_args(**kw), NULL, 0, NULL) == status
    assert native_lib.pt_scan_step(scan_args(**{"len": 1, **kw}), NULL) == status
    assert native_lib.pt_scan_workspace_bytes(scan_args(**kw)) == 0
    assert native_lib.pt_scan_bwd_workspace_bytes(scan_args(**kw)) == 0


def test_scan_pointers_and_checkpoints(native_lib):
    assert native_lib.pt_scan(scan_args(y=NULL), NULL, 0, NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_scan_bwd(scan_args(dy=NULL), NULL, 0, NULL) == _lib.PT_ERR_ARGS
    assert native_lib.pt_scan_bwd(scan_args(checkpoints=NULL), NULL, 0, NULL) == _lib.PT_ERR_ARGS
    # One state [dim, state] of float32 for every 16 steps.
    assert native_lib.pt_scan_checkpoint_bytes(scan_args(len=33)) == 4 * 2 * 3 * 8 * 16
    assert native_lib.pt_scan_checkpoint_bytes(scan_args(len=0)) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=7), _lib.PT_ERR_ARGS),
    (dict(rows=-1), _lib.PT_ERR_ARGS),
    (dict(groups=3), _lib.PT_ERR_ARGS),
    (dict(dim=32769, groups=1), _lib.PT_ERR_UNSUPPORTED),
    (dict(x=NULL), _lib.PT_ERR_ARGS),
    (dict(weight=NULL), _lib.PT_ERR_ARGS),
    (dict(residual=FAKE, r=NULL), _lib.PT_ERR_ARGS),
    (dict(rows=0, x=NULL), _lib.PT_OK),
])
def test_norm_argument_checks(native_lib, kw, status):
    assert native_lib.pt_fused_norm(norm_args(**kw), NULL) == status
    assert native_lib.pt_fused_norm_bwd(norm_args(**kw), NULL, 0, NULL) == status


def test_the_structs_have_the_headers_layout(tmp_path):
    import shutil
    import subprocess

    from conftest import ROOT
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "sizes.c"
    checks = []
    for struct, c_name in ((_lib.ConvArgs, "pt_conv_args"), (_lib.ScanArgs, "pt_scan_args"), (_lib.NormArgs, "pt_norm_args")):
        checks.append((ctypes.sizeof(struct), f"sizeof({c_name})"))
        checks += [(getattr(struct, n).offset, f"offsetof({c_name}, {n})") for n, _ in struct._fields_]
    src.write_text('#include <stddef.h>\n#include "pathtile_b200.h"\n' +
                   "".join(f'_Static_assert({what} == {size}, "{what}");\n' for size, what in checks))
    subprocess.run([cc, "-std=c11", "-fsyntax-only", f"-I{ROOT / 'include'}", str(src)], check=True)


# ---------------------------------------------------------------- Python checks
def test_only_cuda_tensors_of_the_supported_types(native_lib):
    x, w = torch.zeros(2, 4, 8), torch.zeros(8, 4)
    for call in (lambda: pt.causal_conv(x, w), lambda: pt.causal_conv_step(torch.zeros(2, 3, 8), x[:, 0], w),
                 lambda: pt.selective_scan(x, x, w, x, x), lambda: pt.fused_norm(x, torch.zeros(8))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: pt.causal_conv(3, w), lambda: pt.selective_scan([1.0], x, w, x, x), lambda: pt.fused_norm(None, w),
                 lambda: pt.causal_conv(x, w, silu="yes"), lambda: pt.selective_scan(x, x, w, x, x, lengths=[1, 2])):
        with pytest.raises(TypeError):
            call()


# ---------------------------------------------------------------- the definitions
def _inputs(b, length, d, n, g, seed=0):
    r = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=r, dtype=torch.float64)
    return dict(x=f(b, length, d), dt=f(b, length, d), A=-f(d, n).exp(), B=f(b, length, g, n), C=f(b, length, g, n),
                D=f(d), z=f(b, length, d), dt_bias=f(d), state=f(b, d, n))


def _autograd_scan(v, lengths, softplus):
    """The scan in differentiable torch operations."""
    b, length, d = v["x"].shape
    per = d // v["B"].shape[2]
    h, ys = v["state"], []
    raw = v["dt"] + v["dt_bias"]
    delta = torch.nn.functional.softplus(raw) if softplus else raw
    for t in range(length):
        B, C = (v[m][:, t].repeat_interleave(per, 1) for m in "BC")
        new = torch.exp(delta[:, t, :, None] * v["A"]) * h + (delta[:, t] * v["x"][:, t])[..., None] * B
        live = (t < lengths)[:, None]
        h = torch.where(live[..., None], new, h)
        y = ((h * C).sum(-1) + v["D"] * v["x"][:, t]) * torch.nn.functional.silu(v["z"][:, t])
        ys.append(torch.where(live, y, 0.0))
    return torch.stack(ys, 1), h


@pytest.mark.parametrize("softplus", [True, False])
def test_scan_definition_against_autograd(softplus):
    v = {k: t.requires_grad_() for k, t in _inputs(3, 7, 6, 5, 2).items()}
    if not softplus:
        v["dt"] = (v["dt"].detach() * 0.1).requires_grad_()
    lengths = torch.tensor([7, 0, 4])
    y, h = _autograd_scan(v, lengths, softplus)
    gen = torch.Generator().manual_seed(5)
    dy, dh = (torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (y, h))
    grads = torch.autograd.grad([y, h], list(v.values()), [dy, dh])
    got = ref.scan(**v, softplus=softplus, lengths=lengths, dy=dy, dlast=dh)
    torch.testing.assert_close(got["y"], y.detach())
    torch.testing.assert_close(got["state"], h.detach())
    for name, grad in zip(v, grads):
        torch.testing.assert_close(got["d" + name], grad, msg=name)


def test_scan_definition_against_differences():
    v = _inputs(1, 4, 2, 3, 1, seed=3)
    dy = torch.randn(1, 4, 2, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    got = ref.scan(**v, softplus=True, dy=dy)
    for name, t in v.items():
        flat = t.view(-1)
        for i in range(flat.numel()):
            ends = []
            for s in (1e-5, -1e-5):
                w = dict(v)
                w[name] = t.clone()
                w[name].view(-1)[i] += s
                ends.append((ref.scan(**w, softplus=True)["y"] * dy).sum())
            assert abs((ends[0] - ends[1]) / 2e-5 - got["d" + name].reshape(-1)[i]) < 1e-7, (name, i)


@pytest.mark.parametrize("taps,silu", [(1, False), (3, True), (4, False), (4, True)])
def test_conv_definition_against_autograd(taps, silu):
    gen = torch.Generator().manual_seed(2)
    f = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).requires_grad_()
    b, length, d = 4, 6, 3
    x, w, bias, state = f(b, length, d), f(d, taps), f(d), f(b, taps - 1, d)
    lengths = torch.tensor([6, 0, 2, 9])
    ys, states = [], []
    for i in range(b):
        end = min(int(lengths[i]), length)
        seq = torch.cat((state[i], x[i, :end]))
        pre = torch.nn.functional.conv1d(seq.t()[None], w[:, None], bias, groups=d)[0].t() if end else x[i, :0]
        y = torch.nn.functional.silu(pre) if silu else pre
        ys.append(torch.cat((y, torch.zeros(length - end, d, dtype=torch.float64))))
        states.append(seq[end:])
    y, last = torch.stack(ys), torch.stack(states)
    dy, dl = (torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (y, last))
    grads = torch.autograd.grad([y, last], [x, w, bias, state], [dy, dl], allow_unused=True)
    got = ref.conv(x, w, bias, silu, state, lengths, dy, dl)
    torch.testing.assert_close(got["y"], y.detach())
    torch.testing.assert_close(got["state"], last.detach())
    for name, grad in zip(("dx", "dweight", "dbias", "dstate"), grads):
        if grad is not None:
            torch.testing.assert_close(got[name], grad, msg=name)


@pytest.mark.parametrize("parts", ["", "gate", "residual", "gate residual scale"])
def test_norm_definition_against_autograd(parts):
    gen = torch.Generator().manual_seed(4)
    f = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).requires_grad_()
    x, w = f(5, 12), f(12)
    gate, residual = (f(5, 12) if p in parts else None for p in ("gate", "residual"))
    scale = f(12) if "scale" in parts else None
    u = x * torch.nn.functional.silu(gate) if gate is not None else x
    u = u * scale if scale is not None else u
    r = u + residual if residual is not None else u
    y = (r.view(5, 3, 4) * torch.rsqrt(r.view(5, 3, 4).square().mean(-1, keepdim=True) + 1e-5)).view(5, 12) * w
    dy, dr = (torch.randn(5, 12, generator=gen, dtype=torch.float64) for _ in range(2))
    named = {k: t for k, t in dict(x=x, weight=w, gate=gate, residual=residual, scale=scale).items() if t is not None}
    outs, given = ([y, r], [dy, dr]) if residual is not None else ([y], [dy])
    grads = torch.autograd.grad(outs, list(named.values()), given)
    got = ref.norm(x, w, gate, residual, scale, 3, 1e-5, dy, dr if residual is not None else None)
    torch.testing.assert_close(got["y"], y.detach())
    for name, grad in zip(named, grads):
        torch.testing.assert_close(got["d" + name], grad, msg=name)


# ---------------------------------------------------------------- the block that calls them
def test_the_model_offers_both_blocks():
    from pathtile_b200 import s4conv, selective

    plain = s4conv.Model(hidden_dim=16, num_blocks=1)
    assert not any("norm" in n for n in plain.state_dict())  # the S4 model's state dict is as it was
    model = s4conv.Model(hidden_dim=16, state_dim=8, num_blocks=2, block="selective")
    assert all(isinstance(b, selective.SelectiveBlock) for b in model.blocks)
    cache = model.blocks[0].make_cache(3)
    assert cache.window.shape == (3, 3, 32) and cache.state.shape == (3, 32, 8)
    with pytest.raises(ValueError, match="block"):
        s4conv.Model(block="other")
