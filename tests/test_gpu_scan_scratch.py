"""GPU: the scratch that the scan's backward pass asks for."""
from __future__ import annotations

import ctypes

import pytest
import torch

import pathtile_b200 as pt
from pathtile_b200 import _lib
from test_gpu_sequence import BF16, F32, Maker, scan_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,lanes", [(8, 2), (16, 4), (32, 8), (64, 16)])
def test_sums_of_dB_and_dC_take_scratch_only_where_they_are_wanted(cuda_device, native_lib, n, lanes):
    b, l, d = 4, 320, 1000
    fake = 0x10000  # not dereferenced: only sizes are asked for
    args = _lib.ScanArgs(dtype=_lib.PT_BF16, batch=b, len=l, dim=d, state=n, groups=1, x=fake, dt=fake, B=fake, C=fake,
                         A=fake, dy=fake, checkpoints=fake)
    sizes = {}
    for dB, dC in ((0, 0), (fake, 0), (0, fake), (fake, fake)):
        args.dB, args.dC = dB or None, dC or None
        sizes[bool(dB), bool(dC)] = native_lib.pt_scan_bwd_workspace_bytes(ctypes.byref(args))
    blocks = -(-d // (256 // lanes))  # of channels; each writes a float for every step and (padded) state, of dB and dC
    assert sizes[True, True] == sizes[True, False] == sizes[False, True] == sizes[False, False] + 4 * blocks * b * l * 8 * lanes


def test_gradients_are_the_same_without_dB_and_dC(cuda_device):
    m = Maker(cuda_device, 101)
    for dtype, l, n in ((BF16, 40, 16), (F32, 700, 64)):
        v = scan_inputs(m, 2, l, 80, n, 1, dtype, True, True, True, True, False)
        dy = m(2, l, 80, dtype=dtype)
        every = {k: t.detach().requires_grad_() for k, t in v.items()}
        some = {k: t.detach().requires_grad_(k not in ("B", "C")) for k, t in v.items()}
        want = dict(zip(every, torch.autograd.grad(pt.selective_scan(**every, dt_softplus=True), list(every.values()), dy)))
        wrt = [k for k in some if k not in ("B", "C")]
        got = torch.autograd.grad(pt.selective_scan(**some, dt_softplus=True), [some[k] for k in wrt], dy)
        assert all(torch.equal(g, want[k]) for k, g in zip(wrt, got))
