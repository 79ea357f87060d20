"""Host side of the sequence operators: imports, refusals, the accuracy that the 8-bit form states.
None needs a GPU."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch


def test_import_without_cuda_bindings():
    """A torch built without CUDA has none of its private bindings; importing the package needs none."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys, torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]: delattr(torch._C, n)\n"
            "import delrec.gated, delrec.block_norm, delrec.checkpoint8, delrec.networks, delrec.neuron\n")
    env = dict(os.environ, PYTHONPATH=os.path.join(root, "snn-delays_b200"))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_more_rows_than_the_scan_counts_are_refused():
    """A block's next row (row and tile, one grid further) is counted in 32 bits: past 2^30 of them it would
    wrap around.  Refused before anything is launched."""
    from delrec import _lib
    lib, p = _lib.lib(), ctypes.c_void_p(4096)
    for B, N in (((1 << 30) + 1, 1), ((1 << 31) - 1, 1)):
        s = _lib.Scan(1, B, N, N, 1)
        assert lib.delrec_gated_scan_forward(ctypes.byref(s), p, p, None, None, None, p, None, None, *(None,) * 5,
                                             None) == 4
        assert lib.delrec_gated_scan_backward(ctypes.byref(s), p, p, *(None,) * 5, None, None, p, p, None, p, p, None,
                                              None, 0, None) == 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_stated_accuracy_of_the_8_bit_form(dtype):
    """Half a step, at most 1/126 of the group's largest magnitude from 2^-120 to 63.5 * 2^122; 2^-127 below; at
    63.5 * 2^122 and above a step of 2^122."""
    from oracle import sequence_oracle as O
    g = torch.Generator().manual_seed(3)
    for top in (2.0 ** -120, 2.0 ** -24, 1.0, 63.1 / 64, 126.0, 126.5, 6e4, 63.4 * 2.0 ** 122):
        if top > torch.finfo(dtype).max or top < torch.finfo(dtype).tiny / 1024:
            continue
        x = (torch.rand(200, 32, generator=g, dtype=torch.float64) * 2 - 1) * top
        x[:, 0] = top
        x = x.to(dtype).double()
        m = x.abs().amax(-1, keepdim=True)
        assert ((O.restore8(x) - x).abs() <= m / 126).all(), top
    worst = torch.tensor([63.001, 0.5], dtype=torch.float64)      # a step of 1: half a one is 1 / 126.002
    assert (O.restore8(worst) - worst).abs().max() / worst.max() > 1 / 126.1
    tiny = torch.tensor([2.0 ** -121, 2.0 ** -127 * 1.001, -2.0 ** -128], dtype=torch.float64)
    assert (O.restore8(tiny) - tiny).abs().max() <= 2.0 ** -127
    huge = torch.tensor([float(torch.finfo(torch.float32).max), -63.6 * 2.0 ** 122, 1e38], dtype=torch.float64)
    assert (O.restore8(huge) - huge).abs().max() <= 2.0 ** 122
