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
