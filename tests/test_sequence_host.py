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
