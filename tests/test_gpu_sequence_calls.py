"""How the sequence operators are called: from several host threads, with forward-mode tangents, with
tensors that autograd watches, in evaluation, on a device that is not the current one."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_norms_from_two_host_threads():
    """Two widths that share a kernel and ask for different amounts of shared memory, launched from two
    threads on two streams: no launch fails and each has the bits it has alone."""
    import ctypes
    from delrec import _lib
    from delrec.block_norm import block_join
    fn = _lib.lib().delrec_block_norm_forward
    failed, wrong, start = [], [], threading.Barrier(2)

    def go(N):
        T, B, stream = 4, 3, torch.cuda.Stream()
        x, y, u = (torch.randn(T, B, N, device="cuda") for _ in range(3))
        want = block_join(x, y, gate=u, next_norm=True)
        out, n = torch.empty_like(x), torch.empty_like(x)
        block = _lib.Block(T, B, N, 0, 1, 0, 1e-5, 0, *(B * N, N) * 5)
        args = (ctypes.byref(block), x.data_ptr(), y.data_ptr(), u.data_ptr(), None, None, None, None, out.data_ptr(),
                n.data_ptr(), None, None, stream.cuda_stream)
        torch.cuda.synchronize()
        start.wait()
        failed.append(sum(fn(*args) != 0 for _ in range(20000)))     # ctypes lets the other thread in
        stream.synchronize()
        if not (torch.equal(out, want[0]) and torch.equal(n, want[1])):
            wrong.append(N)

    threads = [threading.Thread(target=go, args=(N,)) for N in (2048, 1920)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert failed == [0, 0] and not wrong
