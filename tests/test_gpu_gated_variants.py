"""The gated scan's kernel variants that need many rows or long sequences, against the float64 loop:
blocks of a cluster that share a row's time, two channels to a lane, segments of 32 steps, 8-bit
checkpoints with infinities and at the largest scale.  Bounds as in test_gpu_gated.

What the sizes reach (the launch's rules; S = ceil(T / 16) segments, 8 warps a block): clusters
where ceil(N / 32) rows of tiles leave SMs empty; two channels to a lane for 16-bit rows of 16-byte
multiples with B ceil(N / 64) min(16, ceil(S / 8)) >= 296; segments of 32 steps for others in
clusters of c blocks with S >= 16 c."""

import pytest
import torch

from oracle import sequence_oracle as O
from sequence_cases import within
from test_gpu_gated import _check, _cuda, _inputs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,N", [(260, 32), (700, 40), (1500, 32), (4200, 32)])
def test_cluster_blocks_past_the_sequence_end(T, N, dtype):
    """Rows much shorter than T: the blocks of a cluster that lie past a row's end reach the exchange
    long before the others have loaded anything.  Launched back to back, the results stay those of the
    first time, which are the oracle's."""
    from delrec.gated import gated_scan
    c = _inputs(T, 6, N, 1, dtype, ragged=True, resets=True)
    c["lengths"][:6] = torch.tensor([0, 1, 17, T, 130, T // 2])
    first = _check(c)
    d = _cuda(c)
    z, f, h0 = (d[k].requires_grad_(True) for k in ("z", "f", "h0"))
    for _ in range(20):
        h, hT = gated_scan(z, f, h0, lengths=d["lengths"].int(), resets=d["resets"])
        grads = torch.autograd.grad((h, hT), (z, f, h0), (d["gh"], d["ghT"]))
        for got, want in zip((h, hT, *grads), (first[0], first[1], *first[2])):
            assert torch.equal(got, want)
