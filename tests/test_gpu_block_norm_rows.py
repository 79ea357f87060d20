"""The block norms with more rows than blocks have in flight: a third row on its way, and rings that
wrap.  Bounds as in test_gpu_block_norm."""

import pytest
import torch

from test_gpu_block_norm import _check, _inputs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("kind", ["sigmoid", "silu"])
@pytest.mark.parametrize("T,B,N,dtype", [(450, 3, 2048, BF16), (450, 3, 2048, F32), (450, 3, 1536, F32), (331, 4, 1536, F16),
                                         (700, 3, 1030, BF16), (900, 3, 511, F32)])
def test_rows_wrap_around(T, B, N, dtype, kind):
    """At most two blocks fit an SM at 2048 channels: 296 blocks, three rows each in flight, walk these
    rows in four rounds and more; ragged, so that rows that are not read lie between."""
    c = _inputs(T, B, N, dtype)
    _check(c, kind)
    _check(c, kind, lengths=torch.tensor([T, 0, T // 2, 1][:B]))


def test_norm_alone_wraps_around():
    from delrec.block_norm import block_norm
    from test_gpu_block_norm import C, EPS
    from oracle import sequence_oracle as O
    from sequence_cases import within
    c = _inputs(800, 3, 2048, BF16)
    _, n = O.block_join(c["x"].double(), None, None, None, "none", None, c["nw"].double(), EPS, True)
    within(block_norm(c["x"].cuda(), c["nw"].cuda(), eps=EPS), n, 2 * C * n.abs(), "n")
