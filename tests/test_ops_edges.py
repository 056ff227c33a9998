"""route_logits, w4_matvec and add_rmsnorm at the edges of their number ranges, and their calls beside other work."""
import math

import pytest
import torch

import gpt_oss_amd_b200 as pkg
from test_ops import BF16, F32, _check_matvec, _check_route, _gen, _randn, _weights

pytestmark = pytest.mark.gpu


def test_matvec_last_tile_and_first_of_the_next_pass():
    """Blocks that go on from a last tile, short and with scales of no multiple of 16 bytes, to the first one of
    another pass: each row has the bits that it has alone."""
    g = _gen(19)
    for N, K, fmt in ((100, 96, "mxfp4"), (1001, 160, "mxfp4"), (37, 96, "int4"), (1003, 352, "int4")):
        codes, scales = _weights(g, (), N, K, fmt, 32)
        x = _randn(g, 256, K).to(BF16)
        want = torch.cat([pkg.w4_matvec(x[m:m + 1], codes, scales, dtype=F32) for m in range(256)])
        for _ in range(20):
            assert torch.equal(pkg.w4_matvec(x, codes, scales, dtype=F32), want)
