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


# -- route_logits: groups whose two best keys sum beyond fp32 ----------------------


# groups with lanes of their own, the last ones empty, more than 256 experts, and groups that share lanes
GROUPS = [(32, 8), (240, 4), (60, 6), (320, 5), (510, 3), (490, 7), (304, 4), (511, 7)]


@pytest.mark.parametrize("E,G", GROUPS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_group_sums_below_the_lowest_value_still_order(E, G, score):
    """A bias of the type's lowest value is a number: its groups come last, but they come."""
    g = _gen(E + G)
    T, size = 21, E // G
    logits = 1.5 * _randn(g, T, E)
    logits[3] = -math.inf
    logits[4, : 2 * size] = -math.inf           # groups that are out stand in front of those that are far down
    logits[5, size // 2 :: 2] = math.nan
    logits[6:13, E - size + 3 :] = -math.inf    # the ordinary group fills three slots
    k = min(16, size + 4)
    for bias in (torch.full((E,), torch.finfo(F32).min, device="cuda"), -2e38 - 1e38 * torch.rand(E, generator=g, device="cuda")):
        bias[-size:] = 0.1 * _randn(g, size)    # one ordinary group, behind the others
        for keep in (2, G - 1, G):
            kw = dict(score=score, bias=bias, n_groups=G, topk_groups=keep, group_top=2)
            r = pkg.route_logits(logits, k, counts=True, **kw)
            _check_route(logits.nan_to_num(nan=-math.inf, neginf=-math.inf), k, r, **kw)


@pytest.mark.parametrize("E,G", GROUPS)
def test_group_sums_above_the_largest_value_still_order(E, G):
    g = _gen(E * G)
    T, size = 21, E // G
    logits = 1.5 * _randn(g, T, E)
    logits[4, size:] = -math.inf
    bias = 1.5e38 + 1.9e38 * torch.rand(E, generator=g, device="cuda")
    bias[:size] = 0.1 * _randn(g, size)
    bias[-1] = math.inf
    k = min(8, size)
    for keep in (1, 2, G - 1):
        kw = dict(score="sigmoid", bias=bias, n_groups=G, topk_groups=keep, group_top=2)
        r = pkg.route_logits(logits, k, **kw)
        _check_route(logits, k, r, **kw)
