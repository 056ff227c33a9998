"""add_rmsnorm, route_logits and w4_matvec on the GPU against their definitions in 64 bits (op_reference.py)."""
import math

import numpy as np
import pytest
import torch

import gpt_oss_amd_b200 as pkg
import op_reference as ref
from gpt_oss_amd_b200 import synth

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _close(got, want, error, dtype, label=""):
    """|got - want| within `error` (absolute, elementwise) and the one rounding to dtype."""
    bound = error + (want.abs() + error) * ref.half_step(dtype) + torch.finfo(dtype).smallest_normal * ref.half_step(dtype)
    over = (got.double() - want).abs() > bound
    assert not over.any(), (label, int(over.sum()), ((got.double() - want).abs() / bound).max().item())


# -- add_rmsnorm ---------------------------------------------------------------


def _check_norm(x, w, res, r, quant, eps=1e-5):
    H = x.shape[1]
    rr, y = ref.rmsnorm(x, w, res, eps)
    err = y.abs() * ref.norm_error(H)
    if res is not None:
        assert torch.equal(r.residual, (x.float() + res.float()).to(res.dtype))
    if r.y is not None:
        _close(r.y, y, err, r.y.dtype, "y")
    if quant is None:
        return
    g = H if quant == "row" else 32 if quant == "mx" else quant
    n = -(-H // g)
    top = torch.nn.functional.pad(y, (0, n * g - H)).abs().view(-1, n, g).amax(2)
    e = ref.norm_error(H)
    if quant == "mx":
        byte = r.q_scales.view(torch.uint8).int()
        lo, hi = (torch.where(top > 0, torch.ceil(torch.log2(top * f / 448)) + 127, 127.0).clamp(0, 254).int() for f in (1 - e, 1 + e))
        assert ((byte >= lo) & (byte <= hi)).all()
        scale = torch.exp2(byte.double() - 127)
    else:
        scale = r.q_scales.double()
        want = torch.where(top > 0, top / 448, 1.0)
        assert ((scale - want).abs() <= want * (e + 2.0**-24 * 2)).all()
    wide = scale.repeat_interleave(g, 1)[:, :H]
    # half a step of e4m3: 2^-4 of the value, 2^-10 below 2^-6; the quotient itself has three more roundings
    bound = torch.maximum(y.abs() / 16, wide * 2.0**-10) + y.abs() * (e + 4 * 2.0**-24)
    assert ((r.q.double() * wide - y).abs() <= bound * (1 + 2.0**-20)).all()


@pytest.mark.parametrize("T,H,xt,rt,yt,quant", [
    (1, 2880, BF16, F32, BF16, None), (1, 2880, F32, None, F32, "row"), (3, 64, BF16, BF16, F16, "mx"), (5, 8, F16, F32, BF16, 32),
    (2, 1, F32, F32, F32, "row"), (4, 31, BF16, None, None, "mx"), (7, 33, F32, BF16, BF16, 32), (6, 200, F16, F16, None, 128),
    (33, 2047, F16, F32, BF16, 128), (300, 2880, F32, F32, BF16, "mx"), (1000, 2888, BF16, F32, None, 64), (700, 4096, BF16, BF16, BF16, "row"),
    (2, 8192, BF16, F32, BF16, 128), (400, 8200, F32, None, F32, 64), (2, 16392, BF16, F32, F16, "row"), (3, 32768, F32, F32, BF16, "mx"),
    (2, 32767, BF16, F16, F32, 128), (2, 9999, F32, F32, BF16, "row"), (3001, 64, BF16, F32, BF16, "row"), (1203, 255, F16, F16, F32, 64)])
def test_add_rmsnorm(T, H, xt, rt, yt, quant):
    g = _gen(T * 40009 + H)
    x = (3 * _randn(g, T, H)).to(xt)
    res = None if rt is None else (2 * _randn(g, T, H)).to(rt)
    w = (1 + 0.2 * _randn(g, H)).to(BF16 if H % 3 else F32)
    r = pkg.add_rmsnorm(x, w, res, dtype=yt, quant=quant)
    _check_norm(x, w, res, r, quant)


@pytest.mark.parametrize("H", [64, 100, 2880])
@pytest.mark.parametrize("quant", ["row", 64, "mx"])
def test_add_rmsnorm_strides_in_place_and_rows_behind(H, quant):
    """Rows inside wider buffers, the residual updated in place; what lies around the rows stays as it was."""
    g = _gen(H)
    T = 5
    xb = _randn(g, T + 1, H + 24).to(BF16)
    rb = _randn(g, T + 1, H + 8)
    yb = torch.full((T + 1, H + 40), 7.0, dtype=F16, device="cuda")
    qb = torch.full((T + 1, H + 16), 1.0, device="cuda").to(torch.float8_e4m3fn)
    n = 1 if quant == "row" else -(-H // (32 if quant == "mx" else quant))
    sb = torch.full((T + 1, n), 3.0, device="cuda") if quant != "mx" else torch.full((T + 1, n), 77, dtype=torch.uint8, device="cuda")
    before = rb.clone()
    w = (1 + 0.1 * _randn(g, H)).to(F16)
    r = pkg.add_rmsnorm(xb[:T, :H], w, rb[:T, :H], residual_out=rb[:T, :H], out=yb[:T, :H], q=qb[:T, :H], q_scales=sb[:T], quant=quant)
    _check_norm(xb[:T, :H], w, before[:T, :H], r, quant)
    assert torch.equal(rb[:T, H:], before[:T, H:]) and torch.equal(rb[T], before[T])
    assert (yb[:T, H:] == 7).all() and (yb[T] == 7).all() and (qb[:T, H:].float() == 1).all() and (qb[T].float() == 1).all()
    assert (sb[T] == (77 if quant == "mx" else 3)).all()


def test_add_rmsnorm_unaligned_rows_equal_aligned_ones():
    """The path for rows off the 16-byte boundaries, on the same values: outputs within the bounds of both."""
    g = _gen(3)
    T, H = 9, 512
    x, res, w = _randn(g, T, H).to(BF16), _randn(g, T, H), (1 + 0.1 * _randn(g, H)).to(BF16)
    buf = torch.empty(T, H + 1, dtype=BF16, device="cuda")
    buf[:, 1:] = x
    for quant in ("row", 32, 128, "mx"):
        a, b = pkg.add_rmsnorm(x, w, res, quant=quant), pkg.add_rmsnorm(buf[:, 1:], w, res, quant=quant)
        _check_norm(x, w, res, a, quant)
        _check_norm(x, w, res, b, quant)


def test_add_rmsnorm_zeros_nan_infinity_and_the_largest_values():
    H = 256
    x = torch.zeros(6, H, device="cuda")
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    x[3] = 1e-30
    x[4] = 1.0
    x[4, 100:] = 0.0
    x[5] = 1e15
    w = torch.ones(H, device="cuda")
    for quant, zero in (("row", 1.0), (64, 1.0), ("mx", 1.0)):
        r = pkg.add_rmsnorm(x, w, dtype=F32, quant=quant, eps=1e-5)
        q, s = r.q.float(), r.q_scales.float()
        assert (r.y[0] == 0).all() and (q[0] == 0).all() and (s[0] == zero).all()
        assert r.y[1].isnan().all() and q[1].isnan().all()  # the sum of squares is NaN
        y = torch.zeros(H, device="cuda")
        y[7] = math.nan  # inf * 0
        assert torch.equal(r.y[2].isnan(), y.isnan()) and (r.y[2].nan_to_num() == 0).all()
        _check_norm(x[3:], w, None, type(r)(r.y[3:], None, r.q[3:], r.q_scales[3:]), quant)
        assert (s[4, -1] == zero) or quant == "row"  # a group of zeros in a row that has others


def test_add_rmsnorm_mx_scale_on_the_border():
    """A group whose largest value is 448 * 2^k exactly takes 2^k, the next float up takes 2^(k + 1)."""
    H = 64
    x = torch.zeros(2, H, device="cuda")
    x[:, 0] = 1.0
    eps = 0.0
    w = torch.ones(2, H, device="cuda")  # y[0] = sqrt(64) * w = 8 w exactly
    for k in (-3, 0, 5):
        w[0, 0] = 56.0 * 2.0**k
        w[1, 0] = torch.nextafter(w[0, 0], torch.tensor(math.inf, device="cuda"))
        for row, want in ((0, k), (1, k + 1)):
            r = pkg.add_rmsnorm(x, w[row].contiguous(), dtype=F32, quant="mx", eps=eps)
            assert r.y[0, 0].item() == 8 * w[row, 0].item()
            assert r.q_scales.view(torch.uint8)[0].tolist() == [127 + want, 127]


# -- route_logits ---------------------------------------------------------------


# Relative error of a weight before its last rounding, in steps of fp32 (2^-23): two exponentials of 2 each, 1 + e,
# the division by it; the sum it is divided by: terms off by 6 each, up to 9 + 4 roundings of half a step in it (a
# softmax over 512 experts: 16 in a lane, 5 levels; its exponentials' arguments are rounded: 0.37); the division, the scale.
WEIGHT_ERROR = (6 + 6 + 11 + 0.37 + 1) * 2.0**-23


def _check_route(logits, k, r, **kw):
    a = dict(score="softmax", bias=None, n_groups=1, topk_groups=1, group_top=2, renormalize=True, scale=1.0)
    a.update(kw)
    idx, w = ref.route(logits, k, a["score"], a["bias"], a["n_groups"], a["topk_groups"], a["group_top"], a["renormalize"], a["scale"])
    assert torch.equal(r.topk_i.cpu(), idx)
    _close(r.topk_w.cpu(), w, w.abs() * WEIGHT_ERROR, F32, "weights")
    if r.counts is not None:
        flat = idx[idx >= 0].long()
        assert torch.equal(r.counts.cpu().long(), torch.bincount(flat, minlength=logits.shape[1]))


ROUTES = [
    dict(), dict(renormalize=False, scale=2.5), dict(score="sigmoid"), dict(score="sigmoid", bias=True, scale=0.5),
    dict(bias=True, renormalize=False), dict(score="sigmoid", bias=True, n_groups=4, topk_groups=2, group_top=2),
    dict(n_groups=2, topk_groups=1, group_top=1), dict(n_groups=4, topk_groups=3, group_top=2, renormalize=False),
    dict(bias=True, n_groups=4, topk_groups=4, group_top=1)]


@pytest.mark.parametrize("T,E,k,dtype", [(1, 4, 1, F32), (3, 20, 4, BF16), (65, 32, 4, F32), (17, 60, 6, F16), (40, 128, 8, F32),
                                         (33, 256, 8, BF16), (7, 300, 12, F32), (5, 512, 16, F16)])
@pytest.mark.parametrize("case", range(len(ROUTES)))
def test_route_logits(T, E, k, dtype, case):
    kw = dict(ROUTES[case])
    if kw.get("n_groups", 1) > 1:
        k = min(k, E // kw["n_groups"] * kw["topk_groups"])
        if E // kw["n_groups"] < kw["group_top"]:
            kw["group_top"] = 1
    g = _gen(T + 100 * E + case)
    logits = (1.5 * _randn(g, T, E)).to(dtype)
    if kw.get("bias"):
        kw["bias"] = 0.1 * _randn(g, E)
    r = pkg.route_logits(logits, k, counts=True, **kw)
    _check_route(logits, k, r, **kw)


@pytest.mark.parametrize("E,G", [(240, 4), (304, 4), (288, 8), (60, 6), (120, 3), (510, 3), (490, 7), (96, 32), (31, 31), (320, 5),
                                 (72, 8), (40, 2), (511, 7), (62, 2), (130, 2), (258, 2)])
@pytest.mark.parametrize("kw", [dict(bias=True, group_top=2), dict(score="sigmoid", bias=True, group_top=1), dict(group_top=2),
                                dict(score="sigmoid", group_top=1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_route_logits_groups_of_any_size(E, G, kw, dtype):
    """Groups that fill their lanes, that leave some empty, and that share lanes."""
    g = _gen(E + G)
    kw = dict(kw, n_groups=G, topk_groups=(G + 1) // 2, group_top=min(kw["group_top"], E // G))
    k = min(8, E // G * kw["topk_groups"])
    logits = (1.5 * _randn(g, 33, E)).to(dtype)
    logits[3, : E // 2] = -math.inf
    logits[4, ::3] = logits[4, 0]
    if kw.get("bias"):
        kw["bias"] = 0.1 * _randn(g, E)
    r = pkg.route_logits(logits, k, counts=True, **kw)
    _check_route(logits, k, r, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(score="sigmoid"), dict(renormalize=False), dict(score="sigmoid", bias=True),
                                dict(score="sigmoid", bias=True, n_groups=5, topk_groups=2, group_top=2),
                                dict(n_groups=5, topk_groups=2, group_top=2), dict(n_groups=5, topk_groups=2, group_top=1)])
def test_route_logits_masked_experts_and_rows(kw):
    g = _gen(11)
    T, E, k = 9, 40, 6
    logits = _randn(g, T, E)
    logits[0] = -math.inf                      # a row that the mask leaves nothing
    logits[1] = math.nan
    logits[2, 3:] = -math.inf                  # fewer experts than slots
    logits[3, ::2] = -math.inf
    logits[4, :32] = -math.inf                 # whole groups
    logits[5, 7] = math.nan
    logits[6, 9] = math.inf
    logits[6, 21] = math.inf
    logits[7] = torch.finfo(F32).min           # the type's lowest value is a number
    logits[8, 1:] = torch.finfo(F32).min
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = 0.1 * _randn(g, E)
        kw["bias"][11] = -math.inf
        kw["bias"][12] = math.nan
    r = pkg.route_logits(logits, k, counts=True, **kw)
    clean = logits.nan_to_num(nan=-math.inf, posinf=torch.finfo(F32).max, neginf=-math.inf)
    if kw.get("bias") is not None:
        kw["bias"] = kw["bias"].nan_to_num(nan=-math.inf, neginf=-math.inf)
    _check_route(clean, k, r, **kw)
    assert (r.topk_i[0] == -1).all() and (r.topk_w[0] == 0).all()


@pytest.mark.parametrize("kw", [dict(), dict(score="sigmoid", bias=True), dict(score="sigmoid", bias=True, n_groups=8, topk_groups=3)])
def test_route_logits_ties_go_to_the_lower_index(kw):
    """Logits on a coarse grid and equal biases: most decisions are ties, in 64 bits too."""
    g = _gen(5)
    T, E, k = 50, 64, 8
    logits = torch.randint(-2, 3, (T, E), generator=g, device="cuda").float()
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.randint(0, 2, (E,), generator=g, device="cuda").float() * 0.25
    _check_route(logits, k, pkg.route_logits(logits, k, counts=True, **kw), **kw)


def test_route_logits_keys_closer_than_fp32():
    """Keys that differ by less than fp32 resolves: the order is that of 64 bits."""
    E, k = 64, 8
    # an fp32 sum of sigmoid(l) + bias cannot tell neighbouring logits apart at a bias of 64
    logits = (0.3 + 2.0**-24 * torch.arange(E, device="cuda").flip(0)).float().repeat(3, 1)
    logits[1] = logits[1].flip(0)
    logits[2] = logits[2][torch.randperm(E, generator=_gen(1), device="cuda")]
    bias = torch.full((E,), 64.0, device="cuda")
    kw = dict(score="sigmoid", bias=bias)
    _check_route(logits, k, pkg.route_logits(logits, k, **kw), **kw)
    kw.update(n_groups=8, topk_groups=4, group_top=2)
    _check_route(logits, k, pkg.route_logits(logits, k, **kw), **kw)


def test_route_logits_groups_of_keys_that_cancel():
    """Group scores that are small sums of large keys: fp32 loses them, the choice is that of 64 bits."""
    g = _gen(12)
    T, E, k = 64, 64, 8
    logits = 2.0**-12 * _randn(g, T, E)
    bias = torch.full((E,), -5000.0, device="cuda")
    bias[::8] = 5000.0  # the best of each group; its second best is -5000 + p
    for G in (8, 4):
        kw = dict(score="sigmoid", bias=bias, n_groups=G, topk_groups=G // 2, group_top=2)
        _check_route(logits, k, pkg.route_logits(logits, k, **kw), **kw)


def test_route_logits_large_batch_strides_and_rows_behind():
    """Many tokens per warp; every expert id of a large batch against the small-batch call, nothing written behind."""
    g = _gen(8)
    T, E, k = 20011, 128, 4
    buf = _randn(g, T, E + 3)
    logits = buf[:, :E]
    bias = 0.1 * _randn(g, E)
    out_i = torch.full((T + 2, k), 99, dtype=torch.int32, device="cuda")
    out_w = torch.full((T + 2, k), 9.0, device="cuda")
    kw = dict(score="sigmoid", bias=bias, scale=2.0)
    r = pkg.route_logits(logits, k, counts=True, topk_i=out_i[:T], topk_w=out_w[:T], **kw)
    assert (out_i[T:] == 99).all() and (out_w[T:] == 9).all()
    assert int(r.counts.sum()) == T * k
    assert torch.equal(r.counts.long(), torch.bincount(r.topk_i.flatten().long(), minlength=E))
    p = torch.sigmoid(logits.double())
    key, idx = (p + bias.double()).sort(dim=1, descending=True, stable=True)
    assert torch.equal(r.topk_i.long(), idx[:, :k])
    w = p.gather(1, idx[:, :k])
    w = w / w.sum(1, keepdim=True) * 2
    _close(r.topk_w, w, w * WEIGHT_ERROR, F32)
    pick = torch.arange(0, T, 1999, device="cuda")
    s = pkg.route_logits(logits[pick].contiguous(), k, **kw)
    assert torch.equal(s.topk_i, r.topk_i[pick]) and torch.equal(s.topk_w, r.topk_w[pick])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_logits_weights_far_below_the_best_expert(score):
    """A bias chooses experts whose scores are below fp32's range beside the best one: the ratios of their
    weights stay."""
    E, k = 40, 4
    logits = torch.full((2, E), -130.0, device="cuda")
    logits[:, 0] = 60.0
    logits[0, 5:9] = torch.tensor([-100.0, -101.0, -102.5, -130.0], device="cuda")
    logits[1, 5:9] = torch.tensor([-300.0, -301.0, -302.5, -300.25], device="cuda")
    bias = torch.zeros(E, device="cuda")
    bias[5:9] = torch.tensor([5.0, 4.0, 3.0, 2.0], device="cuda")
    kw = dict(score=score, bias=bias)
    _check_route(logits, k, pkg.route_logits(logits, k, **kw), **kw)


def test_route_logits_agrees_with_the_block():
    """On the block's own router scores: the block's indices and weights."""
    shape = pkg.MoEShape(hidden=256, intermediate=64, n_experts=40, top_k=4)
    lw = synth.make_layer(shape, seed=3)
    with pkg.MoEEngine(shape, max_tokens=128) as eng:
        eng.load_layer(0, lw)
        t = torch.from_numpy(synth.make_tokens(100, 256, seed=3).view(np.int16)).cuda().view(BF16)
        _, sc, ti, tw = eng.forward(0, t, side=True)
        r = pkg.route_logits(sc, 4)
        assert torch.equal(r.topk_i, ti)
        assert (r.topk_w - tw).abs().max() < 1e-6


# -- w4_matvec -------------------------------------------------------------------


def _weights(g, lead, N, K, fmt, group):
    codes = torch.randint(0, 256, (*lead, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    if fmt == "mxfp4":
        return codes, torch.randint(119, 124, (*lead, N, K // 32), generator=g, device="cuda", dtype=torch.uint8)
    return codes, (0.01 + 0.01 * torch.rand(*lead, N, K // group, generator=g, device="cuda")).to(BF16)


def _x(g, rows, K, kind):
    """-> (x, x_scales, x in fp64)"""
    x = _randn(g, rows, K)
    if kind in (BF16, F16):
        return x.to(kind), None, x.to(kind).double()
    r = pkg.add_rmsnorm(x, torch.ones(K, device="cuda"), dtype=None, quant=kind)
    gs = K if kind == "row" else 32 if kind == "mx" else kind
    return r.q, r.q_scales, r.q.double() * r.q_scales.double().repeat_interleave(gs, 1)[:, :K]


def _check_matvec(got, x64, codes, scales, bias, group, ids, rpx, swiglu=None, label=""):
    K = x64.shape[1]
    y, size = ref.matvec(x64, codes, scales, bias, group, ids, rpx)
    err = size * ref.matvec_error(K)
    if swiglu:
        y, grow = ref.swiglu(y, err, *swiglu)
        err = grow + y.abs() * 8 * 2.0**-24
    _close(got, y, err, got.dtype, label)


@pytest.mark.parametrize("N,K,M,fmt,group,kind,out,bias", [
    (16, 32, 1, "mxfp4", 32, BF16, F32, False), (1, 64, 1, "mxfp4", 32, F16, F32, True), (17, 96, 2, "mxfp4", 32, "mx", BF16, True),
    (33, 160, 3, "int4", 32, BF16, F16, True), (48, 128, 5, "int4", 128, "row", F32, False), (100, 320, 8, "int4", 64, 64, F32, True),
    (2880, 2880, 1, "mxfp4", 32, BF16, F32, True), (5120, 2880, 2, "mxfp4", 32, "mx", F32, False), (2881, 2848, 4, "mxfp4", 32, 128, F32, True),
    (515, 4096, 7, "int4", 128, F16, F32, True), (96, 8192, 9, "mxfp4", 32, 32, F32, False), (31, 16384, 3, "mxfp4", 32, BF16, F32, True),
    (64, 16384, 8, "int4", 64, "row", F32, True), (64, 1024, 17, "mxfp4", 32, BF16, F32, True), (40, 1056, 256, "int4", 32, F16, F32, True),
    (20000, 512, 1, "int4", 64, BF16, F32, False)])
def test_w4_matvec(N, K, M, fmt, group, kind, out, bias):
    g = _gen(N + K + M)
    codes, scales = _weights(g, (), N, K, fmt, group)
    b = 0.1 * _randn(g, N) if bias else None
    x, xsc, x64 = _x(g, M, K, kind)
    y = pkg.w4_matvec(x, codes, scales, b, x_scales=xsc, dtype=out)
    _check_matvec(y, x64, codes, scales, b, group, None, 1)


@pytest.mark.parametrize("n,N,K,ids,rpx,kind", [
    (4, 64, 128, [2, 0, 3, 1], 4, BF16),
    (8, 100, 288, [7, 7, 7, 7, 7, 7, 7, 7, 7, 7, 7], 1, "mx"),       # more rows of one matrix than a pass takes
    (5, 48, 96, [-1, 5, 4, -7, 4, 99, 0], 1, F16),                  # rows without a matrix
    (3, 34, 64, [-1, -1], 2, BF16),                                 # nothing at all
    (6, 70, 1312, [0, 5, 5, 3, 0, 5, 2, 2, 0, 1], 2, "row"),
    (32, 2880, 2880, [int(v) for v in np.random.default_rng(0).integers(0, 32, 32)], 4, 64)])
@pytest.mark.parametrize("fmt", ["mxfp4", "int4"])
@pytest.mark.parametrize("act", [None, (1.702, 7.0)])
def test_w4_matvec_of_chosen_matrices(n, N, K, ids, rpx, kind, fmt, act):
    g = _gen(n * N + K)
    codes, scales = _weights(g, (n,), N, K, fmt, 32)
    bias = 0.1 * _randn(g, n, N)
    rows = -(-len(ids) // rpx)
    x, xsc, x64 = _x(g, rows, K, kind)
    idt = torch.tensor(ids, dtype=torch.int32, device="cuda")
    out = torch.full((len(ids) + 1, (N // 2 if act else N) + 3), 5.0, device="cuda")
    n_out = out.shape[1] - 3
    y = pkg.w4_matvec(x, codes, scales, bias, x_scales=xsc, ids=idt, rows_per_x=rpx, swiglu=act, out=out[:-1, :n_out])
    _check_matvec(y, x64, codes, scales, bias, 32, idt, rpx, act)
    assert (out[-1] == 5).all() and (out[:, n_out:] == 5).all()
    for m, e in enumerate(ids):
        if not 0 <= e < n:
            assert (y[m] == 0).all()


def test_w4_matvec_256_chosen_rows():
    g = _gen(77)
    n, N, K = 9, 40, 160
    codes, scales = _weights(g, (n,), N, K, "mxfp4", 32)
    ids = torch.randint(-1, n, (256,), generator=g, device="cuda", dtype=torch.int32)
    x, xsc, x64 = _x(g, 64, K, BF16)
    y = pkg.w4_matvec(x, codes, scales, ids=ids, rows_per_x=4, dtype=F32)
    _check_matvec(y, x64, codes, scales, None, 32, ids, 4)


def test_w4_matvec_checkpoint_blocks_and_every_code():
    """The checkpoint's [N, K / 32, 16] blocks as they are; unit rows of x read single weights, all 16 codes."""
    N, K = 8, 64
    codes = torch.arange(N * K // 2, device="cuda").to(torch.uint8).view(N, K // 32, 16)
    scales = torch.full((N, K // 32), 126, dtype=torch.uint8, device="cuda")
    x = torch.eye(K, device="cuda", dtype=BF16)
    y = pkg.w4_matvec(x, codes, scales, dtype=F32)
    assert torch.equal(y.double().T, ref.dequant(codes.view(N, -1), scales, 32))
    s4 = torch.full((N, K // 32), 0.5, dtype=BF16, device="cuda")
    y = pkg.w4_matvec(x, codes.view(N, -1), s4, dtype=F32)
    assert torch.equal(y.double().T, ref.dequant(codes.view(N, -1), s4, 32))


def test_w4_matvec_every_scale_byte():
    """Each e8m0 byte is 2^(byte - 127), exact while fp32 holds the result; 255 is NaN, as the format has it."""
    N, K = 256, 32
    scales = torch.arange(256, device="cuda").to(torch.uint8).view(N, 1)
    codes = torch.zeros(N, K // 2, dtype=torch.uint8, device="cuda")
    codes[:, 0] = 0x02  # 1.0 in column 0
    for v in (1.0, 2.0**-20, 2.0**20):
        x = torch.zeros(1, K, dtype=BF16, device="cuda")
        x[0, 0] = v
        y = pkg.w4_matvec(x, codes, scales, dtype=F32)[0].double()
        assert y[255].isnan()
        y = y[:255]
        want = (torch.arange(255, device="cuda").double() - 127).exp2() * v
        inside = (want < 2.0**128) & (want >= 2.0**-149)
        assert torch.equal(y[inside], want[inside])
        assert (y[want >= 2.0**128] == math.inf).all()
    # codes of zero stay zero under the largest scale
    codes[:, 0] = 0
    assert (pkg.w4_matvec(torch.ones(1, K, dtype=BF16, device="cuda"), codes, scales, dtype=F32)[0, :255] == 0).all()


@pytest.mark.parametrize("N,K,M,fmt,group,kind", [
    # two pairs of rows per pass: many tiles, or many rows
    (12000, 160, 3, "mxfp4", 32, BF16), (12001, 2880, 4, "int4", 32, "mx"), (320, 4096, 255, "mxfp4", 32, F16),
    (12003, 8192, 4, "mxfp4", 32, "row"), (12007, 12288, 3, "int4", 64, BF16), (12010, 16384, 4, "int4", 128, 128),
    # one, rows whole and in pieces
    (300, 5760, 1, "mxfp4", 32, BF16), (300, 6144, 2, "int4", 128, 64), (299, 8192, 1, "mxfp4", 32, F16),
    (301, 11264, 2, "int4", 32, "mx"), (303, 11296, 1, "mxfp4", 32, BF16), (300, 16384, 1, "mxfp4", 32, "row"),
    (5003, 4096, 1, "mxfp4", 32, BF16), (5000, 16352, 1, "int4", 32, BF16)])
def test_w4_matvec_rings(N, K, M, fmt, group, kind):
    """Each way to divide shared memory among x, stages and blocks."""
    g = _gen(N + K + M)
    codes, scales = _weights(g, (), N, K, fmt, group)
    b = 0.1 * _randn(g, N)
    x, xsc, x64 = _x(g, M, K, kind)
    y = pkg.w4_matvec(x, codes, scales, b, x_scales=xsc, dtype=F32)
    _check_matvec(y, x64, codes, scales, b, group, None, 1)


def test_w4_matvec_one_and_two_pairs_agree():
    """The same bits alone and in a batch that passes over the weights with two pairs of rows."""
    g = _gen(5)
    n, N, K = 4, 3000, 544
    codes, scales = _weights(g, (n,), N, K, "int4", 32)
    x, _, x64 = _x(g, 16, K, BF16)
    ids = torch.tensor([0, 1, 2, 3, 3, 2, 1, 0, 0, 0, 1, 1, 2, 2, 3, 3], dtype=torch.int32, device="cuda")
    y = pkg.w4_matvec(x, codes, scales, ids=ids, dtype=F32)
    _check_matvec(y, x64, codes, scales, None, 32, ids, 1)
    for m in range(16):
        assert torch.equal(y[m:m + 1], pkg.w4_matvec(x[m:m + 1], codes, scales, ids=ids[m:m + 1], dtype=F32))


def test_w4_matvec_x_scale_bytes():
    """The e8m0 scales of x: 2^(byte - 127), 255 is NaN and stays in its row."""
    K = 32
    codes = torch.zeros(16, K // 2, dtype=torch.uint8, device="cuda")
    codes[:, 0] = 0x02  # 1.0 in column 0
    scales = torch.full((16, 1), 127, dtype=torch.uint8, device="cuda")
    x = torch.zeros(256, K, device="cuda")
    x[:, 0] = 1.0
    x = x.to(torch.float8_e4m3fn)
    sx = torch.arange(256, device="cuda").to(torch.uint8).view(256, 1)
    y = pkg.w4_matvec(x, codes, scales, x_scales=sx, dtype=F32).double()
    assert y[255].isnan().all()
    assert torch.equal(y[:255], (torch.arange(255, device="cuda").double() - 127).exp2()[:, None].expand(255, 16))


@pytest.mark.parametrize("mag", [1e-30, 1e-6, 1.0, 1e6, 1e30])
def test_w4_matvec_bf16_of_any_size(mag):
    """bf16 x far outside fp16's range, groups of very different size in one row."""
    g = _gen(2)
    N, K = 50, 512
    codes, scales = _weights(g, (), N, K, "mxfp4", 32)
    x = (_randn(g, 3, K) * mag).to(BF16)
    x[1] = (x[1].view(-1, 32).double() * torch.logspace(-6, 0, K // 32, device="cuda", dtype=torch.float64)[:, None]).view(-1).to(BF16)
    x[2, 40:] = 0
    _check_matvec(pkg.w4_matvec(x, codes, scales, dtype=F32), x.double(), codes, scales, None, 32, None, 1)


def test_w4_matvec_infinity_and_nan_stay_in_their_row():
    g = _gen(4)
    N, K = 64, 256
    codes, scales = _weights(g, (), N, K, "mxfp4", 32)
    x = _randn(g, 4, K).to(BF16)
    clean = pkg.w4_matvec(x, codes, scales, dtype=F32)
    x[1, 17] = math.nan
    x[2, 40] = math.inf
    y = pkg.w4_matvec(x, codes, scales, dtype=F32)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
    assert y[1].isnan().all()
    w = ref.dequant(codes, scales, 32)[:, 40]
    assert y[2][w == 0].isnan().all()
    assert (y[2][w != 0].double() == w[w != 0].sign() * math.inf).all()
    act = pkg.w4_matvec(x, codes, scales, swiglu=(1.702, 7.0), dtype=F32)
    assert act[1].isnan().all() and not act[[0, 3]].isnan().any()  # the clamps of the SwiGLU keep NaN


def test_w4_matvec_one_x_for_all_rows_and_strided_rows():
    g = _gen(6)
    N, K = 96, 352
    codes, scales = _weights(g, (), N, K, "int4", 32)
    buf = _randn(g, 6, K + 8).to(F16)
    x = buf[:, :K]
    _check_matvec(pkg.w4_matvec(x, codes, scales, dtype=F32), x.double(), codes, scales, None, 32, None, 1)
    same = x[:1].expand(5, K)
    a = pkg.w4_matvec(same, codes, scales, dtype=F32)
    assert torch.equal(a, pkg.w4_matvec(same.contiguous(), codes, scales, dtype=F32))
    assert torch.equal(a, pkg.w4_matvec(x[:1], codes, scales, rows_per_x=5, dtype=F32))


def test_w4_matvec_a_row_does_not_depend_on_the_batch():
    """The order of a row's sums is the same in every batch and beside any other rows."""
    g = _gen(9)
    n, N, K = 5, 144, 1440
    codes, scales = _weights(g, (n,), N, K, "mxfp4", 32)
    x = _randn(g, 12, K).to(BF16)
    ids = torch.tensor([3, 1, 3, 3, 0, 1, 3, 3, 3, 3, 3, 3], dtype=torch.int32, device="cuda")
    y = pkg.w4_matvec(x, codes, scales, ids=ids, dtype=F32)
    for m in range(12):
        assert torch.equal(y[m:m + 1], pkg.w4_matvec(x[m:m + 1], codes, scales, ids=ids[m:m + 1], dtype=F32))
        assert torch.equal(y[m:m + 1], pkg.w4_matvec(x[m:m + 1], codes[int(ids[m])], scales[int(ids[m])], dtype=F32))


def test_wrappers_refuse_on_the_device():
    """What the CPU cannot show behind its own refusal: shapes, types and ranges of CUDA tensors, before any launch."""
    from types import SimpleNamespace

    x = torch.zeros(4, 64, dtype=BF16, device="cuda")
    w, res = torch.ones(64, device="cuda"), torch.zeros(4, 64, device="cuda")
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.zeros(8, 2, dtype=torch.uint8, device="cuda")
    q = torch.zeros(4, 64, dtype=torch.float8_e4m3fn, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    wide = torch.zeros(4, 67, dtype=BF16, device="cuda")[:, :64]
    elsewhere = SimpleNamespace(device=torch.device("cuda", torch.cuda.device_count()))
    for call in [
        lambda: pkg.add_rmsnorm(x[0], w), lambda: pkg.add_rmsnorm(x.double(), w), lambda: pkg.add_rmsnorm(x.t(), w),
        lambda: pkg.add_rmsnorm(x, w[:63]), lambda: pkg.add_rmsnorm(x, w.cpu()), lambda: pkg.add_rmsnorm(x, w, res[:3]),
        lambda: pkg.add_rmsnorm(x, w, residual_out=x), lambda: pkg.add_rmsnorm(x, w, x, residual_out=res),
        lambda: pkg.add_rmsnorm(x, w, quant=16), lambda: pkg.add_rmsnorm(x, w, q=q), lambda: pkg.add_rmsnorm(x, w, dtype=torch.int8),
        lambda: pkg.add_rmsnorm(x, w, quant="mx", q_scales=torch.zeros(4, 2, device="cuda")),
        lambda: pkg.add_rmsnorm(x, w, eps=1e300), lambda: pkg.add_rmsnorm(x, w, eps=-1.0), lambda: pkg.add_rmsnorm(x, w, dtype=None),
        lambda: pkg.add_rmsnorm(x[:1].expand(4, 64), w, out=x[:1].expand(4, 64)), lambda: pkg.add_rmsnorm(x, w, stream=elsewhere),
        lambda: pkg.route_logits(x[0], 4), lambda: pkg.route_logits(x, 0), lambda: pkg.route_logits(x, -1),
        lambda: pkg.route_logits(x, 65), lambda: pkg.route_logits(x, 17), lambda: pkg.route_logits(x, 4, score="max"),
        lambda: pkg.route_logits(x, 4, bias=w[:63]), lambda: pkg.route_logits(x, 4, topk_i=torch.zeros(4, 4, device="cuda")),
        lambda: pkg.route_logits(x, 4, n_groups=3), lambda: pkg.route_logits(x, 4, n_groups=2**40),
        lambda: pkg.route_logits(x, 4, scale=math.inf), lambda: pkg.route_logits(x, 4, stream=elsewhere),
        lambda: pkg.w4_matvec(x.float(), codes, scales), lambda: pkg.w4_matvec(x, codes[:, :31], scales),
        lambda: pkg.w4_matvec(x, codes, scales[:7]), lambda: pkg.w4_matvec(x, codes, scales.float()),
        lambda: pkg.w4_matvec(x, codes[None], scales[None]), lambda: pkg.w4_matvec(x, codes, scales, ids=ids.long()),
        lambda: pkg.w4_matvec(x, codes[None], scales[None], ids=ids[:0]), lambda: pkg.w4_matvec(q, codes, scales),
        lambda: pkg.w4_matvec(q, codes, scales, x_scales=torch.zeros(4, 5, device="cuda")), lambda: pkg.w4_matvec(wide, codes, scales),
        lambda: pkg.w4_matvec(x, codes, scales, x_scales=torch.zeros(4, 1, device="cuda")),
        lambda: pkg.w4_matvec(x, codes, scales, rows_per_x=0), lambda: pkg.w4_matvec(x, codes, scales, rows_per_x=65),
        lambda: pkg.w4_matvec(x, codes, scales, rows_per_x=2**40), lambda: pkg.w4_matvec(x, codes, scales, out=torch.zeros(4, 7, device="cuda")),
        lambda: pkg.w4_matvec(x, codes, scales, swiglu=(1.7, -1.0)), lambda: pkg.w4_matvec(x, codes, scales, stream=elsewhere),
    ]:
        with pytest.raises((ValueError, pkg.capi.MoEError)):
            call()


def test_one_row_of_any_stride():
    """The stride of a single row means nothing: rows cut out of odd buffers."""
    g = _gen(3)
    codes, scales = _weights(g, (), 40, 64, "mxfp4", 32)
    wide = _randn(g, 3, 67).to(BF16)
    x = wide[:1, :64]
    assert torch.equal(pkg.w4_matvec(x, codes, scales, rows_per_x=3), pkg.w4_matvec(x.contiguous(), codes, scales, rows_per_x=3))
    w = _randn(g, 64)
    for a, b in zip(pkg.add_rmsnorm(x, w, x, quant="mx"), pkg.add_rmsnorm(x.contiguous(), w, x.contiguous(), quant="mx")):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in zip(pkg.route_logits(x, 5)[:2], pkg.route_logits(x.contiguous(), 5)[:2]):
        assert torch.equal(a, b)


# -- streams, graphs, the run of them together -------------------------------------


def _token_step(x, res, p, K):
    """A block's feed-forward half from the stand-alone operators."""
    n = pkg.add_rmsnorm(x, p["w"], res, dtype=BF16)
    r = pkg.route_logits(n.y.float() @ p["router"].T + p["router_b"], K)
    ids = r.topk_i.view(-1)
    h = pkg.w4_matvec(n.y, p["c1"], p["s1"], p["b1"], ids=ids, rows_per_x=K, swiglu=(1.702, 7.0))
    y = pkg.w4_matvec(h, p["c2"], p["s2"], p["b2"], ids=ids, dtype=F32)
    return n.residual + (y.view(len(x), K, -1) * r.topk_w.unsqueeze(2)).sum(1), r


def _layer(shape, seed):
    lw = synth.make_layer(shape, seed=seed)
    c = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    p = dict(router=c(synth.bf16_bits_to_f32(lw.w_router)), router_b=c(lw.b_router), c1=c(lw.blocks1), s1=c(lw.scales1),
             b1=c(lw.bias1), c2=c(lw.blocks2), s2=c(lw.scales2), b2=c(lw.bias2))
    p["w"] = 1 + 0.1 * _randn(_gen(seed), shape.hidden)
    return lw, p


@pytest.mark.parametrize("T", [1, 5, 32])
def test_token_step_equals_the_block(T):
    """residual add, norm, routing, gate/up and down products of a few tokens: the handle's block on the same weights."""
    shape = pkg.MoEShape(hidden=576, intermediate=320, n_experts=32, top_k=4)
    lw, p = _layer(shape, 21)
    g = _gen(T)
    x, res = _randn(g, T, 576), 2 * _randn(g, T, 576)
    out, r = _token_step(x, res, p, 4)
    with pkg.MoEEngine(shape, max_tokens=64) as eng:
        eng.load_layer(0, lw)
        want, _, ti, tw = eng.forward_norm(0, x + res, p["w"], out=(x + res).clone(), accumulate=True, side=True)
        assert torch.equal(ti, r.topk_i)
        assert (tw - r.topk_w).abs().max() < 1e-5
        d = (out - want).double()
        # both round y and h to bf16; where their fp32 sums differ in the last bits, single values of h land on
        # the neighbouring one, as between any two correct evaluations (the parity rules of the block)
        assert d.norm() / want.double().norm() < 2e-3 and d.abs().max() < 0.1


def test_token_step_in_8_bits_follows_the_64_bit_formulas():
    """norm with MX codes -> products on them: against the formulas on the codes that the norm gave."""
    shape = pkg.MoEShape(hidden=576, intermediate=320, n_experts=32, top_k=4)
    _, p = _layer(shape, 5)
    g = _gen(1)
    x, res = _randn(g, 3, 576).to(BF16), _randn(g, 3, 576)
    n = pkg.add_rmsnorm(x, p["w"], res, dtype=F32, quant="mx")
    r = pkg.route_logits(n.y @ p["router"].T + p["router_b"], 4)
    ids = r.topk_i.view(-1)
    h = pkg.w4_matvec(n.q, p["c1"], p["s1"], p["b1"], x_scales=n.q_scales, ids=ids, rows_per_x=4, swiglu=(1.702, 7.0))
    x64 = n.q.double() * n.q_scales.double().repeat_interleave(32, 1)
    _check_matvec(h, x64, p["c1"].flatten(-2), p["s1"], p["b1"], 32, ids, 4, (1.702, 7.0))


@pytest.mark.parametrize("T", [1, 3, 300])
def test_long_chain_without_waits_between(T):
    """Each call reads what the one or two in front wrote and overwrites what they read: the same bits as with the
    device idle between the calls, eagerly and replayed."""
    g = _gen(T)
    H, E, K, M = 256, 16, 4, min(T, 64)
    w = 1 + 0.1 * _randn(g, H)
    codes, scales = _weights(g, (E,), H, H, "mxfp4", 32)
    start = _randn(g, T, H)
    x, res, y = (torch.empty(T, H, device="cuda", dtype=d) for d in (F32, F32, BF16))
    q, qs = torch.empty(T, H, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(T, H // 32, dtype=torch.uint8, device="cuda")
    ti, tw = torch.empty(T, K, dtype=torch.int32, device="cuda"), torch.empty(T, K, device="cuda")
    counts = torch.empty(E, dtype=torch.int32, device="cuda")
    seen = torch.empty(20, E, dtype=torch.int32, device="cuda")

    def chain(pause=lambda: None):
        x.copy_(start)
        res.zero_()
        for i in range(20):
            pkg.add_rmsnorm(x, w, res, residual_out=res, out=y, quant="mx", q=q, q_scales=qs)
            pause()
            pkg.route_logits(y[:, :E], K, counts=counts, topk_i=ti, topk_w=tw)
            pause()
            pkg.w4_matvec(q[:M], codes, scales, x_scales=qs[:M], ids=ti[:M, i % K].contiguous() if i % 2 else ti.view(-1)[:M], out=x[:M])
            pause()
            seen[i].copy_(counts)
        return [t.clone() for t in (x, res, y, ti, tw, seen)]

    want = chain(torch.cuda.synchronize)
    assert all(torch.equal(a, b) for a, b in zip(chain(), want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_other_streams_and_overlapping_calls():
    """Calls on streams of their own at the same time give what they give one after the other."""
    shape = pkg.MoEShape(hidden=576, intermediate=320, n_experts=32, top_k=4)
    _, p = _layer(shape, 8)
    g = _gen(2)
    data = [(_randn(g, 4, 576), _randn(g, 4, 576)) for _ in range(4)]
    want = [_token_step(x, r, p, 4)[0] for x, r in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [None] * 4
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _token_step(*data[i], p, 4)[0]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    s = torch.cuda.Stream()
    x = data[0][0].to(BF16)
    torch.cuda.synchronize()
    r = pkg.add_rmsnorm(x, p["w"], stream=s)
    s.synchronize()
    assert torch.equal(r.y, pkg.add_rmsnorm(x, p["w"]).y)


def test_stream_argument_of_every_operator():
    """Results on a stream of the caller's, freshly allocated while the current stream still works on freed memory."""
    shape = pkg.MoEShape(hidden=576, intermediate=320, n_experts=32, top_k=4)
    _, p = _layer(shape, 4)
    g = _gen(5)
    x, res = _randn(g, 8, 576), _randn(g, 8, 576)
    n0 = pkg.add_rmsnorm(x, p["w"], res, quant="mx")
    r0 = pkg.route_logits(x[:, :32].contiguous(), 4, counts=True)
    h0 = pkg.w4_matvec(n0.y, p["c1"], p["s1"], p["b1"], ids=r0.topk_i.view(-1), rows_per_x=4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    n = pkg.add_rmsnorm(x, p["w"], res, quant="mx", stream=s)
    s.synchronize()
    r = pkg.route_logits(x[:, :32].contiguous(), 4, counts=True, stream=s)
    s.synchronize()
    h = pkg.w4_matvec(n.y, p["c1"], p["s1"], p["b1"], ids=r.topk_i.view(-1), rows_per_x=4, stream=s)
    s.synchronize()
    for a, b in zip((*n0, *r0, h0), (*n, *r, h)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_offsets_beyond_32_bits():
    """The last rows of tensors of more than 2^31 elements or bytes."""
    g = _gen(14)
    T, H = 66000, 32768  # 2.16e9 elements
    x = torch.zeros(T, H, dtype=BF16, device="cuda")
    x[-3:] = _randn(g, 3, H).to(BF16)
    w = torch.ones(H, dtype=BF16, device="cuda")
    r = pkg.add_rmsnorm(x, w, quant="row")
    _check_norm(x[-3:], w, None, type(r)(r.y[-3:], None, r.q[-3:], r.q_scales[-3:]), "row")
    assert (r.y[:2] == 0).all()
    del x, r
    T, E = 4200000, 512  # 2.15e9 logits
    logits = torch.zeros(T, E, dtype=F16, device="cuda")
    logits[-5:] = _randn(g, 5, E).to(F16)
    r = pkg.route_logits(logits, 6, counts=True)
    _check_route(logits[-5:], 6, type(r)(r.topk_i[-5:], r.topk_w[-5:], None))
    assert torch.equal(r.topk_i[:3].cpu(), torch.arange(6, dtype=torch.int32).repeat(3, 1)) and int(r.counts.sum()) == T * 6
    del logits, r
    n, N, K = 300, 5760, 2880  # 2.5e9 bytes of codes
    codes = torch.zeros(n, N, K // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, N, K // 32), 127, dtype=torch.uint8, device="cuda")
    codes[-1], scales[-1] = _weights(g, (), N, K, "mxfp4", 32)
    x, _, x64 = _x(g, 1, K, BF16)
    ids = torch.tensor([n - 1, 0], dtype=torch.int32, device="cuda")
    y = pkg.w4_matvec(x, codes, scales, ids=ids, rows_per_x=2, dtype=F32)
    _check_matvec(y[:1], x64, codes[-1], scales[-1], None, 32, None, 1)
    assert (y[1] == 0).all()


def test_captured_and_replayed():
    """The whole step in a CUDA graph, two graphs of it replayed in turn on new inputs."""
    shape = pkg.MoEShape(hidden=576, intermediate=320, n_experts=32, top_k=4)
    _, p = _layer(shape, 9)
    g = _gen(3)
    sets = []
    for T in (2, 7):
        x, res = _randn(g, T, 576), _randn(g, T, 576)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _token_step(x, res, p, 4)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, r = _token_step(x, res, p, 4)
            cnt = pkg.route_logits(x[:, :32], 4, counts=True).counts
        sets.append((graph, x, res, out, cnt))
    for _ in range(3):
        for graph, x, res, out, cnt in sets:
            x.normal_(generator=g)
            res.normal_(generator=g)
            graph.replay()
            assert torch.equal(out, _token_step(x, res, p, 4)[0])
            assert torch.equal(cnt, pkg.route_logits(x[:, :32], 4, counts=True).counts)


def test_empty_batches():
    x = torch.empty(0, 64, dtype=BF16, device="cuda")
    r = pkg.add_rmsnorm(x, torch.ones(64, device="cuda"), quant="mx")
    assert r.y.shape == (0, 64) and r.q_scales.shape == (0, 2)
    r = pkg.route_logits(torch.empty(0, 8, device="cuda"), 2, counts=torch.full((8,), 5, dtype=torch.int32, device="cuda"))
    assert (r.counts == 0).all() and r.topk_i.shape == (0, 2)
    g = _gen(0)
    codes, scales = _weights(g, (), 16, 64, "mxfp4", 32)
    assert pkg.w4_matvec(x, codes, scales).shape == (0, 16)
