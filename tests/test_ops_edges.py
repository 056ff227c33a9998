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


# -- w4_matvec: x and scales of any size ----------------------------------------------


def _wide_x(g, rows, K, lo, hi):
    """bf16 values whose exponents are spread over lo..hi inside every group of 32."""
    e = lo + (hi - lo) * torch.rand(rows, K, generator=g, device="cuda", dtype=torch.float64)
    sign = torch.randint(0, 2, (rows, K), generator=g, device="cuda").double() * 2 - 1
    return (sign * torch.exp2(e)).to(BF16)


def _zero_codes(codes, where, fmt):
    """Clears the weights of the columns `where` (bool [K])."""
    zero = 8 if fmt == "int4" else 0
    lo, hi = codes & 15, codes >> 4
    lo[..., where[0::2]] = zero
    hi[..., where[1::2]] = zero
    return lo | hi << 4


def test_matvec_a_small_value_beside_a_large_one():
    """What is left of 2^k beside 1 where the weight of the large one is zero."""
    codes = torch.zeros(16, 16, dtype=torch.uint8, device="cuda")
    codes[:, 0] = 0x20  # 0 in column 0, 1.0 in column 1
    scales = torch.full((16, 1), 127, dtype=torch.uint8, device="cuda")
    x = torch.zeros(127, 32, dtype=BF16, device="cuda")
    x[:, 0] = torch.exp2(torch.arange(1, 128, device="cuda").double()).to(BF16)
    x[:, 1] = 1.6015625
    assert (pkg.w4_matvec(x, codes, scales, dtype=F32) == 1.6015625).all()
    x[:, 1] = -(2.0**-126)
    assert (pkg.w4_matvec(x, codes, scales, dtype=F32) == -(2.0**-126)).all()


@pytest.mark.parametrize("fmt,group", [("mxfp4", 32), ("int4", 32), ("int4", 128)])
@pytest.mark.parametrize("N,K,M", [(17, 32, 1), (40, 416, 3), (12001, 160, 4), (48, 2880, 9), (300, 6144, 2), (33, 16384, 4)])
@pytest.mark.parametrize("lo,hi", [(-60, 60), (-120, -40), (-126, 100)])
def test_matvec_bf16_of_any_size_inside_a_group(fmt, group, N, K, M, lo, hi):
    """Exponents spread inside every group, the largest values on weights of zero in some of the columns."""
    if K % group:
        K = -(-K // group) * group
    g = _gen(N + K + M + lo)
    codes, scales = _weights(g, (), N, K, fmt, group)
    x = _wide_x(g, M, K, lo, hi)
    # columns that are large in the first row have no weights: that row's result is what is left
    large = x[0].double().abs() > 2.0 ** ((lo + hi) / 2 - 20)
    codes = _zero_codes(codes, large, fmt)
    x[-1, ::3] = 0
    y = pkg.w4_matvec(x, codes, scales, dtype=F32)
    _check_matvec(y, x.double(), codes, scales, None, group, None, 1)


def test_matvec_mixed_rows_keep_their_bits():
    """A row that spans many powers of two beside ordinary ones: each row as alone, whatever the batch and the ring."""
    g = _gen(31)
    for n, N, K in ((4, 3000, 544), (3, 100, 11264)):
        codes, scales = _weights(g, (n,), N, K, "mxfp4", 32)
        x = _randn(g, 12, K).to(BF16)
        x[1] = _wide_x(g, 1, K, -90, 90)[0]
        x[6, 64:] = _wide_x(g, 1, K, -90, 90)[0, 64:]
        x[7] = 0
        ids = torch.tensor([0, 1, 1, 0, 2, 1, 1, 1, 0, 1, 1, 1], dtype=torch.int32, device="cuda")
        y = pkg.w4_matvec(x, codes, scales, ids=ids, dtype=F32)
        _check_matvec(y, x.double(), codes, scales, None, 32, ids, 1)
        for m in range(12):
            e = int(ids[m])
            assert torch.equal(y[m:m + 1], pkg.w4_matvec(x[m:m + 1], codes[e], scales[e], dtype=F32))


@pytest.mark.parametrize("P", [1, 4])
def test_matvec_large_x_times_small_scales(P):
    """Products whose parts leave fp32 although they do not."""
    g = _gen(13)
    N, K = 80, 256
    codes, scales = _weights(g, (), N, K, "mxfp4", 32)
    x = (_randn(g, P, K).clamp(-3.9, 3.9).double() * 2.0**125).to(BF16)
    for shift in (-60, -100):  # scales 2^(-8..-4) more
        s = (scales.int() + shift).to(torch.uint8)
        _check_matvec(pkg.w4_matvec(x, codes, s, dtype=F32), x.double(), codes, s, None, 32, None, 1)
    x = (_randn(g, P, K).double() * 2.0**-127).to(BF16)  # the smallest are subnormal
    for shift in (60, 130):
        s = (scales.int() + shift).to(torch.uint8)
        _check_matvec(pkg.w4_matvec(x, codes, s, dtype=F32), x.double(), codes, s, None, 32, None, 1)


@pytest.mark.parametrize("fmt", ["mxfp4", "int4"])
def test_matvec_every_x_scale_times_its_counterpart(fmt):
    """e4m3 rows whose MX scale and weight scale are far apart and meet around 1; fp32 scales likewise."""
    g = _gen(17)
    K, R = 64, 255
    q = _randn(g, R, K).to(torch.float8_e4m3fn)
    sx = torch.arange(R, device="cuda").to(torch.uint8)
    codes = torch.randint(0, 256, (R, 16, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    back = (254 - sx.int()).clamp(1, 254)
    if fmt == "mxfp4":
        scales = back.to(torch.uint8)[:, None, None].expand(R, 16, K // 32).contiguous()
    else:
        scales = torch.exp2(back.double() - 127).to(BF16)[:, None, None].expand(R, 16, K // 32).contiguous()
    ids = torch.arange(R, dtype=torch.int32, device="cuda")
    x64 = q.double() * torch.exp2(sx.double() - 127)[:, None]
    y = pkg.w4_matvec(q, codes, scales, x_scales=sx[:, None].expand(R, K // 32).contiguous(), ids=ids, dtype=F32)
    _check_matvec(y, x64, codes, scales, None, 32, ids, 1)
    row = torch.exp2(sx.double() - 127).float()[:, None].contiguous()
    y = pkg.w4_matvec(q, codes, scales, x_scales=row, ids=ids, dtype=F32)
    _check_matvec(y, x64, codes, scales, None, 32, ids, 1)


def test_matvec_x_scales_of_zero_infinity_and_nan():
    codes = torch.full((16, 32), 0x22, dtype=torch.uint8, device="cuda")  # 1.0 everywhere
    scales = torch.full((16, 2), 127, dtype=torch.uint8, device="cuda")
    q = torch.ones(4, 64, device="cuda").to(torch.float8_e4m3fn)
    s = torch.tensor([[0.0, 1.0], [math.inf, 1.0], [math.nan, 1.0], [-2.0, 0.5]], device="cuda")
    y = pkg.w4_matvec(q, codes, scales, x_scales=s, dtype=F32)
    assert (y[0] == 32).all() and (y[1] == math.inf).all() and y[2].isnan().all() and (y[3] == -48).all()


@pytest.mark.parametrize("fmt,K", [("mxfp4", 544), ("int4", 544), ("mxfp4", 11264)])
@pytest.mark.parametrize("kind", ["values", "group", "e4m3"])
def test_matvec_far_rows_through_chosen_matrices(fmt, K, kind):
    """Rows that need the slower path, shared by several matrices, with a bias and the SwiGLU, beside rows that do not
    and rows without a matrix."""
    g = _gen(K)
    n, N, rows, rpx = 5, 70, 6, 3
    codes, scales = _weights(g, (n,), N, K, fmt, 32)
    bias = 0.1 * _randn(g, n, N)
    ids = torch.tensor([0, 4, 4, -1, 4, 2, 4, 4, 0, 9, 3, 3, 4, 0, 1, 2, 2, 2], dtype=torch.int32, device="cuda")
    wide = _randn(g, rows, K + 8).to(BF16)
    x, xs, x64 = wide[:, :K], None, None
    if kind == "values":
        x[1, 5::96] = 2.0**-70
        x[4, K - 1] = -(2.0**-40)
    elif kind == "group":
        x[1, 32:96] *= 2.0**-110
        x[4, K - 32:] *= 2.0**120
        scales[:, :, K // 32 - 1:] = 10 if fmt == "mxfp4" else 2.0**-115
    else:
        x = x.float().to(torch.float8_e4m3fn)
        e = torch.zeros(rows, K // 32, device="cuda")
        e[1, 1:3] = -112
        e[4, -1] = 110
        xs = (e + 127).to(torch.uint8)
        scales[:, :, K // 32 - 1:] = 10 if fmt == "mxfp4" else 2.0**-115
        x64 = x.double() * torch.exp2(e.double()).repeat_interleave(32, 1)
    x64 = x.double() if x64 is None else x64
    for act in (None, (1.702, 7.0)):
        y = pkg.w4_matvec(x, codes, scales, bias, x_scales=xs, ids=ids, rows_per_x=rpx, swiglu=act, dtype=F32)
        _check_matvec(y, x64, codes, scales, bias, 32, ids, rpx, act)
        assert (y[[3, 9]] == 0).all()
        for m in (1, 4, 13):
            one = pkg.w4_matvec(x[m // rpx:m // rpx + 1], codes, scales, bias, x_scales=None if xs is None else xs[m // rpx:m // rpx + 1],
                                ids=ids[m:m + 1], swiglu=act, dtype=F32)
            assert torch.equal(y[m:m + 1], one)


# -- calls beside other work ---------------------------------------------------------------


def test_inputs_of_a_call_on_another_stream_may_be_dropped():
    """The memory of an input that the caller lets go is not handed out before the call on the other stream has read it."""
    g = _gen(23)
    s = torch.cuda.Stream()
    T, H, E = 64, 4096, 128
    w = torch.ones(H, device="cuda")
    codes, scales = _weights(g, (), 512, H, "mxfp4", 32)
    x, logits = _randn(g, T, H), _randn(g, T, E)
    xb = x.to(BF16)
    want = pkg.add_rmsnorm(x, w, x, quant="mx"), pkg.route_logits(logits, 4), (pkg.w4_matvec(xb, codes, scales),)
    calls = [lambda: pkg.add_rmsnorm(x.clone(), w, x.clone(), quant="mx", stream=s),
             lambda: pkg.route_logits(logits.clone(), 4, stream=s),
             lambda: (pkg.w4_matvec(xb.clone(), codes, scales, stream=s),)]
    for call, ref_out in zip(calls, want):
        for t in (x, xb, logits):
            t.clone()  # the sizes that the call's temporaries have are in the allocator's lists
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(20_000_000)  # about 10 ms
        got = call()
        s_busy = not s.query()
        trash = [torch.full_like(t, 7.0) for t in (x, x, xb, logits) for _ in range(2)]
        torch.cuda.synchronize()
        assert s_busy, "the call has to be waiting while its inputs' memory could be reused"
        for a, b in zip(got, ref_out):
            assert (a is None and b is None) or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        del trash


def test_a_refused_launch_leaves_no_error_behind():
    """CUDA refuses work on the legacy stream while an ordinary stream of the thread is being captured.  The call
    says so, and the next call of the library starts from a clean state."""
    from cuda.bindings import runtime as rt

    from gpt_oss_amd_b200 import capi

    x, w = torch.ones(4, 64, device="cuda"), torch.ones(64, device="cuda")
    y = torch.empty(4, 64, device="cuda")
    logits, ti, tw = torch.ones(4, 8, device="cuda"), torch.empty(4, 2, dtype=torch.int32, device="cuda"), torch.empty(4, 2, device="cuda")
    q, codes, scales = x.to(BF16), torch.zeros(16, 32, dtype=torch.uint8, device="cuda"), torch.zeros(16, 2, dtype=torch.uint8, device="cuda")
    out = torch.empty(4, 16, device="cuda")
    blocks = torch.zeros(4, 2, 16, dtype=torch.uint8, device="cuda")
    sc = torch.full((4, 2), 127, dtype=torch.uint8, device="cuda")
    un = torch.empty(4, 64, dtype=torch.int16, device="cuda")
    L = capi.lib()
    norm = capi.packer(capi.AddRmsnormArgs)(4, 64, x.data_ptr(), 0, 64, 0, 0, 0, 0, 0, w.data_ptr(), 0, 1e-5, y.data_ptr(), 0, 64, 0, 0, 0, 0)
    route = capi.packer(capi.RouteLogitsArgs)(4, 8, 2, logits.data_ptr(), 0, 8, 0, 0, 1, 1, 1, 1, 1.0, ti.data_ptr(), tw.data_ptr(), 0)
    matvec = capi.packer(capi.W4MatvecArgs)(0, 32, 1, 16, 64, codes.data_ptr(), scales.data_ptr(), 0, q.data_ptr(), 1, 64, 0, 0, 4, 1, 0,
                                            0, 0.0, 0.0, out.data_ptr(), 0, 16)
    torch.cuda.synchronize()
    for fn, args in ((L.moe_b200_add_rmsnorm, norm), (L.moe_b200_route_logits, route), (L.moe_b200_w4_matvec, matvec)):
        err, stream = rt.cudaStreamCreate()
        assert err == rt.cudaError_t.cudaSuccess
        err, = rt.cudaStreamBeginCapture(stream, rt.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal)
        assert err == rt.cudaError_t.cudaSuccess
        status = fn(args, None)
        text = L.moe_b200_last_error(None)
        rt.cudaStreamEndCapture(stream)
        rt.cudaGetLastError()
        rt.cudaStreamDestroy(stream)
        assert status == capi.ERR_CUDA and b"captur" in text, (status, text)
        assert fn(args, None) == capi.OK
        status = L.moe_b200_mxfp4_unpack(blocks.data_ptr(), sc.data_ptr(), 4, 2, un.data_ptr(), None)
        assert status == capi.OK, L.moe_b200_last_error(None)
    torch.cuda.synchronize()


def test_branches_of_a_captured_graph_join():
    """Two operators on streams of their own, and one behind both, behind a copy and in front of everything: captured
    and replayed on new inputs."""
    g = _gen(41)
    T, H, E, K = 8, 576, 32, 4
    w = 1 + 0.1 * _randn(g, H)
    codes, scales = _weights(g, (E,), 300, H, "mxfp4", 32)
    x, logits = _randn(g, T, H), _randn(g, T, E)
    keep = torch.empty(T * K, 300, device="cuda")

    def step(main, side):
        if side is not main:
            side.wait_stream(main)
        with torch.cuda.stream(side):
            r = pkg.route_logits(logits, K, counts=True)
        n = pkg.add_rmsnorm(x, w, quant="mx")
        if side is not main:
            main.wait_stream(side)
        y = pkg.w4_matvec(n.q, codes, scales, x_scales=n.q_scales, ids=r.topk_i.view(-1), rows_per_x=K, dtype=F32)
        keep.copy_(y)
        z = pkg.add_rmsnorm(keep, torch.ones(300, device="cuda"), keep, dtype=F32)
        return r.topk_i, r.counts, n.y, y, z.y

    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        step(main, side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        got = step(main, side)
    for _ in range(5):
        x.normal_(generator=g)
        logits.normal_(generator=g)
        graph.replay()
        s = torch.cuda.current_stream()
        for a, b in zip(got, step(s, s)):
            assert torch.equal(a, b)


def _three_calls():
    x = torch.ones(4, 64, device="cuda", dtype=BF16)
    n = pkg.add_rmsnorm(x, torch.ones(64, device="cuda"))
    r = pkg.route_logits(n.y, 4, counts=True)
    codes, scales = torch.zeros(16, 32, dtype=torch.uint8, device="cuda"), torch.zeros(16, 2, dtype=torch.uint8, device="cuda")
    return pkg.w4_matvec(n.y, codes, scales), r


_EDGES = """
import torch
import sys
sys.path.insert(0, "tests")
from cuda.bindings import runtime as rt
from test_ops_edges import _three_calls
_three_calls()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph(keep_graph=True)
with torch.cuda.graph(g):
    _three_calls()
raw = rt.cudaGraph_t(init_value=g.raw_cuda_graph())
err, _, _, _, n = rt.cudaGraphGetEdges_v2(raw, 0)
err, _, _, data, n = rt.cudaGraphGetEdges_v2(raw, n)
assert err == rt.cudaError_t.cudaSuccess
print("programmatic", sum(int(d.type) == int(rt.cudaGraphDependencyType.cudaGraphDependencyTypeProgrammatic) for d in data))
"""


@pytest.mark.parametrize("off", [False, True])
def test_the_switch_for_dependent_launches_reaches_the_operators(off):
    """MOE_B200_NO_PDL: every kernel behind the end of the one in front."""
    import os
    import subprocess
    import sys

    env = {k: v for k, v in os.environ.items() if k != "MOE_B200_NO_PDL"}
    if off:
        env["MOE_B200_NO_PDL"] = "1"
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _EDGES], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    n = int(r.stdout.split("programmatic")[1])
    assert n == 0 if off else n >= 2
