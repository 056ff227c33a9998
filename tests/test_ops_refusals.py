"""The stand-alone operators refuse wrong arguments with a status and a text, before anything is launched:
no GPU is needed (the pointers below are never followed)."""
import ctypes

import pytest
import torch

import gpt_oss_amd_b200 as pkg
from gpt_oss_amd_b200 import capi

A = 4096  # an aligned address


def _norm(**kw):
    a = dict(T=4, H=64, x=A, xt=capi.DTYPE_BF16, xs=64, r=A, rt=capi.DTYPE_F32, rs=64, ro=A, ros=64, w=A, wt=capi.DTYPE_F32,
             eps=1e-5, y=A, yt=capi.DTYPE_BF16, ys=64, q=A, qs=64, sc=A, kind=capi.SCALE_ROW)
    a.update(kw)
    return capi.lib().moe_b200_add_rmsnorm(ctypes.byref(capi.AddRmsnormArgs(*a.values())), None)


def _route(**kw):
    a = dict(T=4, E=64, K=4, l=A, dt=capi.DTYPE_F32, s=64, score=capi.SCORE_SOFTMAX, bias=None, ng=1, kg=1, gt=1, rn=1, scale=1.0,
             i=A, w=A, c=None)
    a.update(kw)
    return capi.lib().moe_b200_route_logits(ctypes.byref(capi.RouteLogitsArgs(*a.values())), None)


def _matvec(mat=None, **kw):
    m = dict(format=capi.W4_MXFP4, group=32, n_mats=1, rows=64, cols=64, codes=A, scales=A, bias=A)
    m.update(mat or {})
    a = dict(x=A, xt=capi.DTYPE_BF16, xs=64, sc=None, kind=capi.SCALE_NONE, M=4, rpx=1, ids=None, sw=0, al=1.702, li=7.0, out=A,
             ot=capi.DTYPE_BF16, os=64)
    a.update(kw)
    return capi.lib().moe_b200_w4_matvec(ctypes.byref(capi.W4MatvecArgs(capi.W4Matrix(**m), *a.values())), None)


def test_null_arguments_are_refused():
    L = capi.lib()
    for fn in (L.moe_b200_add_rmsnorm, L.moe_b200_route_logits, L.moe_b200_w4_matvec):
        assert fn(None, None) == capi.ERR_INVALID


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(H=0), dict(H=32769), dict(xt=3), dict(rt=9), dict(wt=-1), dict(yt=3), dict(eps=-1.0), dict(eps=float("nan")),
    dict(eps=float("inf")), dict(y=None, q=None), dict(r=None), dict(kind=0), dict(kind=6), dict(x=None), dict(w=None), dict(sc=None),
    dict(xs=-1), dict(rs=-64), dict(ros=63), dict(ys=63), dict(qs=63), dict(x=A + 1), dict(w=A + 2), dict(r=A + 2), dict(ro=A + 1),
    dict(y=A + 1), dict(sc=A + 2)])
def test_add_rmsnorm_refuses(kw):
    assert _norm(**kw) == capi.ERR_INVALID
    assert b"add_rmsnorm" in capi.lib().moe_b200_last_error(None)


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(T=16777217), dict(E=0), dict(E=513), dict(K=0), dict(K=17), dict(E=3, K=4), dict(dt=3), dict(score=2), dict(ng=0), dict(ng=3),
    dict(E=66, ng=33), dict(ng=4, kg=0), dict(ng=4, kg=5), dict(ng=4, kg=1, gt=0), dict(ng=4, kg=1, gt=3), dict(ng=32, kg=1, gt=1),
    dict(E=32, ng=32, kg=8, gt=2), dict(scale=float("nan")), dict(scale=float("inf")), dict(l=None), dict(i=None), dict(w=None),
    dict(s=-1), dict(l=A + 2), dict(bias=A + 1), dict(i=A + 1), dict(w=A + 2), dict(c=A + 3)])
def test_route_logits_refuses(kw):
    assert _route(**kw) == capi.ERR_INVALID
    assert b"route_logits" in capi.lib().moe_b200_last_error(None)


@pytest.mark.parametrize("mat,kw", [
    (dict(format=2), {}), (dict(group=64), {}), (dict(format=1, group=16), {}), (dict(rows=0), {}), (dict(rows=4194305), {}),
    (dict(cols=0), {}), (dict(cols=48), {}), (dict(cols=16416), {}), (dict(format=1, group=128), {}), (dict(n_mats=0), {}),
    (dict(n_mats=2), {}), (dict(codes=None), {}), (dict(scales=None), {}), (dict(codes=A + 8), {}), (dict(bias=A + 2), {}),
    (dict(format=1, scales=A + 1), {}),
    ({}, dict(M=-1)), ({}, dict(M=257)), ({}, dict(rpx=0)), ({}, dict(xt=capi.DTYPE_F32)), ({}, dict(xt=capi.DTYPE_E4M3)),
    ({}, dict(kind=capi.SCALE_ROW, sc=A)), ({}, dict(xt=capi.DTYPE_E4M3, kind=6, sc=A)), ({}, dict(xt=capi.DTYPE_E4M3, kind=1)),
    ({}, dict(xt=capi.DTYPE_E4M3, kind=1, sc=A + 2)), ({}, dict(ot=capi.DTYPE_E4M3)), (dict(rows=63), dict(sw=1)),
    ({}, dict(sw=1, li=-1.0)), ({}, dict(sw=1, li=float("nan"))), ({}, dict(sw=1, al=float("nan"))), ({}, dict(x=None)),
    ({}, dict(out=None)), ({}, dict(xs=-64)), ({}, dict(os=63)), ({}, dict(x=A + 8)), ({}, dict(xs=68)), ({}, dict(out=A + 1)),
    ({}, dict(ids=A + 2))])
def test_w4_matvec_refuses(mat, kw):
    assert _matvec(mat, **kw) == capi.ERR_INVALID
    assert b"w4_matvec" in capi.lib().moe_b200_last_error(None)


def test_packed_arguments_are_the_struct():
    for cls in (capi.AddRmsnormArgs, capi.RouteLogitsArgs, capi.W4MatvecArgs):
        flat = []

        def fill(t, at):
            out = []
            for _, ft in t._fields_:
                if issubclass(ft, ctypes.Structure):
                    out.append(fill(ft, at))
                else:
                    at[0] += 1
                    v = float(at[0]) if ft is ctypes.c_float else at[0]
                    flat.append(v)
                    out.append(v)
            return t(*out)

        s = fill(cls, [0])
        packed, names = capi.packer(cls)(*flat), [n for n, _ in cls._fields_]
        back = cls.from_buffer_copy(packed)
        for n in names:
            a, b = getattr(s, n), getattr(back, n)
            assert a == b if not isinstance(a, ctypes.Structure) else bytes(a)[:20] == bytes(b)[:20] and a.bias == b.bias


def test_nothing_to_do_is_fine():
    assert _norm(T=0, x=None, y=None) == capi.OK
    assert _route(T=0, l=None, i=None, w=None) == capi.OK
    assert _matvec(M=0, x=None, out=None) == capi.OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_no_cpu_path():
    assert _norm() == capi.ERR_NO_DEVICE
    assert _route() == capi.ERR_NO_DEVICE
    assert _matvec() == capi.ERR_NO_DEVICE


def test_error_text_belongs_to_the_calling_thread():
    import threading

    assert _norm(H=0) == capi.ERR_INVALID
    seen = []
    t = threading.Thread(target=lambda: seen.append((_route(K=0), capi.lib().moe_b200_last_error(None))))
    t.start()
    t.join()
    assert seen[0][0] == capi.ERR_INVALID and b"route_logits" in seen[0][1]
    assert b"add_rmsnorm" in capi.lib().moe_b200_last_error(None)


def test_python_wrappers_refuse():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.ones(64)
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    q = torch.zeros(4, 64, dtype=torch.float8_e4m3fn)
    for call in [
        lambda: pkg.add_rmsnorm(x, w),  # no CPU path
        lambda: pkg.add_rmsnorm(x[0], w),
        lambda: pkg.add_rmsnorm(x.to(torch.float64), w),
        lambda: pkg.add_rmsnorm(x.t(), w),
        lambda: pkg.add_rmsnorm(x, w[:63]),
        lambda: pkg.add_rmsnorm(x, w, torch.zeros(3, 64)),
        lambda: pkg.add_rmsnorm(x, w, residual_out=x),
        lambda: pkg.add_rmsnorm(x, w, x, residual_out=torch.zeros(4, 64)),
        lambda: pkg.add_rmsnorm(x, w, quant=16),
        lambda: pkg.add_rmsnorm(x, w, q=q),
        lambda: pkg.add_rmsnorm(x, w, quant="mx", q_scales=torch.zeros(4, 2)),
        lambda: pkg.route_logits(x, 4),
        lambda: pkg.route_logits(x[0], 4),
        lambda: pkg.route_logits(x, 4, score="max"),
        lambda: pkg.route_logits(x, 4, bias=torch.zeros(63)),
        lambda: pkg.route_logits(x, 4, topk_i=torch.zeros(4, 4)),
        lambda: pkg.w4_matvec(x, codes, scales),
        lambda: pkg.w4_matvec(x.float(), codes, scales),
        lambda: pkg.w4_matvec(x, codes[:, :31], scales),
        lambda: pkg.w4_matvec(x, codes, scales[:7]),
        lambda: pkg.w4_matvec(x, codes, scales.float()),
        lambda: pkg.w4_matvec(x, codes[None], scales[None]),
        lambda: pkg.w4_matvec(x, codes[None], scales[None], ids=torch.zeros(5, dtype=torch.int32)),
        lambda: pkg.w4_matvec(x, codes, scales, ids=torch.zeros(4, dtype=torch.int64)),
        lambda: pkg.w4_matvec(q, codes, scales, x_scales=torch.zeros(4, 5)),
        lambda: pkg.w4_matvec(x, codes, scales, rows_per_x=0),
        lambda: pkg.w4_matvec(x, codes, scales, out=torch.zeros(4, 7)),
    ]:
        with pytest.raises(ValueError):
            call()


def test_numbers_that_do_not_fit_the_structs():
    pack, n = capi.packer(capi.RouteLogitsArgs), len(capi.RouteLogitsArgs._fields_)

    def with_value(at, v):
        values = [0] * n
        values[at] = v
        return pack(*values)

    for at, v in [(0, 2**31), (1, -2**31 - 1), (5, 2**63), (2, 1.5)]:
        with pytest.raises(ValueError):
            with_value(at, v)
    # a float too large becomes infinity, as in C, which the library refuses
    assert capi.RouteLogitsArgs.from_buffer_copy(with_value(12, 1e300)).scale == float("inf")
    assert _route(scale=float("inf")) == capi.ERR_INVALID
    assert _norm(eps=float("inf")) == capi.ERR_INVALID
