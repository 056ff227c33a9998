"""The checks of the Python wrappers of the stand-alone operators, each by the text that names the argument.  No GPU is
needed: tensors of the host stand in for those of a device, and the call of the library is cut off."""
import pytest
import torch

from gpt_oss_amd_b200 import capi, ops


class Reached(Exception):
    """All checks passed."""


@pytest.fixture(autouse=True)
def host_tensors(monkeypatch):
    def call(name, dev, args):
        raise Reached(name)

    monkeypatch.setattr(ops, "_device", lambda t: -1)  # what get_device() says of the host's
    monkeypatch.setattr(ops, "_call", call)


T, H, E, N = 4, 64, 16, 8
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _norm(**kw):
    a = dict(x=torch.zeros(T, H, dtype=BF16), weight=torch.ones(H))
    a.update(kw)
    return ops.add_rmsnorm(a.pop("x"), a.pop("weight"), **a)


def _route(**kw):
    a = dict(logits=torch.zeros(T, E), k=4)
    a.update(kw)
    return ops.route_logits(a.pop("logits"), a.pop("k"), **a)


def _matvec(**kw):
    a = dict(x=torch.zeros(T, H, dtype=BF16), codes=torch.zeros(N, H // 2, dtype=torch.uint8), scales=torch.zeros(N, H // 32, dtype=torch.uint8))
    a.update(kw)
    return ops.w4_matvec(a.pop("x"), a.pop("codes"), a.pop("scales"), **a)


def _stack(n=3):
    return dict(codes=torch.zeros(n, N, H // 2, dtype=torch.uint8), scales=torch.zeros(n, N, H // 32, dtype=torch.uint8))


def _strided(rows, cols, dtype):
    """Columns that are not neighbours."""
    return torch.zeros(rows, 2 * cols, dtype=dtype)[:, ::2]


@pytest.mark.parametrize("call,kw", [
    (_norm, dict()), (_norm, dict(residual=torch.zeros(T, H), quant="mx")), (_norm, dict(x=torch.zeros(T, H + 3)[:, :H], quant="row")),
    (_norm, dict(residual=torch.zeros(T, H), residual_out=torch.zeros(T, H), out=torch.zeros(T, H), q=torch.zeros(T, H).to(E4M3),
                 q_scales=torch.zeros(T, 1), quant=64)),
    (_norm, dict(quant="mx", q_scales=torch.zeros(T, 2, dtype=torch.uint8))), (_norm, dict(dtype=None, quant=32)),
    (_route, dict()), (_route, dict(k=E, bias=torch.zeros(E), counts=True)), (_route, dict(counts=torch.zeros(E, dtype=torch.int32))),
    (_route, dict(topk_i=torch.zeros(T, 4, dtype=torch.int32), topk_w=torch.zeros(T, 4), score="sigmoid")),
    (_matvec, dict()), (_matvec, dict(codes=torch.zeros(N, H // 32, 16, dtype=torch.uint8))), (_matvec, dict(rows_per_x=64)),
    (_matvec, dict(scales=torch.zeros(N, 1, dtype=BF16))), (_matvec, dict(bias=torch.zeros(N), swiglu=(1.702, 7.0), out=torch.zeros(T, N // 2))),
    (_matvec, dict(ids=torch.zeros(T, dtype=torch.int32), **_stack())), (_matvec, dict(ids=torch.zeros(7, dtype=torch.int32), rows_per_x=2)),
    (_matvec, dict(x=torch.zeros(T, H).to(E4M3), x_scales=torch.zeros(T, 2))),
    (_matvec, dict(x=torch.zeros(T, H).to(E4M3), x_scales=torch.zeros(T, 2, dtype=torch.uint8)))])
def test_right_arguments_reach_the_library(call, kw):
    with pytest.raises(Reached):
        call(**kw)


@pytest.mark.parametrize("text,call,kw", [
    ("x: needs two", _norm, dict(x=torch.zeros(H))), ("^x: needs contiguous rows", _norm, dict(x=torch.zeros(T, H, dtype=torch.float64))),
    ("^x: needs contiguous rows", _norm, dict(x=_strided(T, H, BF16))), ("^weight: needs", _norm, dict(weight=torch.ones(H - 1))),
    ("^weight: needs", _norm, dict(weight=torch.ones(2 * H)[::2])), ("^residual: needs", _norm, dict(residual=torch.zeros(T - 1, H))),
    ("^residual: needs", _norm, dict(residual=torch.zeros(T, H, dtype=torch.int32))),
    ("residual_out without", _norm, dict(residual_out=torch.zeros(T, H))),
    ("residual_out: needs residual's", _norm, dict(residual=torch.zeros(T, H), residual_out=torch.zeros(T, H, dtype=BF16))),
    ("^residual_out: needs contiguous rows", _norm, dict(residual=torch.zeros(T, H), residual_out=torch.zeros(T + 1, H))),
    ("^out: needs", _norm, dict(out=torch.zeros(T, H + 1))), ("^out: needs", _norm, dict(dtype=torch.int8)),
    ("quant: one of", _norm, dict(quant=16)), ("q without quant", _norm, dict(q=torch.zeros(T, H).to(E4M3))),
    ("q without quant", _norm, dict(q_scales=torch.zeros(T, 1))), ("^q: needs", _norm, dict(quant="row", q=torch.zeros(T, H))),
    ("^q_scales: needs", _norm, dict(quant="mx", q_scales=torch.zeros(T, 2))), ("^q_scales: needs", _norm, dict(quant=32, q_scales=torch.zeros(T, 1))),
    ("does not fit", _norm, dict(eps="1")),
    ("logits: needs two", _route, dict(logits=torch.zeros(E))), ("^logits: needs contiguous", _route, dict(logits=_strided(T, E, torch.float32))),
    ("k: needs 1", _route, dict(k=0)), ("k: needs 1", _route, dict(k=E + 1)), ("score: one of", _route, dict(score="max")),
    ("^bias: needs", _route, dict(bias=torch.zeros(E - 1))), ("^bias: needs", _route, dict(bias=torch.zeros(E, dtype=BF16))),
    ("^topk_i: needs", _route, dict(topk_i=torch.zeros(T, 4))), ("^topk_w: needs", _route, dict(topk_w=torch.zeros(T, 3))),
    ("^counts: needs", _route, dict(counts=torch.zeros(E))), ("does not fit", _route, dict(n_groups=2**40)), ("does not fit", _route, dict(topk_groups=1.5)),
    ("x: needs two", _matvec, dict(x=torch.zeros(H, dtype=BF16))), ("^x: needs contiguous", _matvec, dict(x=torch.zeros(T, H))),
    ("^x: needs contiguous", _matvec, dict(x=_strided(T, H, BF16))), ("scales: needs", _matvec, dict(scales=torch.zeros(N, dtype=torch.uint8))),
    ("scales: their number", _matvec, dict(scales=torch.zeros(N, 3, dtype=torch.uint8))), ("^scales: needs", _matvec, dict(scales=torch.zeros(N, 2))),
    ("^codes: needs", _matvec, dict(codes=torch.zeros(N, H // 2 - 1, dtype=torch.uint8))),
    ("^codes: needs", _matvec, dict(scales=torch.zeros(N - 1, H // 32, dtype=torch.uint8))),
    ("^codes: needs", _matvec, dict(codes=torch.zeros(N, H // 2, dtype=torch.int8))), ("^bias: needs", _matvec, dict(bias=torch.zeros(N + 1))),
    ("rows_per_x: at least", _matvec, dict(rows_per_x=0)), ("a stack of matrices", _matvec, _stack()),
    ("ids: one per row", _matvec, dict(ids=torch.zeros(5, dtype=torch.int32), **_stack())),
    ("ids: one per row", _matvec, dict(ids=torch.zeros(6, dtype=torch.int32), rows_per_x=2)),
    ("^ids: needs", _matvec, dict(ids=torch.zeros(T, dtype=torch.int64))), ("^ids: needs", _matvec, dict(ids=torch.zeros(2, 2, dtype=torch.int32))),
    ("x_scales: needs two", _matvec, dict(x=torch.zeros(T, H).to(E4M3), x_scales=torch.zeros(T))),
    ("x_scales: one per", _matvec, dict(x=torch.zeros(T, H).to(E4M3), x_scales=torch.zeros(T, 5))),
    ("^x_scales: needs", _matvec, dict(x=torch.zeros(T, H).to(E4M3), x_scales=torch.zeros(T - 1, 2))),
    ("^x_scales: needs", _matvec, dict(x=torch.zeros(T, H).to(E4M3), x_scales=torch.zeros(T, 2, dtype=BF16))),
    ("at most 256 rows", _matvec, dict(rows_per_x=65)), ("^out: needs", _matvec, dict(out=torch.zeros(T, N - 1))),
    ("^out: needs", _matvec, dict(out=torch.zeros(T, N), swiglu=(1.702, 7.0))), ("^out: needs", _matvec, dict(dtype=E4M3))])
def test_wrong_arguments_are_refused_by_name(text, call, kw):
    with pytest.raises(ValueError, match=text):
        call(**kw)


@pytest.mark.parametrize("call,x", [(_norm, "x"), (_route, "logits"), (_matvec, "x")])
def test_tensors_of_two_devices(call, x, monkeypatch):
    """The first tensor's device is the call's."""
    monkeypatch.setattr(ops, "_device", lambda t: 0)
    with pytest.raises(ValueError, match=f"^{x}: needs .* cuda:0"):
        call()


def test_a_stream_of_another_device():
    from types import SimpleNamespace

    s = SimpleNamespace(device=torch.device("cuda", 0))
    for call in (_norm, _route, _matvec):
        with pytest.raises(ValueError, match="stream: needs the device"):
            call(stream=s)


def test_every_refusal_of_the_library_is_an_error(monkeypatch):
    """The status of a call becomes an exception with the library's text."""
    with pytest.raises(capi.MoEError, match="hidden_dim"):
        capi.check(capi.lib().moe_b200_add_rmsnorm(capi.packer(capi.AddRmsnormArgs)(*[0] * 20), None))
