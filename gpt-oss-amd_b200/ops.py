"""The stand-alone operators of the C ABI on torch tensors.

``add_rmsnorm``, ``route_logits`` and ``w4_matvec`` are the steps around and beside the MoE
block for tensors of the caller's own (include/moe_b200.h): they take no handle and keep
nothing.  Results go where the caller says or into new tensors; the calls are asynchronous
on ``stream`` (a ``torch.cuda.Stream``; by default the current stream of the tensors' device).
A call on a ``stream`` of its own waits for nothing on the stream that made its inputs: order the two
with ``wait_stream``, as for any torch operator.  Inputs may be dropped after the call: their memory is
kept until ``stream`` has passed it.
A wrong argument raises ``ValueError`` here or ``capi.MoEError`` with the library's text.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import capi

_FLOATS = {torch.float32: capi.DTYPE_F32, torch.bfloat16: capi.DTYPE_BF16, torch.float16: capi.DTYPE_F16}
_X4 = {torch.bfloat16: capi.DTYPE_BF16, torch.float16: capi.DTYPE_F16, torch.float8_e4m3fn: capi.DTYPE_E4M3}
_PACK_NORM = capi.packer(capi.AddRmsnormArgs)
_PACK_ROUTE = capi.packer(capi.RouteLogitsArgs)
_PACK_MATVEC = capi.packer(capi.W4MatvecArgs)
_QUANT = {"row": capi.SCALE_ROW, 32: capi.SCALE_G32, 64: capi.SCALE_G64, 128: capi.SCALE_G128, "mx": capi.SCALE_MX}
_MX_TYPES = (torch.float8_e8m0fnu, torch.uint8)
_F32, _I32, _U8 = (torch.float32,), (torch.int32,), (torch.uint8,)
_E4M3 = {torch.float8_e4m3fn: capi.DTYPE_E4M3}
_W4_SCALES, _X_SCALES = (torch.bfloat16, *_MX_TYPES), (torch.float32, *_MX_TYPES)


class NormResult(NamedTuple):
    y: torch.Tensor | None
    residual: torch.Tensor | None
    q: torch.Tensor | None
    q_scales: torch.Tensor | None


class Routing(NamedTuple):
    topk_i: torch.Tensor
    topk_w: torch.Tensor
    counts: torch.Tensor | None


def _need(ok, text):
    if not ok:
        raise ValueError(text)


# These run in front of kernels of a few microseconds: a tensor's shape, strides and device are asked for once each.


def _wrong(t, name, shape, types, dev, what):
    raise ValueError(f"{name}: needs {what} {tuple(shape)} on cuda:{dev}, one of {[str(d) for d in types]}; "
                     f"got {tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")


def _rows(t, name, shape, types, dev):
    """Checks a 2-d tensor with neighbouring columns; returns its address, its type's code and its row stride."""
    code = types.get(t.dtype)
    if code is None or t.get_device() != dev or t.shape != shape:
        _wrong(t, name, shape, types, dev, "contiguous rows of")
    stride, one = t.stride()
    if one != 1 and shape[1] > 1:
        _wrong(t, name, shape, types, dev, "contiguous rows of")
    return t.data_ptr(), code, stride


def _dense(t, name, shape, types, dev):
    """Checks a contiguous tensor; returns its address."""
    if t.dtype not in types or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        _wrong(t, name, shape, types, dev, "contiguous")
    return t.data_ptr()


def _device(t):
    """The CUDA device index of the first tensor of a call."""
    dev = t.get_device()
    if dev < 0:
        raise ValueError("needs CUDA tensors: there is no CPU path")
    return dev


def _on(stream, fn, x, *args, **kw):
    """The call with `stream` as the current one: new results come from that stream's memory, and the memory of the
    tensors of the caller's is not handed out again before `stream` has passed the call."""
    _need(stream.device == x.device, "stream: needs the device of the tensors")
    with torch.cuda.stream(stream):
        result = fn(x, *args, **kw)
    for t in (x, *args, *kw.values()):
        if isinstance(t, torch.Tensor):
            t.record_stream(stream)
    return result


def _call(name, dev, args):
    fn = getattr(capi.lib(), name)
    raw = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch._C._cuda_getDevice():
        status = fn(args, raw)
    else:
        with torch.cuda.device(dev):
            status = fn(args, raw)
    if status:
        capi.check(status)


def add_rmsnorm(x, weight, residual=None, *, eps=1e-5, dtype=torch.bfloat16, quant=None, residual_out=None, out=None,
                q=None, q_scales=None, stream=None):
    """``r = x + residual``; ``y = r / sqrt(mean(r^2) + eps) * weight`` per row of x [T, H]; y once more as e4m3.

    Returns ``NormResult(y, residual, q, q_scales)``.  ``dtype``: type of y, None for no y
    (``out``: where to).  ``residual``: x's shape, its sum with x goes to ``residual_out`` (which may
    be ``residual`` itself), in residual's type.  ``quant``: "row", 32, 64 or 128 (fp32 scales per row or
    group of columns) or "mx" (e8m0 per 32): q is float8_e4m3fn [T, H], q_scales [T, scales per row]
    float32, with "mx" float8_e8m0fnu (uint8 is taken too)."""
    if stream is not None:
        return _on(stream, add_rmsnorm, x, weight, residual, eps=eps, dtype=dtype, quant=quant, residual_out=residual_out,
                   out=out, q=q, q_scales=q_scales)
    dev = _device(x)
    _need(x.dim() == 2, "x: needs two dimensions")
    shape = x.shape
    T, H = shape
    xp, xt, xs = _rows(x, "x", shape, _FLOATS, dev)
    wp = _dense(weight, "weight", (H,), _FLOATS, dev)
    rp = rop = yp = qp = sp = rt = rs = ros = yt = ys = qs = kind = 0
    if residual is not None:
        rp, rt, rs = _rows(residual, "residual", shape, _FLOATS, dev)
        if residual_out is None:
            residual_out = torch.empty(T, H, dtype=residual.dtype, device=x.device)
        rop, same, ros = _rows(residual_out, "residual_out", shape, _FLOATS, dev)
        if same != rt:
            raise ValueError("residual_out: needs residual's type")
    elif residual_out is not None:
        raise ValueError("residual_out without residual")
    if out is not None or dtype is not None:
        if out is None:
            out = torch.empty(T, H, dtype=dtype, device=x.device)
        yp, yt, ys = _rows(out, "out", shape, _FLOATS, dev)
    if quant is not None:
        kind = _QUANT.get(quant)
        if kind is None:
            raise ValueError(f"quant: one of {list(_QUANT)}")
        n = 1 if quant == "row" else -(-H // (32 if quant == "mx" else quant))
        if q is None:
            q = torch.empty(T, H, dtype=torch.float8_e4m3fn, device=x.device)
        if q_scales is None:
            q_scales = torch.empty(T, n, dtype=torch.float8_e8m0fnu if quant == "mx" else torch.float32, device=x.device)
        qp, _, qs = _rows(q, "q", shape, _E4M3, dev)
        sp = _dense(q_scales, "q_scales", (T, n), _MX_TYPES if quant == "mx" else _F32, dev)
    elif q is not None or q_scales is not None:
        raise ValueError("q without quant")
    _call("moe_b200_add_rmsnorm", dev, _PACK_NORM(
        T, H, xp, xt, xs, rp, rt, rs, rop, ros, wp, _FLOATS[weight.dtype], eps, yp, yt, ys, qp, qs, sp, kind))
    return NormResult(out, residual_out, q, q_scales)


_SCORES = {"softmax": capi.SCORE_SOFTMAX, "sigmoid": capi.SCORE_SIGMOID}


def route_logits(logits, k, *, score="softmax", bias=None, n_groups=1, topk_groups=1, group_top=2, renormalize=True,
                 scale=1.0, counts=False, topk_i=None, topk_w=None, stream=None):
    """The ``k`` experts of each token and their weights from router logits [T, E]; returns
    ``Routing(topk_i int32 [T, k], topk_w float32 [T, k], counts)``.

    ``score`` "softmax" or "sigmoid"; ``bias`` float32 [E] is added for the choice only.  With
    ``n_groups`` > 1 only experts of the ``topk_groups`` best groups take part, a group being scored by
    its ``group_top`` (1 or 2) best experts.  ``renormalize`` divides the weights by their sum, then
    ``scale`` multiplies them.  Ties go to the lower index.  Experts with a logit of -inf or NaN take no
    part; empty slots have index -1 and weight 0.  ``counts``: True or an int32 [E] tensor for the number
    of slots per expert.  ``topk_i``, ``topk_w``: where the results go."""
    if stream is not None:
        return _on(stream, route_logits, logits, k, score=score, bias=bias, n_groups=n_groups, topk_groups=topk_groups,
                   group_top=group_top, renormalize=renormalize, scale=scale, counts=counts, topk_i=topk_i, topk_w=topk_w)
    dev = _device(logits)
    _need(logits.dim() == 2, "logits: needs two dimensions")
    shape = logits.shape
    T, E = shape
    lp, lt, ls = _rows(logits, "logits", shape, _FLOATS, dev)
    _need(1 <= k <= E, "k: needs 1 to the number of experts")
    _need(score in _SCORES, f"score: one of {list(_SCORES)}")
    bp = 0 if bias is None else _dense(bias, "bias", (E,), _F32, dev)
    if topk_i is None:
        topk_i = torch.empty(T, k, dtype=torch.int32, device=logits.device)
    if topk_w is None:
        topk_w = torch.empty(T, k, dtype=torch.float32, device=logits.device)
    ip = _dense(topk_i, "topk_i", (T, k), _I32, dev)
    wp = _dense(topk_w, "topk_w", (T, k), _F32, dev)
    cp = 0
    if counts is True:
        counts = torch.empty(E, dtype=torch.int32, device=logits.device)
    elif counts is False:
        counts = None
    if counts is not None:
        cp = _dense(counts, "counts", (E,), _I32, dev)
    _call("moe_b200_route_logits", dev, _PACK_ROUTE(
        T, E, k, lp, lt, ls, _SCORES[score], bp, n_groups, topk_groups, group_top, bool(renormalize), scale, ip, wp, cp))
    return Routing(topk_i, topk_w, counts)


def w4_matvec(x, codes, scales, bias=None, *, x_scales=None, ids=None, rows_per_x=1, swiglu=None, out=None,
              dtype=torch.bfloat16, stream=None):
    """``out[m] = W[ids[m]] @ x[m // rows_per_x] (+ bias[ids[m]])`` for few rows and 4-bit matrices.

    ``codes``: uint8 [N, K / 2], or a stack [n, N, K / 2] with ``ids``; the checkpoint's blocks [..., K / 32,
    16] are taken as they are.  ``scales`` uint8 or float8_e8m0fnu [..., N, K / 32]: MXFP4; bfloat16
    [..., N, K / group] with groups of 32, 64 or 128: INT4 (value code - 8).  ``bias`` float32 [..., N].
    ``x`` bfloat16, float16, or float8_e4m3fn with ``x_scales`` as ``add_rmsnorm`` returns them.  ``ids``:
    int32 [M], one matrix per row of the result, an index outside the stack gives zeros; without
    it M = x rows * rows_per_x.  ``swiglu``: (alpha, limit) for the framework's clamped SwiGLU over
    interleaved gate and up rows.  At most 256 rows."""
    if stream is not None:
        return _on(stream, w4_matvec, x, codes, scales, bias, x_scales=x_scales, ids=ids, rows_per_x=rows_per_x, swiglu=swiglu,
                   out=out, dtype=dtype)
    dev = _device(x)
    _need(x.dim() == 2, "x: needs two dimensions")
    rows, K = x.shape
    xp, xt, xs = _rows(x, "x", x.shape, _X4, dev)
    shape = scales.shape
    stack = len(shape) == 3
    _need(stack or len(shape) == 2, "scales: needs [N, groups] or [n, N, groups]")
    N, G = shape[-2], shape[-1]
    lead = shape[:-1]
    _need(G > 0 and K % G == 0, "scales: their number must divide the columns of x")
    cp = _dense(codes, "codes", (*lead, G, 16) if codes.dim() == len(shape) + 1 else (*lead, K // 2), _U8, dev)
    sp = _dense(scales, "scales", shape, _W4_SCALES, dev)
    bp = 0 if bias is None else _dense(bias, "bias", lead, _F32, dev)
    _need(rows_per_x >= 1, "rows_per_x: at least 1")
    M = rows * rows_per_x
    ip = 0
    if ids is not None:
        n = ids.numel()
        _need(M - rows_per_x < n <= M, "ids: one per row, rows_per_x for each row of x")
        M = n
        ip = _dense(ids, "ids", (M,), _I32, dev)
    else:
        _need(not stack, "a stack of matrices needs ids")
    kind, xsp = capi.SCALE_NONE, 0
    if x_scales is not None:
        _need(x_scales.dim() == 2, "x_scales: needs two dimensions")
        m = x_scales.shape[1]
        if x_scales.dtype in _MX_TYPES:
            kind, want = capi.SCALE_MX, -(-K // 32)
        elif m == 1:
            kind, want = capi.SCALE_ROW, 1
        else:
            fits = [s for s in (32, 64, 128) if -(-K // s) == m]
            _need(len(fits) == 1, "x_scales: one per row or per 32, 64 or 128 columns")
            kind, want = _QUANT[fits[0]], m
        xsp = _dense(x_scales, "x_scales", (rows, want), _X_SCALES, dev)
    _need(M <= capi.W4_MATVEC_MAX_ROWS, "w4_matvec: at most 256 rows (larger batches are matrix products)")
    alpha, limit = swiglu if swiglu is not None else (0.0, 0.0)
    n_out = N if swiglu is None else N // 2
    if out is None:
        out = torch.empty(M, n_out, dtype=dtype, device=x.device)
    op, ot, os_ = _rows(out, "out", (M, n_out), _FLOATS, dev)
    _call("moe_b200_w4_matvec", dev, _PACK_MATVEC(
        capi.W4_INT4 if scales.dtype == torch.bfloat16 else capi.W4_MXFP4, K // G, shape[0] if stack else 1, N, K, cp, sp, bp,
        xp, xt, xs, xsp, kind, M, rows_per_x, ip, swiglu is not None, alpha, limit, op, ot, os_))
    return out
