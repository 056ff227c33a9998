"""What the performance of the stand-alone operators is measured on: the three steps around
and beside the MoE block that an engine calls with tensors of its own.

A case is a dict of plain values; "op" names the operator:

  norm    add_rmsnorm: r = x + residual, y = rmsnorm(r) * w, y once more as e4m3 with scales
          T H        rows and columns        x, res   types of x and of the residual
          y          type of y, "" for none  quant    "", "row", "g32", "g64", "g128" or "mx"
          pad        columns between two rows of x that belong to something else
  route   route_logits: expert indices and weights from router logits
          T E K      tokens, experts, experts per token      dtype    type of the logits
          score      "softmax" or "sigmoid"                  bias     selection bias for balance
          groups keep top    groups, groups kept, best experts a group is scored by
          renorm scale counts                                masked   some experts are switched off, some rows wholly
  matvec  w4_matvec: products of few rows with 4-bit matrices in groups
          N K R      outputs, inputs, rows   fmt      "mxfp4" or "int4" (with "group")
          mats top   matrices; rows of x take `top` different ones each (0: one matrix for all)
          x          "bf16", "f16", or e4m3 with scales: "row", "g32", "g64", "g128", "mx"
          bias swiglu out

Values are those of the benchmark's synthetic checkpoint: N(0, 1) activations, uniform codes,
scale exponents -8..-4, small biases; everything follows from the seed.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS, _ALPHA, _LIMIT = 1e-5, 1.702, 7.0


def _norm(**kw):
    return {"op": "norm", "T": 1, "H": 2880, "x": "bf16", "res": "f32", "y": "bf16", "quant": "", "pad": 0, **kw}


def _route(**kw):
    return {"op": "route", "T": 1, "E": 128, "K": 4, "dtype": "f32", "score": "softmax", "bias": False, "groups": 1,
            "keep": 1, "top": 1, "renorm": True, "scale": 1.0, "counts": False, "masked": False, **kw}


def _matvec(**kw):
    return {"op": "matvec", "N": 2880, "K": 2880, "R": 1, "fmt": "mxfp4", "group": 32, "mats": 1, "top": 0, "x": "bf16",
            "bias": True, "swiglu": False, "out": "bf16", **kw}


def listed():
    return [
        # one user's token between two layers
        _norm(name="norm_1x2880"),
        # the serving batch, the block's fp32 output added, input for the router (bf16) and for 4-bit products (MX)
        _norm(name="norm_256x2880_mx", T=256, x="f32", quant="mx"),
        # odd rows inside a wider buffer, half-precision stream
        _norm(name="norm_777x2047_g128", T=777, H=2047, x="f16", res="f16", y="", quant="g128", pad=5),
        # a full prefill batch
        _norm(name="norm_16384x2880_row", T=16384, x="bf16", quant="row"),
        # one token, the benchmark's larger router
        _route(name="route_1x128"),
        # the serving batch of a model with many narrow experts, groups and a bias for balance
        _route(name="route_256x256_groups", T=256, E=256, K=8, score="sigmoid", bias=True, groups=8, keep=4, top=2,
               scale=2.5, counts=True),
        # an odd batch, bf16 logits, experts switched off and padded rows
        _route(name="route_3001x60_masked", T=3001, E=60, K=6, dtype="bf16", renorm=False, masked=True),
        # prefill, every expert a candidate, the bias alone moves the choice
        _route(name="route_16384x256_bias", T=16384, E=256, K=8, score="sigmoid", bias=True, counts=True),
        # one token through a dense projection (queries, keys and values)
        _matvec(name="matvec_qkv_1", N=5120),
        # one token through the gate/up matrices of its four experts
        _matvec(name="matvec_gate_up_1", N=5760, R=4, mats=32, top=4, swiglu=True, x="mx"),
        # eight tokens through the down matrices of theirs, every slot with a row of its own
        _matvec(name="matvec_down_8", R=32, mats=32, top=1),
        # the vocabulary for three streams, another 4-bit format, fp32 logits
        _matvec(name="matvec_vocab_3", N=201088, R=3, fmt="int4", group=64, bias=False, out="f32"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "route", "matvec"])
    most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        if op == "norm":
            c = _norm(T=log_int(1, 16384), H=log_int(64, 8192), x=rng.choice(["bf16", "f16", "f32"]),
                      res=rng.choice(["", "bf16", "f16", "f32", "f32"]), y=rng.choice(["bf16", "bf16", "f16", "f32"]),
                      quant=rng.choice(["", "row", "g32", "g64", "g128", "mx"]), pad=rng.choice([0, 0, 0, 3, 16]))
            if rng.random() < 0.6:
                c["H"] = 64 * max(1, round(c["H"] / 64))
            if c["quant"] and rng.random() < 0.4:
                c["y"] = ""
        elif op == "route":
            c = _route(T=log_int(1, 16384), dtype=rng.choice(["f32", "bf16", "f16"]), score=rng.choice(["softmax", "sigmoid"]),
                       bias=rng.random() < 0.5, groups=rng.choice([1, 1, 2, 4, 8]), renorm=rng.random() < 0.7,
                       scale=rng.choice([1.0, 2.5]), counts=rng.random() < 0.5, masked=rng.random() < 0.3)
            c["E"] = c["groups"] * rng.randint(4, 320 // c["groups"])
            c["keep"] = rng.randint(1, c["groups"])
            c["top"] = rng.choice([1, 2])
            c["K"] = rng.randint(1, min(12, c["E"] // c["groups"] * c["keep"]))
        else:
            c = _matvec(N=2 * log_int(32, 32768), K=32 * log_int(2, 256), R=rng.randint(1, 8), bias=rng.random() < 0.5,
                        x=rng.choice(["bf16", "bf16", "f16", "row", "g32", "g64", "g128", "mx"]),
                        out=rng.choice(["bf16", "bf16", "f16", "f32"]), swiglu=rng.random() < 0.3)
            if rng.random() < 0.3:
                c.update(fmt="int4", group=rng.choice([32, 64, 128]))
                c["K"] = c["group"] * max(1, round(c["K"] / c["group"]))
            if rng.random() < 0.4:
                c.update(mats=rng.randint(8, 32), top=rng.choice([1, 2, 4]), N=2 * log_int(32, 2880))
                c["R"] *= c["top"]
        if work(c)["bytes"] <= most and _slowest(c) <= 32 * 5760 * 2880:
            return c


def _slowest(case):
    """Weights that the plain form lays out in 32 bits, one matrix for each row with ids."""
    return case["N"] * case["K"] * (case["R"] if case["top"] else 1) if case["op"] == "matvec" else 0


# -- inputs -------------------------------------------------------------------


def _bytes(shape, gen):
    n = math.prod(shape)
    words = torch.randint(-2**63, 2**63 - 1, ((n + 7) // 8,), generator=gen, device="cuda", dtype=torch.int64)
    return words.view(torch.uint8)[:n].view(shape)


def _q_groups(quant, n):
    return {"row": 1, "mx": -(-n // 32)}.get(quant) or -(-n // int(quant[1:]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7000 + seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] == "norm":
        T, H = case["T"], case["H"]
        s["x"] = randn(T, H + case["pad"]).to(_TYPES[case["x"]])[:, :H]
        s["w"] = (1.0 + 0.1 * randn(H)).to(torch.bfloat16)
        s["res"] = (4.0 * randn(T, H)).to(_TYPES[case["res"]]) if case["res"] else None
        # where the engine wants the results
        s["res_out"] = torch.empty_like(s["res"]) if case["res"] else None
        s["y"] = torch.empty(T, H, dtype=_TYPES[case["y"]], device="cuda") if case["y"] else None
        s["q"] = s["q_scales"] = None
        if case["quant"]:
            s["q"] = torch.empty(T, H, dtype=torch.float8_e4m3fn, device="cuda")
            s["q_scales"] = torch.empty(T, _q_groups(case["quant"], H), device="cuda",
                                        dtype=torch.float8_e8m0fnu if case["quant"] == "mx" else torch.float32)
    elif case["op"] == "route":
        T, E, K = case["T"], case["E"], case["K"]
        logits = 1.1 * randn(T, E) + 0.1 * randn(E)
        if case["masked"]:  # one expert in sixteen is off, and the last rows of the batch are padding
            logits[:, torch.rand(E, generator=gen, device="cuda") < 1 / 16] = -math.inf
            logits[T - T // 8:] = -math.inf
        s["logits"] = logits.to(_TYPES[case["dtype"]])
        s["bias"] = 0.05 * randn(E) if case["bias"] else None
        s["out"] = (torch.empty(T, K, dtype=torch.int32, device="cuda"), torch.empty(T, K, device="cuda"),
                    torch.empty(E, dtype=torch.int32, device="cuda") if case["counts"] else None)
    else:
        N, K, R, M, top = (case[k] for k in ("N", "K", "R", "mats", "top"))
        lead = (M,) if top else ()
        s["codes"] = _bytes((*lead, N, K // 2), gen)
        if case["fmt"] == "mxfp4":
            s["scales"] = torch.randint(127 - 8, 127 - 4 + 1, (*lead, N, K // 32), generator=gen, device="cuda",
                                        dtype=torch.uint8)
        else:
            s["scales"] = (0.004 + 0.02 * torch.rand(*lead, N, K // case["group"], generator=gen, device="cuda")).to(torch.bfloat16)
        s["bias"] = 0.01 * randn(*lead, N) if case["bias"] else None
        s["ids"] = None
        if top:  # `top` different matrices for each token; a serving batch meets most of them
            order = torch.rand(R // top, M, generator=gen, device="cuda").argsort(dim=1)
            s["ids"] = order[:, :top].to(torch.int32).reshape(R).contiguous()
        rows = R // top if top else R
        x = randn(rows, K)
        s["x_scales"] = None
        if case["x"] in _TYPES:
            s["x"] = x.to(_TYPES[case["x"]])
        else:
            g = -(-K // _q_groups(case["x"], K)) if case["x"] in ("row", "mx") else int(case["x"][1:])
            amax = torch.nn.functional.pad(x, (0, -K % g)).view(rows, -1, g).abs().amax(-1)
            sc = torch.exp2(torch.ceil(torch.log2(amax / 448))) if case["x"] == "mx" else amax / 448
            wide = sc.repeat_interleave(g, 1)[:, :K]
            s["x"] = (x / wide).to(torch.float8_e4m3fn)
            s["x_scales"] = sc.to(torch.float8_e8m0fnu) if case["x"] == "mx" else sc
        s["out"] = torch.empty(R, N // 2 if case["swiglu"] else N, dtype=_TYPES[case["out"]], device="cuda")
    return s


# -- one pass -----------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import gpt_oss_amd_b200 as pkg

    c = s["case"]
    if c["op"] == "norm":
        quant = c["quant"] and (int(c["quant"][1:]) if c["quant"][0] == "g" else c["quant"])
        r = pkg.add_rmsnorm(s["x"], s["w"], s["res"], eps=_EPS, dtype=_TYPES[c["y"]] if c["y"] else None,
                            quant=quant or None, residual_out=s["res_out"], out=s["y"], q=s["q"], q_scales=s["q_scales"])
        return [v for v in (r.residual, r.y, r.q, r.q_scales) if v is not None]
    if c["op"] == "route":
        r = pkg.route_logits(s["logits"], c["K"], score=c["score"], bias=s["bias"], n_groups=c["groups"],
                             topk_groups=c["keep"], group_top=c["top"], renormalize=c["renorm"], scale=c["scale"],
                             topk_i=s["out"][0], topk_w=s["out"][1], counts=s["out"][2])
        return [v for v in r if v is not None]
    return pkg.w4_matvec(s["x"], s["codes"], s["scales"], s["bias"], x_scales=s["x_scales"], ids=s["ids"],
                         rows_per_x=c["top"] or 1, swiglu=(_ALPHA, _LIMIT) if c["swiglu"] else None, out=s["out"])


def _run_plain(s):
    return {"norm": _plain_norm, "route": _plain_route, "matvec": _plain_matvec}[s["case"]["op"]](s)


def _plain_norm(s):
    c, out = s["case"], []
    r = s["x"].float()
    if c["res"]:
        r = r + s["res"].float()
        out.append(r.to(_TYPES[c["res"]]))
    y = r * torch.rsqrt((r * r).mean(dim=1, keepdim=True) + _EPS) * s["w"].float()
    if c["y"]:
        out.append(y.to(_TYPES[c["y"]]))
    if c["quant"]:
        T, H = y.shape
        n = _q_groups(c["quant"], H)
        g = H if c["quant"] == "row" else 32 if c["quant"] == "mx" else int(c["quant"][1:])
        if H % g:
            y = torch.cat((y, y.new_zeros(T, n * g - H)), dim=1)
        y = y.view(T, n, g)
        amax = y.abs().amax(dim=2)
        if c["quant"] == "mx":
            m, e = torch.frexp(amax)  # amax = m 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9
            scale = torch.where(amax > 0, torch.exp2((e - 9 + (m > 0.875).int()).clamp(-127, 127).float()), 1.0)
        else:
            scale = torch.where(amax > 0, amax / 448, 1.0)
        q = (y / scale.unsqueeze(2)).clamp(-448, 448).view(T, n * g)[:, :H].to(torch.float8_e4m3fn)
        out += [q, scale.to(torch.float8_e8m0fnu) if c["quant"] == "mx" else scale]
    return out


def _plain_route(s):
    c = s["case"]
    T, E, K, G = c["T"], c["E"], c["K"], c["groups"]
    l = s["logits"].double()  # 64 bits: neighbouring scores decide whole numbers
    off = torch.isneginf(l) | torch.isnan(l)
    l = l.masked_fill(off, -math.inf)
    if c["score"] == "softmax":
        p = torch.exp(l - l.amax(dim=1, keepdim=True).clamp(min=-1e300))
        p = p / p.sum(dim=1, keepdim=True).clamp(min=1e-300)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    key = l if s["bias"] is None else (p + s["bias"].double()).masked_fill(off, -math.inf)
    if G > 1:
        by = (l if s["bias"] is None and c["top"] == 1 else p if s["bias"] is None else key).masked_fill(off, -math.inf)
        best = by.view(T, G, -1).sort(dim=2, descending=True).values[:, :, :c["top"]]
        score = best.masked_fill(torch.isneginf(best), 0.0).sum(dim=2).masked_fill(torch.isneginf(best[:, :, 0]), -math.inf)
        kept = score.sort(dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        mask = torch.zeros(T, G, dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        key = key.view(T, G, -1).masked_fill(~mask.unsqueeze(2), -math.inf).view(T, E)
    key, index = key.sort(dim=1, descending=True, stable=True)
    empty = torch.isneginf(key[:, :K])
    index = index[:, :K]
    w = p.gather(1, index).masked_fill(empty, 0.0)
    if c["renorm"]:
        w = w / w.sum(dim=1, keepdim=True).clamp(min=1e-300)
    index = index.masked_fill(empty, -1)
    out = [index.int(), (w * c["scale"]).float()]
    if c["counts"]:
        out.append((torch.bincount(index.reshape(-1) + 1, minlength=E + 1)[1:]).int())
    return out


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _plain_matvec(s):
    c = s["case"]
    K = c["K"]
    codes, scales, bias, ids = s["codes"], s["scales"], s["bias"], s["ids"]
    if ids is not None:
        pick = ids.long()
        codes, scales = codes[pick], scales[pick]
        bias = bias[pick] if bias is not None else None
    v = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    if c["fmt"] == "mxfp4":
        v = torch.tensor(_E2M1, device=v.device)[v.int()]
        scale = torch.exp2(scales.float() - 127.0)
    else:
        v = v.float() - 8.0
        scale = scales.float()
    w = (v.view(*scale.shape, -1) * scale.unsqueeze(-1)).flatten(-2)
    x = s["x"].float()
    if s["x_scales"] is not None:
        n = s["x_scales"].shape[1]
        x = x * s["x_scales"].float().repeat_interleave(K if n == 1 else 32 if c["x"] == "mx" else int(c["x"][1:]), 1)[:, :K]
    if ids is None:
        y = x @ w.T
    else:
        x = x.repeat_interleave(c["top"], 0)
        y = (w @ x.unsqueeze(2)).squeeze(2)
    if bias is not None:
        y = y + bias
    if c["swiglu"]:
        gate, up = y[:, 0::2].clamp(max=_LIMIT), y[:, 1::2].clamp(-_LIMIT, _LIMIT)
        y = gate / (1.0 + torch.exp(-_ALPHA * gate)) * (up + 1.0)
    return y.to(_TYPES[c["out"]])


# -- what a pass cannot do without ---------------------------------------------


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "": 0}
    if case["op"] == "norm":
        T, H = case["T"], case["H"]
        b = T * H * (size[case["x"]] + 2 * size[case["res"]] + size[case["y"]]) + 2 * H
        if case["quant"]:
            b += T * H + T * _q_groups(case["quant"], H) * (1 if case["quant"] == "mx" else 4)
        return {"bytes": b, "flops": 8 * T * H}
    if case["op"] == "route":
        T, E, K = case["T"], case["E"], case["K"]
        return {"bytes": T * E * size[case["dtype"]] + T * K * 8 + E * 4 * (case["bias"] + case["counts"]), "flops": 10 * T * E}
    N, K, R, M, top = (case[k] for k in ("N", "K", "R", "mats", "top"))
    used = M * (1.0 - (1.0 - top / M) ** (R // top)) if top else 1  # expected value
    per = N * K / 2 + (N * K / 32 if case["fmt"] == "mxfp4" else 2 * N * K / case["group"]) + (4 * N if case["bias"] else 0)
    rows = R // top if top else R
    x = rows * K * 2 if case["x"] in _TYPES else rows * (K + _q_groups(case["x"], K) * (1 if case["x"] == "mx" else 4))
    return {"bytes": used * per + x + R * N // (2 if case["swiglu"] else 1) * size[case["out"]] + (4 * R if top else 0),
            "flops": 2 * R * N * K}


# -- the definitions in 64 bits -------------------------------------------------


def exact(case, seed):
    return {"norm": _exact_norm, "route": _exact_route, "matvec": _exact_matvec}[case["op"]](case, prepare(case, seed))


def _exact_norm(case, s):
    """An 8-bit code stands for the quotient that it is the nearest code of; the exponent of an MX
    scale is a whole number and has no other value."""
    H, out = case["H"], []
    r = s["x"].double()
    if case["res"]:
        r = r + s["res"].double()
        out.append(r)
    y = s["w"].double() * (r / torch.sqrt((r * r).sum(dim=1, keepdim=True) / H + _EPS))
    if case["y"]:
        out.append(y)
    if case["quant"]:
        g = {"row": H, "mx": 32}.get(case["quant"]) or int(case["quant"][1:])
        q, scales = torch.empty_like(y), []
        for at in range(0, H, g):
            part = y[:, at:at + g]
            top = part.abs().amax(dim=1, keepdim=True)
            sc = torch.exp2(torch.ceil(torch.log2(top / 448.0))) if case["quant"] == "mx" else top / 448.0
            sc = torch.where(top > 0, sc, torch.ones_like(sc))
            q[:, at:at + g] = part / sc
            scales.append(sc)
        out += [q, None if case["quant"] == "mx" else torch.cat(scales, dim=1)]
    return out


def _exact_route(case, s):
    """By ranks: an expert's place is the number of experts in front of it."""
    E, K, G = case["E"], case["K"], case["groups"]
    weights = []
    lower = torch.arange(E, device="cuda").unsqueeze(1) > torch.arange(E, device="cuda")  # [i, j]: j in front at a tie
    glower = torch.arange(G, device="cuda").unsqueeze(1) > torch.arange(G, device="cuda")

    def rank(v, lower):
        a, b = v.unsqueeze(2), v.unsqueeze(1)
        return ((b > a) | ((b == a) & lower)).sum(dim=2)

    for l in s["logits"].double().split(256):
        live = l > -math.inf
        p = torch.softmax(torch.where(live.any(1, keepdim=True), l, 0.0), dim=1) if case["score"] == "softmax" else torch.sigmoid(l)
        p = torch.where(live, p, 0.0)
        key = l if s["bias"] is None else p + s["bias"].double()
        if G > 1:
            by = key if s["bias"] is not None else l if case["top"] == 1 else p
            by = torch.where(live, by, -math.inf).view(-1, G, E // G)
            some = live.view(by.shape)
            inside = rank(by.reshape(-1, E // G), lower[:E // G, :E // G]).view(by.shape)
            score = torch.where(some & (inside < case["top"]), by, 0.0).sum(dim=2)
            score = torch.where(some.any(2), score, -math.inf)
            live = live & (rank(score, glower) < case["keep"]).repeat_interleave(E // G, 1)
        place = rank(torch.where(live, key, -math.inf), lower)
        w = torch.zeros(l.shape[0], K, dtype=torch.float64, device="cuda")
        row, e = (live & (place < K)).nonzero(as_tuple=True)
        w[row, place[row, e]] = p[row, e]
        if case["renorm"]:
            total = w.sum(dim=1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
        weights.append(w * case["scale"])
    return [None, torch.cat(weights)] + ([None] if case["counts"] else [])


def _exact_matvec(case, s):
    def matrix(codes, scales):
        n = torch.stack((codes % 16, codes // 16), dim=2).view(codes.shape[0], -1).short()
        if case["fmt"] == "mxfp4":  # sign, two bits of exponent, one of mantissa
            e, m = n // 2 % 4, (n % 2).double()
            v = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * 2.0 ** (e.double() - 1.0))
            v = torch.where(n >= 8, -v, v)
            sc = 2.0 ** (scales.double() - 127.0)
        else:
            v, sc = n.double() - 8.0, scales.double()
        return v * sc.repeat_interleave(v.shape[1] // sc.shape[1], 1)

    x = s["x"].double()
    if s["x_scales"] is not None:
        sc = s["x_scales"].double()
        g = {"row": x.shape[1], "mx": 32}.get(case["x"]) or int(case["x"][1:])
        x = x * sc.repeat_interleave(g, 1)[:, :x.shape[1]]
    y = torch.empty(case["R"], case["N"], dtype=torch.float64, device="cuda")
    if s["ids"] is None:
        for at in range(0, case["N"], 16384):
            y[:, at:at + 16384] = x @ matrix(s["codes"][at:at + 16384], s["scales"][at:at + 16384]).T
        y = y if s["bias"] is None else y + s["bias"].double()
    else:
        for row, e in enumerate(s["ids"].tolist()):
            y[row] = matrix(s["codes"][e], s["scales"][e]) @ x[row // case["top"]]
            if s["bias"] is not None:
                y[row] += s["bias"][e].double()
    if case["swiglu"]:
        gate, up = y[:, 0::2].clamp(max=_LIMIT), y[:, 1::2].clamp(-_LIMIT, _LIMIT)
        y = gate * torch.sigmoid(_ALPHA * gate) * (up + 1.0)
    return y
