"""The stand-alone operators from their definitions in 64 bits, for the tests, with the error that a correct
fp32 evaluation may have (half a step of the result's type for each rounding to fewer bits)."""
import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rmsnorm(x, w, res, eps):
    r = x.double() + (0 if res is None else res.double())
    return r, r / torch.sqrt((r * r).mean(1, keepdim=True) + eps) * w.double()


def norm_error(H):
    """Relative error of y before its rounding: the sum x + residual (one step), the sum of squares (at most 32
    additions in a thread, 10 levels between threads, halved by the root), division, root, reciprocal, two products."""
    return (1 + 42 / 2 + 1 + 5) * 2.0**-24 + 2.0**-40


def route(logits, k, score, bias, n_groups, topk_groups, group_top, renorm, scale):
    """Plain loops over tokens and experts: small cases only."""
    T, E = logits.shape
    idx = torch.full((T, k), -1, dtype=torch.int32)
    w = torch.zeros(T, k, dtype=torch.float64)
    L = logits.detach().cpu().double()
    B = None if bias is None else bias.detach().cpu().double()
    fmax = torch.finfo(torch.float32).max
    for t in range(T):
        live = [e for e in range(E) if L[t, e] > -math.inf and (B is None or B[e] > -math.inf)]
        l = {e: min(float(L[t, e]), fmax) for e in range(E) if L[t, e] > -math.inf}
        if not l:
            continue
        m = max(l.values())
        if score == "softmax":
            z = sum(math.exp(v - m) for v in l.values())
            p = {e: math.exp(v - m) / z for e, v in l.items()}
            logp = {e: v - m - math.log(z) for e, v in l.items()}
        else:
            p = {e: 1 / (1 + math.exp(-v)) if v > -700 else 0.0 for e, v in l.items()}
            logp = {e: -math.log1p(math.exp(-v)) if v > -700 else v for e, v in l.items()}
        key = {e: l[e] if B is None else p[e] + min(float(B[e]), fmax) for e in live}
        if n_groups > 1:
            size = E // n_groups
            by = key if B is not None or group_top == 1 else p
            scores = []
            for g in range(n_groups):
                inside = sorted((by[e] for e in live if e // size == g), reverse=True)
                if inside:
                    scores.append((-sum(inside[:group_top]), g))
            kept = {g for _, g in sorted(scores)[:topk_groups]}
            key = {e: v for e, v in key.items() if e // size in kept}
        chosen = sorted(key, key=lambda e: (-key[e], e))[:k]
        # p / sum of the selected p; relative to the largest of them, which 64 bits hold whatever the logits
        big = max((logp[e] for e in chosen), default=0.0)
        total = sum(math.exp(logp[e] - big) for e in chosen)
        for j, e in enumerate(chosen):
            idx[t, j] = e
            w[t, j] = (math.exp(logp[e] - big) / total if renorm else p[e]) * scale
    return idx, w


def dequant(codes, scales, group):
    """codes u8 [..., K / 2], scales u8 (e8m0) or bf16 [..., K / group] -> fp64 [..., K]."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    if scales.dtype == torch.bfloat16:
        v, s = n.double() - 8, scales.double()
    else:
        table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
        v, s = table[n], torch.exp2(scales.view(torch.uint8).double() - 127)
    return v * s.repeat_interleave(group, -1)


def matvec(x, codes, scales, bias, group, ids, rows_per_x):
    """-> (y, sum |w x| + |bias|), fp64 [M, N]; x in fp64."""
    W = dequant(codes, scales, group)
    if W.dim() == 2:
        W = W.unsqueeze(0)
    M = len(ids) if ids is not None else x.shape[0] * rows_per_x
    y = torch.zeros(M, W.shape[1], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    ids = [0] * M if ids is None else ids.tolist()
    for m, e in enumerate(ids):
        if 0 <= e < W.shape[0]:
            v = x[m // rows_per_x]
            y[m] = W[e] @ v
            size[m] = W[e].abs() @ v.abs()
            if bias is not None:
                b = bias.view(-1, W.shape[1])[e].double()
                y[m] += b
                size[m] += b.abs()
    return y, size


def matvec_error(K):
    """Error of y over sum |w x|: products are exact; a tensor-core step adds 16 of them to its accumulator with
    an error of at most two bits below fp32's last for each of its 8 instructions, a warp adds up to
    ceil(K / 1024) steps, then 8 warps, four columns, the bias; each scale product is one rounding."""
    return (8 * 4 + math.ceil(K / 1024) + 8 + 4 + 4) * 2.0**-23


def swiglu(y, size, alpha, limit):
    """-> (value, its change for an error of one in y scaled by `size`)."""
    g, u = y[:, 0::2].clamp(max=limit), y[:, 1::2].clamp(-limit, limit)
    a = g * torch.sigmoid(alpha * g)
    return a * (u + 1), 1.1 * (u + 1).abs() * size[:, 0::2] + a.abs() * size[:, 1::2]
