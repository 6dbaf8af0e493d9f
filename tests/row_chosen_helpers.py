"""Plain 64-bit forms of the operators whose weights are chosen per row, and operands for them."""
import numpy as np

from cpu_ops_b200 import _capi

FIELDS = {_capi.FMT_E4M3: (3, 4, 7), _capi.FMT_E5M2: (2, 5, 15), _capi.FMT_E2M1: (1, 2, 1)}


def decode_mx(codes, scales, fmt, k):
    """Rows of MX elements as float64 numbers."""
    codes = np.asarray(codes)
    if fmt == _capi.FMT_E2M1:
        codes = np.stack((codes & 15, codes >> 4), axis=-1).reshape(codes.shape[0], -1)
    mantissa, bits, bias = FIELDS[fmt]
    v = codes[:, :k].astype(np.int64)
    exponent = (v >> mantissa) & ((1 << bits) - 1)
    fraction = (v & ((1 << mantissa) - 1)) / (1 << mantissa)
    size = np.ldexp(fraction + (exponent > 0), np.maximum(exponent, 1) - bias)
    sign = 1 - 2 * ((v >> (mantissa + bits)) & 1)
    s = np.asarray(scales).astype(np.int64)[:, np.arange(k) // 32] - 127
    return np.ldexp(sign * size, s)


def plan_of(ids, groups):
    flat = np.asarray(ids).ravel().astype(np.int64)
    valid = (flat >= 0) & (flat < groups)
    members = [np.nonzero(flat == g)[0] for g in range(groups)]
    offsets = np.concatenate(([0], np.cumsum([m.size for m in members]))).astype(np.int32)
    order = np.concatenate(members + [np.full(int((~valid).sum()), -1)]).astype(np.int32)
    return offsets, order


def route(logits, bias, top_k, sigmoid, n_groups, top_groups, group_best, renormalize, scale):
    """ids, weights by the definition, expert by expert, in float64."""
    x = np.asarray(logits, np.float64)
    tokens, experts = x.shape
    x = np.where(np.isposinf(x), float(np.finfo(np.float32).max), x)
    out = ~(x > -np.inf)
    if bias is not None:
        out |= ~(np.asarray(bias, np.float64) > -np.inf)[None, :]
    ids = np.full((tokens, top_k), -1, np.int32)
    weights = np.zeros((tokens, top_k))
    per = experts // n_groups
    for t in range(tokens):
        live = np.nonzero(~out[t])[0]
        score = np.zeros(experts)
        if live.size:
            v = x[t, live]
            with np.errstate(over="ignore", under="ignore"):
                if sigmoid:
                    score[live] = np.where(v >= 0, 1 / (1 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1 + np.exp(-np.abs(v))))
                else:
                    e = np.exp(v - v.max())
                    score[live] = e / e.sum()
        choice = np.full(experts, -np.inf)
        choice[live] = score[live] + (0 if bias is None else np.asarray(bias, np.float64)[live])
        if n_groups > 1:
            best = np.full(n_groups, -np.inf)
            for g in range(n_groups):
                s = np.sort(choice[g * per:(g + 1) * per])[::-1][:group_best]
                if np.isfinite(s[0]) or s[0] == np.inf:
                    best[g] = s[s > -np.inf].sum()
            kept = sorted(range(n_groups), key=lambda g: (-best[g], g))[:top_groups]
            for g in range(n_groups):
                if g not in kept:
                    choice[g * per:(g + 1) * per] = -np.inf
        picked = sorted([e for e in range(experts) if choice[e] > -np.inf], key=lambda e: (-choice[e], e))[:top_k]
        w = score[picked]
        if renormalize:
            w = w / w.sum() if len(picked) and w.sum() > 0 else np.zeros(len(picked))
        ids[t, :len(picked)] = picked
        weights[t, :len(picked)] = w * scale
    return ids, weights


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-v))


def grouped(A, B, ids, n, gated, pairs_per_a_row, row_weights, pairs_per_d_row, before):
    """A (float64 rows), B (groups x n_b x k): the products, and for each how far f32 sums may be
    off: the tensor cores' running sums lose at most 8 eps per element of k (the bound the MX
    GEMMs are held to), what follows them a few roundings."""
    eps = float(np.finfo(np.float32).eps)
    flat = np.asarray(ids).ravel()
    k = A.shape[1]
    y, err = np.zeros((flat.size, n)), np.zeros((flat.size, n))
    live = (flat >= 0) & (flat < B.shape[0])
    for q in np.nonzero(live)[0]:
        row, w = A[q // pairs_per_a_row], B[flat[q]]
        acc, size = w @ row, np.abs(w) @ np.abs(row)
        e = 8 * k * eps * size
        if gated:
            g, u, eg, eu = acc[:n], acc[n:], e[:n], e[n:]
            s = silu(g)
            # |silu'| < 1.1; expf, a sum, a quotient and two products
            v = s * u
            ev = 1.1 * eg * (np.abs(u) + eu) + (np.abs(s)) * eu + 16 * eps * np.abs(v)
        else:
            v, ev = acc[:n], e[:n]
        if row_weights is not None:
            weight = float(np.asarray(row_weights).ravel()[q])
            v, ev = v * weight, ev * abs(weight) + eps * np.abs(v * weight)
        y[q], err[q] = v, ev
    if pairs_per_d_row > 1:
        s = pairs_per_d_row
        total, bound = y.reshape(-1, s, n).sum(1), err.reshape(-1, s, n).sum(1)
        return total, bound + s * eps * np.abs(y).reshape(-1, s, n).sum(1) + 1e-30
    want = np.array(before, np.float64)
    want[live] = y[live]
    return want, np.where(live[:, None], err + 1e-30, 0.0)


def adapters(x, A, B, ids, scales, C):
    """D in float64, and how far f32 sums of the same products may be off: k + 8 roundings of
    a sum of k terms and then rank + 4 of one of rank, relative to the sums of sizes."""
    eps = float(np.finfo(np.float32).eps)
    D = np.asarray(C, np.float64).copy()
    err = np.zeros_like(D)
    rank, k = A.shape[1:]
    for t, g in enumerate(np.asarray(ids)):
        if g < 0 or g >= A.shape[0]:
            continue
        s = 1.0 if scales is None else float(scales[g])
        u, size = A[g] @ x[t], np.abs(A[g]) @ np.abs(x[t])
        y, total = B[g] @ u, np.abs(B[g]) @ size
        D[t] += s * y
        err[t] = eps * ((k + rank + 12) * abs(s) * total + np.abs(D[t]) + np.abs(np.asarray(C, np.float64)[t]))
    return D, err


def quantise_e4m3(x):
    """Rows of f32 torch values as MX e4m3: elements and scales, the largest of 32 in the top binade."""
    import torch
    blocks = x.unflatten(-1, (-1, 32))
    exponent = torch.frexp(blocks.abs().amax(-1).clamp_min(2.0 ** -60))[1] - 9
    y = torch.ldexp(blocks, -exponent.unsqueeze(-1)).flatten(-2)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), (exponent + 127).to(torch.uint8)
