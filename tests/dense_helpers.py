"""Plain 64-bit forms of the 16-bit layers' operators, and how far results of their types may be off.

Every form returns (value, bound).  A stored value of type t is rounded once, by at most half a step:
eps(t) / 2 of its size, or half of the smallest subnormal.  Sums are f32: a sum of k terms that is formed
in any order loses at most k roundings of eps32 / 2 of the sum of sizes; the tensor cores, which drop
low bits of a running sum, at most 8 eps32 per term (the bound the MX GEMMs are held to)."""
import math

import torch

EPS32 = float(torch.finfo(torch.float32).eps)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GELU_C, GELU_A = math.sqrt(2 / math.pi), 0.044715


def rounding(value, kind):
    """What storing `value` in the type may lose."""
    info = torch.finfo(TYPES[kind])
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def logistic(z):
    small = torch.exp(-z.abs())
    return torch.where(z >= 0, 1 / (1 + small), small / (1 + small))


def act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return z * logistic(2 * GELU_C * z * (1 + GELU_A * z * z))
    if name == "silu":
        return z * logistic(z)
    return z


def slope(z, name):
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), torch.ones_like(z))
    if name in ("gelu", "silu"):
        v = 2 * GELU_C * z * (1 + GELU_A * z * z) if name == "gelu" else z
        dv = 2 * GELU_C * (1 + 3 * GELU_A * z * z) if name == "gelu" else torch.ones_like(z)
        s = logistic(v)
        return s + z * s * (1 - s) * dv
    return torch.ones_like(z)


def product(a, b, bias, name, C, alpha, beta, d_type):
    """a (m x k), b (k x n) in 64 bits; -> (D, its bound), (z, its bound)."""
    k = a.shape[1]
    z = alpha * (a @ b)
    err = abs(alpha) * 8 * EPS32 * k * (a.abs() @ b.abs()) + EPS32 * z.abs()
    if bias is not None:
        z = z + bias
        err = err + EPS32 * z.abs()
    # |act'| is below 1.13; expf, a cubic argument and a quotient: its argument's error acts like one of z
    d = act(z, name)
    derr = 1.13 * err + (16 * EPS32 * d.abs() + 8 * EPS32 * z.abs() * (z.abs() < 20) if name in ("gelu", "silu") else 0)
    if C is not None:
        d = d + beta * C
        derr = derr + EPS32 * (d.abs() + (beta * C).abs())
    return (d, derr + rounding(d.abs() + derr, d_type)), (z, err + rounding(z.abs() + err, d_type))


def epilogue_grad(dy, z, name, kind):
    """-> (dZ, its bound), (dbias, its bound)."""
    s = slope(z, name) if name != "none" else torch.ones_like(dy)
    dz = dy * s
    # a slope of at most 1.13 from expf of an argument that is off by a few roundings of its own size (at most
    # 90, where exp still counts; what it then loses is below t |v| of the result), a quotient, products
    err = dy.abs() * (64 * EPS32 if name in ("gelu", "silu") else 0) + EPS32 * dz.abs()
    m = dy.shape[0]
    total = err.sum(0) + m * EPS32 * dz.abs().sum(0)
    return (dz, err + rounding(dz.abs() + err, kind)), (dz.sum(0), total + 1e-30)


def layer_norm(x, gamma, beta, eps, y_type):
    """-> (y, bound), (mean, bound), (rstd, bound)."""
    n = x.shape[1]
    mean = x.mean(1, keepdim=True)
    # f32 sums over a tree of threads: at most 16 elements in a row, then 10 levels; 32 roundings cover both
    # (long rows: n / 1024 elements in a row)
    steps = (32 + n / 1024) * EPS32
    mean_err = steps * x.abs().mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    var_err = 2 * (mean_err + EPS32 * x.abs().amax(1, keepdim=True)) * d.abs().mean(1, keepdim=True) + mean_err ** 2 + (steps + 2 * EPS32) * var
    rstd = 1 / torch.sqrt(var + eps)
    rstd_err = rstd * (0.5 * var_err / (var + eps) + 4 * EPS32)
    g = torch.ones_like(mean) if gamma is None else gamma
    xhat = d * rstd
    y = xhat * g + (0 if beta is None else beta)
    err = ((mean_err + EPS32 * d.abs()) * rstd + d.abs() * rstd_err + 2 * EPS32 * xhat.abs()) * g.abs() + EPS32 * y.abs()
    return (y, err + rounding(y.abs() + err, y_type)), (mean[:, 0], mean_err[:, 0] + EPS32 * mean[:, 0].abs()), (rstd[:, 0], rstd_err[:, 0])


def layer_norm_grad(dy, x, gamma, mean, rstd, dr, x_type):
    """mean and rstd as given (exact); -> (dx, bound), (dgamma, bound), (dbeta, bound)."""
    m, n = x.shape
    steps = (32 + n / 1024) * EPS32
    xhat = (x - mean[:, None]) * rstd[:, None]
    xhat_err = 2 * EPS32 * xhat.abs()
    g = dy if gamma is None else dy * gamma
    s1, s2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    e1 = steps * g.abs().mean(1, keepdim=True)
    e2 = (steps + 4 * EPS32) * (g * xhat).abs().mean(1, keepdim=True)
    core = g - s1 - xhat * s2
    err = rstd[:, None] * (3 * EPS32 * (g.abs() + s1.abs() + (xhat * s2).abs()) + e1 + xhat.abs() * e2 + xhat_err * s2.abs())
    dx = rstd[:, None] * core
    if dr is not None:
        dx = dx + dr
        err = err + EPS32 * (dx.abs() + dr.abs())
    rows = (m + 8) * EPS32
    return ((dx, err + rounding(dx.abs() + err, x_type)), ((dy * xhat).sum(0), rows * (dy * xhat).abs().sum(0) + 1e-30),
            (dy.sum(0), rows * dy.abs().sum(0) + 1e-30))


def balance(logits, ids, sigmoid, coefficient, upstream, kind):
    """-> counts, (loss, bound), (dlogits, bound); logits in 64 bits, ids tokens x top_k."""
    x = torch.where(torch.isposinf(logits), torch.full_like(logits, torch.finfo(torch.float32).max), logits)
    out = ~(x > -math.inf)
    tokens, experts = x.shape
    valid = (ids >= 0) & (ids < experts)
    counts = torch.bincount(ids[valid].long(), minlength=experts)
    live = valid.any(1) if tokens else valid.new_zeros((0,))
    T, pairs = int(live.sum()), int(valid.sum())
    p = torch.zeros_like(x)
    rest = torch.ones_like(x)
    for t in range(tokens):
        e = (~out[t]).nonzero().flatten()
        if e.numel() == 0:
            continue
        v = x[t, e]
        if sigmoid:
            # logistics over a common factor exp(min(max, 0))
            top = min(float(v.max()), 0.0)
            s = torch.exp(v.clamp_max(0) - top) / (1 + torch.exp(-v.abs()))
            rest[t, e] = logistic(-v)
        else:
            s = torch.exp(v - v.max())
        p[t, e] = s / s.sum()
    if T == 0:
        zero = torch.zeros((), dtype=torch.float64)
        return counts, (zero, zero + 1e-30), (torch.zeros_like(x), torch.zeros_like(x))
    f = counts.double() / pairs
    P = p[live].sum(0) / T
    loss = coefficient * experts * (f * P).sum()
    size = upstream * coefficient * experts / T
    along = (p * (f - 1 / experts)).sum(1, keepdim=True)
    w = p * rest if sigmoid else p
    grad = size * w * ((f - 1 / experts) - along)
    grad[~live] = 0
    # p: expf of an argument off by a rounding of its size, a sum, a quotient; then sums of at most 10 + experts / 32 steps
    off = (x.masked_fill(out, 0.0).abs().clamp_max(104) + 24 + experts / 32) * EPS32
    spread = (f - 1 / experts).abs()
    err = abs(size) * w * (2 * off * ((p * spread).sum(1, keepdim=True) + spread) + 8 * EPS32 * (spread + along.abs()))
    off_loss = float(off.max()) + (T + 64) * EPS32
    return counts, (loss, abs(loss) * off_loss), (grad, torch.where(live[:, None], err + rounding(grad.abs() + err, kind), 0.0))


def worst(got, want):
    """How much of its bound the worst element takes (infinite where only one of both is finite)."""
    value, bound = want
    got = got.detach().double().cpu()
    value, bound = value.cpu(), bound.cpu()
    fine = torch.isfinite(value)
    if not torch.equal(fine, torch.isfinite(got)) or not torch.equal(torch.isnan(value), torch.isnan(got)):
        return math.inf
    if not fine.any():
        return 0.0
    return float(((got - value).abs()[fine] / bound[fine].clamp_min(1e-300)).max())
