"""The 16-bit layers' operators at particular values: how near f32 results of the activations are, and that infinities and
NaN stay in their rows and columns (of whatever lies in a row's padding nothing is read)."""
import math

import pytest
import torch

import cpu_ops_b200 as c
from tests import dense_helpers as H
from tests.test_dense_gpu import ACT, GUARD, STORAGE, held, matrix, ok, ref, unguarded

pytestmark = pytest.mark.gpu
U = 2.0 ** -24   # what an f32 operation rounds by; exp2 is within 4 U, the reciprocal within 2 U


@pytest.mark.parametrize("m", [1, 200])
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("name", ["gelu", "silu", "relu"])
def test_f32_activations_of_every_f16_value(gpu, name, pad, m):
    """z = 1 * b is exact; act(z) = z s with s = 1 / (1 + t), t = exp(-v).  v is off by 5 roundings (gelu; silu: 1.25, of log2(e) and the
    product), so t by (5 |v| + 4) U and s by s (1 - s) (5 |v| + 4) U + 3 s U; with the last product 3.0e-7 at most.
    Infinities: inf as the limit, -inf is -inf / inf and so NaN (relu: 0)."""
    b = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.float16).cuda()
    n = b.numel()
    a = torch.ones((m, 1), dtype=torch.float16, device="cuda")
    D, Z = held(m, n, pad, "f32"), held(m, n, pad, "f32")
    op = c.GemmF16(c.RowMajor, c.ColumnMajor, storage_d=c.f32_t)
    ok(op(op.Arguments(c.GemmCoord(m, n, 1), c.TensorRef(a, 1), c.TensorRef(b, 1), c.TensorRef(), ref(D),
                       c.BiasActivation(None, ACT[name]), ref(Z))))
    z = b.double()
    want = H.act(z, name)
    if name != "relu":
        want = torch.where(torch.isneginf(z), torch.full_like(z, math.nan), want)
    assert torch.equal(torch.nan_to_num(Z[:m, :n].double(), 0.5), torch.nan_to_num(z, 0.5).expand(m, n))
    got, far = D[:m, :n].double(), (torch.isinf(z) | torch.isnan(z)).expand(m, n)
    assert torch.equal(torch.nan_to_num(got[far], 0.5, 1.0, -1.0), torch.nan_to_num(want.expand(m, n)[far], 0.5, 1.0, -1.0))
    off = (got - want).abs()[~far]
    assert float((off - (0.0 if name == "relu" else 3.0e-7) * z.abs().expand(m, n)[~far]).max()) <= 1e-37
    assert unguarded(D, m, n) and unguarded(Z, m, n)


@pytest.mark.parametrize("name,most", [("gelu", 7.6e-7), ("silu", 5.7e-7)])
def test_f32_slopes(gpu, name, most):
    """s (1 + w (1 - s)) dy with t off by e = (4 |v| + 4) U (silu: 1.25 |v|), s by (1 - s) e + 3 U, t s by s e + 4 U, w by 4 U (silu: 0), and
    three roundings more: the largest of s |1 + w (1 - s)| ((1 - s) e + 6 U) + s |w| (1 - s) (s e + 8 U) over z is 7.54e-7 (silu: 4 U
    for 8 U and 5.65e-7)."""
    z = torch.linspace(-12, 12, 1 << 20, device="cuda").view(1 << 10, 1 << 10)
    dy, dz = matrix(1 << 10, 1 << 10, 0, "f32", 1), torch.zeros_like(z)
    op = c.BiasActivationGrad(c.f32_t, ACT[name])
    ok(op(op.Arguments(c.RowsCoord(1 << 10, 1 << 10), ref(dy), ref(z), ref(dz))))
    off = (dz.double() - dy.double() * H.slope(z.double(), name)).abs() / dy.double().abs().clamp_min(1e-30)
    assert float(off.max()) <= most


def equal_where_not_finite(got, want):
    got, want = got.double().cpu(), want.cpu()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want)) and \
        torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])


def worst_finite(got, want):
    """H.worst of the elements that are finite in 64 bits."""
    value, bound = want
    fine = torch.isfinite(value)
    return H.worst(got.cpu()[fine], (value[fine], bound[fine]))


# few and many rows; a warp's, a CTA's, in the ring, in pairs of elements, too long for registers
NORMS = [(40, 200, 3), (700, 200, 8), (9, 1000, 0), (700, 1000, 8), (700, 2048, 8), (650, 4096, 8), (600, 6000, 8), (20, 6000, 8), (20, 1001, 2),
         (700, 4001, 4), (600, 8001, 3), (12, 9000, 5)]


@pytest.mark.parametrize("x_type,y_type", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("m,n,pad", NORMS)
def test_layer_norm_keeps_infinities_and_nan_in_their_rows(gpu, x_type, y_type, m, n, pad):
    x = matrix(m, n, pad, x_type, 1, 2.0)
    x[:, n:] = math.nan
    x[1, n - 1], x[3, 0], x[m - 1, n // 2] = math.inf, math.nan, -math.inf
    bad = torch.zeros((m,), dtype=torch.bool)
    bad[[1, 3, m - 1]] = True
    gamma, beta = matrix(1, n, 0, "f32", 2)[0], matrix(1, n, 0, "f32", 3)[0]
    y, mean, rstd = held(m, n, pad, y_type), torch.zeros((m,), device="cuda"), torch.zeros((m,), device="cuda")
    op = c.LayerNorm(STORAGE[x_type], STORAGE[y_type])
    ok(op(op.Arguments(c.RowsCoord(m, n), ref(x), gamma, beta, ref(y), mean, rstd, 1e-5)))
    want = H.layer_norm(x[:, :n].double().cpu(), gamma.double().cpu(), beta.double().cpu(), 1e-5, y_type)
    for got, w in zip((y[:m, :n], mean, rstd), want):
        assert equal_where_not_finite(got, w[0]) and worst_finite(got, w) <= 1
    assert bool(torch.isnan(y[:m, :n].cpu()[bad]).all()) and bool(torch.isfinite(y[:m, :n].cpu()[~bad]).all())
    assert unguarded(y, m, n)


@pytest.mark.parametrize("x_type,y_type", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("m,n,pad", NORMS)
def test_layer_norm_grad_keeps_infinities_and_nan_in_their_rows(gpu, x_type, y_type, m, n, pad):
    x, dy, dr = matrix(m, n, pad, x_type, 1, 2.0), matrix(m, n, pad, y_type, 2), matrix(m, n, pad, x_type, 3)
    x64 = x[:, :n].double().cpu()
    mean, rstd = x64.mean(1).float().cuda(), (1 / torch.sqrt(x64.var(1, correction=0) + 1e-5)).float().cuda()
    for v in (x, dy, dr):
        v[:, n:] = math.nan
    x[1, n - 1], dy[3, 0], dy[m - 1, n // 2], dr[5, 7] = math.nan, math.inf, math.nan, -math.inf
    gamma = matrix(1, n, 0, "f32", 4)[0]
    for residual in (False, True):
        dx, dgamma, dbeta = held(m, n, pad, x_type), torch.zeros((n,), device="cuda"), torch.zeros((n,), device="cuda")
        op = c.LayerNormGrad(STORAGE[x_type], STORAGE[y_type])
        ok(op(op.Arguments(c.RowsCoord(m, n), ref(dy), ref(x), gamma, mean, rstd, ref(dx), dgamma, dbeta, ref(dr if residual else None))))
        want = H.layer_norm_grad(dy[:, :n].double().cpu(), x[:, :n].double().cpu(), gamma.double().cpu(), mean.double().cpu(),
                                 rstd.double().cpu(), dr[:, :n].double().cpu() if residual else None, x_type)
        for got, w in zip((dx[:m, :n], dgamma, dbeta), want):
            assert equal_where_not_finite(got, w[0]) and worst_finite(got, w) <= 1
        assert unguarded(dx, m, n)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,pad", [(70, 515, 3), (1000, 264, 8), (301, 1023, 2)])
def test_epilogue_grad_keeps_infinities_and_nan_in_their_columns(gpu, kind, m, n, pad):
    dy, z = matrix(m, n, pad, kind, 1), matrix(m, n, pad, kind, 2)
    dy[:, n:], z[:, n:] = math.nan, math.nan
    dy[3, 0], dy[m - 1, n - 1], z[9, 5] = math.inf, math.nan, math.nan
    for name in ("none", "relu", "gelu", "silu"):
        dz, dbias = held(m, n, pad, kind), torch.full((n + 1,), GUARD, device="cuda")
        op = c.BiasActivationGrad(STORAGE[kind], ACT[name])
        ok(op(op.Arguments(c.RowsCoord(m, n), ref(dy), ref(None if name == "none" else z), ref(dz), dbias)))
        z64, dy64 = z[:, :n].double().cpu(), dy[:, :n].double().cpu()
        if name == "relu":   # (a slope of zero is not a product with zero)
            dy64 = torch.where(z64 <= 0, torch.zeros_like(dy64), dy64)
        want, sums = H.epilogue_grad(dy64, z64, name, kind)
        for got, w in ((dz[:m, :n], want), (dbias[:n], sums)):
            assert equal_where_not_finite(got, w[0]) and worst_finite(got, w) <= 1
        assert unguarded(dz, m, n) and float(dbias[n]) == GUARD


@pytest.mark.parametrize("m,n,k", [(200, 300, 100), (8, 300, 500), (600, 520, 1000)])
@pytest.mark.parametrize("d", ["f32", "bf16"])
def test_product_beside_infinities(gpu, m, n, k, d):
    """Rows and columns without them have their values, whatever lies behind the rows of A and W."""
    a, w = matrix(m, k, 12, "bf16", 1), matrix(n, k, 4, "bf16", 2)
    a[:, k:], w[:, k:] = math.nan, math.inf
    a[3, 5], w[7, 2] = math.inf, math.nan
    for pad in (0, 1):
        D = held(m, n, pad, d)
        op = c.GemmBF16(c.RowMajor, c.ColumnMajor, storage_d=STORAGE[d])
        ok(op(op.Arguments(c.GemmCoord(m, n, k), ref(a), ref(w), c.TensorRef(), ref(D))))
        value, bound = H.product(a[:, :k].double().cpu(), w[:, :k].double().cpu().t(), None, "none", None, 1.0, 0.0, d)[0]
        assert equal_where_not_finite(D[:m, :n], value)
        keep = torch.ones((m, n), dtype=torch.bool)
        keep[3], keep[:, 7] = False, False
        assert bool(torch.isfinite(value[keep]).all())
        assert H.worst(D[:m, :n].cpu()[keep], (value[keep], bound[keep])) <= 1
        assert unguarded(D, m, n)
