"""16-bit layers and their gradients on the GPU, against their formulas in 64 bits."""
import math

import pytest
import torch

import cpu_ops_b200 as c
from cpu_ops_b200 import _capi
from tests import dense_helpers as H

pytestmark = pytest.mark.gpu
S = c.Status
STORAGE = {"f32": c.f32_t, "f16": c.f16_t, "bf16": c.bf16_t}
ACT = {"none": None, "relu": c.Relu(), "gelu": c.Gelu(), "silu": c.Silu()}
GEMM = {"f16": c.GemmF16, "bf16": c.GemmBF16}
GUARD = 77.0


def ok(status):
    assert status == S.kSuccess, _capi.last_error()


def matrix(rows, cols, pad, kind, seed, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, cols + pad), generator=g) * sigma).to(H.TYPES[kind]).cuda()


def held(rows, cols, pad, kind):
    """An output whose every element, padding and the row behind the last included, holds a guard."""
    return torch.full((rows + 1, cols + pad), GUARD, dtype=H.TYPES[kind], device="cuda")


def unguarded(out, rows, cols):
    rest = out.clone()
    rest[:rows, :cols] = GUARD
    return bool((rest == GUARD).all())


def ref(x):
    return c.TensorRef() if x is None else c.TensorRef(x, x.shape[1])


def run_product(m, n, k, kind="bf16", d="bf16", a="row", b="col", name="none", bias=True, residual=False, z=False, pad=0,
                alpha=1.0, beta=1.0, slices=0, seed=1, **force):
    A = matrix(m, k, pad, kind, seed) if a == "row" else matrix(k, m, pad, kind, seed)
    sigma = 1 / math.sqrt(max(1, k))
    B = matrix(k, n, pad, kind, seed + 1, sigma) if b == "row" else matrix(n, k, pad, kind, seed + 1, sigma)
    C = matrix(m, n, pad, d, seed + 2) if residual else None
    v = matrix(1, n, 0, "f32", seed + 3)[0] if bias else None
    D, Z = held(m, n, pad, d), held(m, n, pad, d) if z else None
    layout = {"row": c.RowMajor, "col": c.ColumnMajor}
    op = GEMM[kind](layout[a], layout[b], storage_d=STORAGE[d], **force)
    ok(op(op.Arguments(c.GemmCoord(m, n, k), ref(A), ref(B), ref(C), ref(D),
                       c.BiasActivation(v, ACT[name], alpha, beta if residual else 0.0), ref(Z), slices)))
    plan = _capi.last_plan()
    a64 = A[:, :k].double().cpu() if a == "row" else A[:, :m].double().cpu().t()
    b64 = B[:, :n].double().cpu() if b == "row" else B[:, :k].double().cpu().t()
    want_d, want_z = H.product(a64, b64, None if v is None else v.double().cpu(), name,
                               None if C is None else C[:, :n].double().cpu(), alpha, beta, d)
    assert H.worst(D[:m, :n], want_d) <= 1
    assert unguarded(D, m, n)
    if z:
        assert H.worst(Z[:m, :n], want_z) <= 1
        assert unguarded(Z, m, n)
    return plan, D


SIZES = [(1, 1, 1), (1, 130, 64), (5, 17, 33), (64, 40, 200), (130, 200, 96), (257, 384, 640), (300, 72, 1000), (16, 512, 2048)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("a", ["row", "col"])
@pytest.mark.parametrize("b", ["row", "col"])
def test_product_layouts(gpu, m, n, k, a, b):
    i = SIZES.index((m, n, k))
    names = ["none", "relu", "gelu", "silu"]
    for j, (kind, d, pad) in enumerate([("bf16", "bf16", 0), ("f16", "f16", 8), ("bf16", "f32", 3), ("f16", "f32", 0)]):
        run_product(m, n, k, kind, d, a, b, names[(i + j) % 4], bias=j != 1, residual=j % 2 == 0, z=j >= 1, pad=pad,
                    alpha=0.5 if j == 3 else 1.0, beta=-1.5 if j == 2 else 1.0)


@pytest.mark.parametrize("pair,tile", [(True, 128), (True, 192), (True, 256), (False, 32), (False, 64),
                                       (False, 128), (False, 256)])
@pytest.mark.parametrize("a,b", [("row", "col"), ("row", "row"), ("col", "row"), ("col", "col")])
def test_product_tiles(gpu, pair, tile, a, b):
    """Each persistent form, more tiles than CTAs take at once among the sizes, all epilogues."""
    if b == "row" and (tile // 2 if pair else tile) % 64:
        pytest.skip("no whole boxes of 64 columns")
    for j, (m, n, k, d, pad) in enumerate([(700, 900, 200, "bf16", 0), (512, 770, 320, "f32", 2), (2500, 2600, 136, "bf16", 0)]):
        plan, _ = run_product(m, n, k, "bf16", d, a, b, ["gelu", "none", "silu"][j], residual=True, z=j != 1, pad=pad + (-n) % 8,
                              pair=pair, tile_n=tile, slices=1)
        assert (plan.pair, plan.tile_n, plan.slices) == (int(pair), tile, 1)


@pytest.mark.parametrize("slices", [1, 2, 4, 8])
@pytest.mark.parametrize("tile", [16, 32, 64, 128])
@pytest.mark.parametrize("m", [3, 40, 200])
def test_product_parts(gpu, slices, tile, m):
    for j, (a, b, d) in enumerate([("row", "col", "bf16"), ("row", "row", "f32"), ("col", "row", "bf16")]):
        if tile < 64 and j:
            continue  # (a narrow tile's operand lies along k)
        if m == 200 and tile == 16 and slices == 1:
            continue  # (whole products of rows come in tiles of 32 columns and more)
        plan, _ = run_product(m, 300, 777, "bf16", d, a, b, "gelu" if j == 0 else "none", residual=j != 1, z=j == 0, pad=3,
                              tile_n=tile, slices=slices)
        assert (plan.slices, plan.tile_n) == (slices, tile)


def test_product_parts_add_to_the_same_sum(gpu):
    """The parts of k are added in order: a repeated call gives the same bits."""
    one = run_product(24, 500, 4096, slices=8, tile_n=32)[1]
    two = run_product(24, 500, 4096, slices=8, tile_n=32)[1]
    assert torch.equal(one, two)


@pytest.mark.parametrize("k", [0, 1])
def test_product_without_k(gpu, k):
    m, n = 37, 70
    bias = matrix(1, n, 0, "f32", 4)[0]
    C, D, Z = matrix(m, n, 2, "f16", 5), held(m, n, 3, "f32"), held(m, n, 1, "f32")
    A = torch.zeros((m, max(k, 1)), dtype=torch.float16, device="cuda")
    B = torch.ones((n, max(k, 1)), dtype=torch.float16, device="cuda")
    op = c.GemmF16(c.RowMajor, c.ColumnMajor, storage_c=c.f16_t, storage_d=c.f32_t)
    ok(op(op.Arguments(c.GemmCoord(m, n, k), ref(A), ref(B), ref(C), ref(D), c.BiasActivation(bias, c.Silu(), beta=2.0), ref(Z))))
    want_d, want_z = H.product(torch.zeros((m, 1), dtype=torch.float64), torch.zeros((1, n), dtype=torch.float64), bias.double().cpu(),
                               "silu", C[:, :n].double().cpu(), 1.0, 2.0, "f32")
    assert H.worst(D[:m, :n], want_d) <= 1 and H.worst(Z[:m, :n], want_z) <= 1
    assert unguarded(D, m, n) and unguarded(Z, m, n)


@pytest.mark.parametrize("m,n,k,pad", [(300, 520, 192, 0), (300, 520, 192, 3), (9, 520, 700, 0)])
def test_product_in_place_and_unread_residual(gpu, m, n, k, pad):
    A, B = matrix(m, k, 0, "bf16", 1), matrix(n, k, 0, "bf16", 2, 0.1)
    start = matrix(m, n, pad, "bf16", 3)
    D = start.clone()
    op = c.GemmBF16(c.RowMajor, c.ColumnMajor)
    ok(op(op.Arguments(c.GemmCoord(m, n, k), ref(A), ref(B), ref(D), ref(D), c.BiasActivation(beta=1.0))))
    want, _ = H.product(A.double().cpu(), B.double().cpu().t(), None, "none", start[:, :n].double().cpu(), 1.0, 1.0, "bf16")
    assert H.worst(D[:, :n], want) <= 1
    nothing = torch.full_like(D, math.nan)
    ok(op(op.Arguments(c.GemmCoord(m, n, k), ref(A), ref(B), ref(nothing), ref(D), c.BiasActivation(beta=0.0))))
    want, _ = H.product(A.double().cpu(), B.double().cpu().t(), None, "none", None, 1.0, 0.0, "bf16")
    assert H.worst(D[:, :n], want) <= 1


@pytest.mark.parametrize("m,n,k", [(200, 300, 100), (8, 300, 500)])
def test_product_infinities_stay_in_their_rows(gpu, m, n, k):
    """NaN and infinities of a row of A and of a row of W reach D's row and column, and nothing else: not from
    what lies behind a row's k elements either."""
    A, B = matrix(m, k, 12, "bf16", 1), matrix(n, k, 4, "bf16", 2)
    A[:, k:] = math.nan
    B[:, k:] = math.inf
    A[3, 5], B[7, 2] = math.inf, math.nan
    D = held(m, n, 0, "f32")
    op = c.GemmBF16(c.RowMajor, c.ColumnMajor, storage_d=c.f32_t)
    ok(op(op.Arguments(c.GemmCoord(m, n, k), ref(A), ref(B), c.TensorRef(), ref(D))))
    want = A[:, :k].double().cpu() @ B[:, :k].double().cpu().t()
    want = torch.where(torch.isfinite(want), want, want)
    assert torch.equal(torch.isnan(D[:m].cpu()), torch.isnan(want)) and torch.equal(torch.isinf(D[:m].cpu()), torch.isinf(want))
    assert unguarded(D, m, n)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
def test_epilogue_grad(gpu, kind, name):
    for m, n, pad in [(1, 1, 0), (1, 300, 0), (33, 256, 0), (70, 515, 3), (1000, 264, 8), (3000, 40, 1), (777, 511, 0), (400, 256, 1), (301, 1023, 2)]:
        dy, z = matrix(m, n, pad, kind, 1), matrix(m, n, pad, kind, 2, 3.0)
        dz, dbias = held(m, n, pad, kind), torch.full((n + 1,), GUARD, device="cuda")
        op = c.BiasActivationGrad(STORAGE[kind], ACT[name])
        ok(op(op.Arguments(c.RowsCoord(m, n), ref(dy), ref(None if name == "none" else z), ref(dz), dbias)))
        want, sums = H.epilogue_grad(dy[:, :n].double().cpu(), z[:, :n].double().cpu(), name, kind)
        assert H.worst(dz[:m, :n], want) <= 1 and H.worst(dbias[:n], sums) <= 1
        assert unguarded(dz, m, n) and float(dbias[n]) == GUARD


def test_epilogue_grad_in_place_and_alone(gpu):
    m, n = 200, 333
    dy, z = matrix(m, n, 1, "bf16", 1), matrix(m, n, 1, "bf16", 2)
    want, sums = H.epilogue_grad(dy[:, :n].double().cpu(), z[:, :n].double().cpu(), "gelu", "bf16")
    op = c.BiasActivationGrad(c.bf16_t, c.Gelu())
    for place in (0, 1):
        a, b = dy.clone(), z.clone()
        ok(op(op.Arguments(c.RowsCoord(m, n), ref(a), ref(b), ref((a, b)[place]))))
        assert H.worst((a, b)[place][:, :n], want) <= 1
    dbias = torch.zeros((n,), device="cuda")
    op = c.BiasActivationGrad(c.bf16_t)
    ok(op(op.Arguments(c.RowsCoord(m, n), ref(dy), dbias=dbias)))
    assert H.worst(dbias, H.epilogue_grad(dy[:, :n].double().cpu(), None, "none", "bf16")[1]) <= 1
    ok(op(op.Arguments(c.RowsCoord(0, n), c.TensorRef(), dbias=dbias)))   # no rows: a sum of nothing
    assert float(dbias.abs().max()) == 0


@pytest.mark.parametrize("name,limits", [("relu", (0, 0, 1, 1)), ("gelu", (0, 0, 1, 1)), ("silu", (0, 0, 1, 1))])
def test_slopes_of_far_values(gpu, name, limits):
    """Infinities and sizes whose square leaves f32 have the limits' slopes; NaN stays."""
    z = torch.tensor([[-math.inf, -1e30, 1e30, math.inf, math.nan, 0.0]], device="cuda")
    dy, dz = torch.full_like(z, 2.0), torch.zeros_like(z)
    op = c.BiasActivationGrad(c.f32_t, ACT[name])
    ok(op(op.Arguments(c.RowsCoord(1, 6), ref(dy), ref(z), ref(dz))))
    got = dz.cpu()[0]
    assert [float(v) for v in got[:4]] == pytest.approx([2.0 * v for v in limits], abs=1e-38)
    assert math.isnan(float(got[4])) == (name != "relu")
    assert float(got[5]) == {"relu": 0.0, "gelu": 1.0, "silu": 1.0}[name]


PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
ROWS = [(1, 1, 0), (3, 5, 0), (1000, 64, 0), (77, 256, 0), (50, 257, 3), (9, 1000, 0), (700, 515, 1), (130, 4096, 0), (5, 4100, 4),
        (400, 8192, 0), (3, 8193, 0), (6, 20000, 8), (700, 2048, 0), (1300, 1032, 8), (601, 4096, 8), (640, 3000, 1), (2, 2047, 2), (300, 300, 0),
        (45, 5001, 0), (640, 264, 0), (600, 5000, 8), (593, 8192, 0), (900, 1000, 0), (2000, 520, 0), (700, 3064, 0),
        (650, 1501, 3), (620, 515, 5), (3, 5001, 7), (600, 5001, 7), (592, 250, 6)]


@pytest.mark.parametrize("x_type,y_type", PAIRS)
@pytest.mark.parametrize("m,n,pad", ROWS)
def test_layer_norm(gpu, x_type, y_type, m, n, pad):
    x = (matrix(m, n, pad, "f32", 1, 2.0) + 3.0).to(H.TYPES[x_type])
    gamma, beta = matrix(1, n, 0, "f32", 2)[0], matrix(1, n, 0, "f32", 3)[0]
    y, mean, rstd = held(m, n, pad, y_type), torch.full((m + 1,), GUARD, device="cuda"), torch.full((m + 1,), GUARD, device="cuda")
    op = c.LayerNorm(STORAGE[x_type], STORAGE[y_type])
    ok(op(op.Arguments(c.RowsCoord(m, n), ref(x), gamma, beta, ref(y), mean, rstd, 1e-5)))
    want = H.layer_norm(x[:, :n].double().cpu(), gamma.double().cpu(), beta.double().cpu(), 1e-5, y_type)
    for got, w in zip((y[:m, :n], mean[:m], rstd[:m]), want):
        assert H.worst(got, w) <= 1
    assert unguarded(y, m, n) and float(mean[m]) == GUARD and float(rstd[m]) == GUARD
    ok(op(op.Arguments(c.RowsCoord(m, n), ref(x), None, None, ref(y))))
    assert H.worst(y[:m, :n], H.layer_norm(x[:, :n].double().cpu(), None, None, 1e-5, y_type)[0]) <= 1


def test_layer_norm_in_place_and_constant_rows(gpu):
    """A row of equal elements has a variance of zero: rstd is 1 / sqrt(eps), y is beta; far from zero too."""
    for n in (200, 4000, 9000):
        x = matrix(6, n, 0, "f32", 1)
        x[2], x[3] = 1e6, -3.0
        beta = matrix(1, n, 0, "f32", 2)[0]
        op = c.LayerNorm(c.f32_t)
        rstd = torch.zeros((6,), device="cuda")
        want = H.layer_norm(x.double().cpu(), None, beta.double().cpu(), 1e-3, "f32")
        ok(op(op.Arguments(c.RowsCoord(6, n), ref(x), None, beta, ref(x), None, rstd, 1e-3)))
        assert H.worst(x, want[0]) <= 1 and H.worst(rstd, want[2]) <= 1


@pytest.mark.parametrize("x_type,y_type", PAIRS)
@pytest.mark.parametrize("m,n,pad", ROWS)
def test_layer_norm_grad(gpu, x_type, y_type, m, n, pad):
    x = (matrix(m, n, pad, "f32", 1, 2.0) + 1.0).to(H.TYPES[x_type])
    dy, dr, gamma = matrix(m, n, pad, y_type, 2), matrix(m, n, pad, x_type, 3), matrix(1, n, 0, "f32", 4)[0]
    x64 = x[:, :n].double().cpu()
    mean = x64.mean(1).float().cuda()
    rstd = (1 / torch.sqrt(x64.var(1, correction=0) + 1e-5)).float().cuda()
    for residual in (False, True):
        dx, dgamma, dbeta = held(m, n, pad, x_type), torch.full((n + 1,), GUARD, device="cuda"), torch.full((n + 1,), GUARD, device="cuda")
        op = c.LayerNormGrad(STORAGE[x_type], STORAGE[y_type])
        ok(op(op.Arguments(c.RowsCoord(m, n), ref(dy), ref(x), gamma, mean, rstd, ref(dx), dgamma, dbeta, ref(dr if residual else None))))
        want = H.layer_norm_grad(dy[:, :n].double().cpu(), x64, gamma.double().cpu(), mean.double().cpu(), rstd.double().cpu(),
                                 dr[:, :n].double().cpu() if residual else None, x_type)
        for got, w in zip((dx[:m, :n], dgamma[:n], dbeta[:n]), want):
            assert H.worst(got, w) <= 1
        assert unguarded(dx, m, n) and float(dgamma[n]) == GUARD and float(dbeta[n]) == GUARD


@pytest.mark.parametrize("n", [100, 3000, 10000])
def test_layer_norm_grad_in_place(gpu, n):
    m = 40
    x, dy, dr = (matrix(m, n, 0, "f16", s) for s in (1, 2, 3))
    x64 = x.double().cpu()
    mean, rstd = x64.mean(1).float().cuda(), (1 / torch.sqrt(x64.var(1, correction=0) + 1e-5)).float().cuda()
    want = H.layer_norm_grad(dy.double().cpu(), x64, None, mean.double().cpu(), rstd.double().cpu(), dr.double().cpu(), "f16")
    op = c.LayerNormGrad(c.f16_t)
    for place in range(3):
        buffers = [x.clone(), dy.clone(), dr.clone()]
        dgamma, dbeta = torch.zeros((n,), device="cuda"), torch.zeros((n,), device="cuda")
        ok(op(op.Arguments(c.RowsCoord(m, n), ref(buffers[1]), ref(buffers[0]), None, mean, rstd, ref(buffers[place]),
                           dgamma if place else None, dbeta, ref(buffers[2]))))
        assert H.worst(buffers[place], want[0]) <= 1 and H.worst(dbeta, want[2]) <= 1
        if place:
            assert H.worst(dgamma, want[1]) <= 1
    ok(op(op.Arguments(c.RowsCoord(0, n), c.TensorRef(), c.TensorRef(), dgamma=dgamma, dbeta=dbeta)))
    assert float(dgamma.abs().max()) == 0 and float(dbeta.abs().max()) == 0


def run_balance(tokens, experts, top_k, kind, sigmoid, pad=0, edit=None, upstream=None):
    logits = matrix(tokens, experts, pad, kind, 1, 1.5)
    g = torch.Generator().manual_seed(5)
    ids = torch.stack([torch.randperm(experts, generator=g)[:top_k] for _ in range(tokens)]) if tokens else torch.zeros((0, top_k))
    ids = ids.int()
    if edit:
        edit(logits, ids)
    counts, loss = torch.full((experts + 1,), -5, dtype=torch.int32, device="cuda"), torch.full((2,), GUARD, device="cuda")
    d = held(tokens, experts, pad, kind)
    op = c.BalanceLoss(STORAGE[kind])
    up = None if upstream is None else torch.tensor([upstream], device="cuda")
    dev_ids = ids.cuda()
    ok(op(op.Arguments(c.RouteCoord(tokens, experts, top_k), ref(logits), dev_ids, counts, loss, ref(d),
                       c.Scoring.kSigmoid if sigmoid else c.Scoring.kSoftmax, 0.02, up)))
    want = H.balance(logits[:, :experts].double().cpu(), ids, sigmoid, float(torch.tensor(0.02)),
                     1.0 if upstream is None else float(torch.tensor(upstream)), kind)
    assert torch.equal(counts[:experts].cpu().long(), want[0].long()) and int(counts[experts]) == -5
    assert H.worst(loss[:1], (want[1][0].reshape(1), want[1][1].reshape(1) + 1e-30)) <= 1 and float(loss[1]) == GUARD
    assert H.worst(d[:tokens, :experts], (want[2][0], want[2][1] + 1e-37)) <= 1
    assert unguarded(d, tokens, experts)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 8, 2), (7, 60, 4), (32, 64, 8), (33, 64, 8), (300, 33, 3), (700, 256, 8),
                                                  (1500, 100, 5), (260, 1000, 6)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_balance_loss(gpu, tokens, experts, top_k, sigmoid):
    for kind, pad, upstream in (("f32", 0, None), ("bf16", 3, 0.7), ("f16", 0, 32.0)):
        run_balance(tokens, experts, top_k, kind, sigmoid, pad, upstream=upstream)


@pytest.mark.parametrize("tokens", [20, 500])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_balance_loss_edges(gpu, tokens, sigmoid):
    """Padding tokens, ids out of range, experts that are out of a token's scores, far logits."""
    def edit(logits, ids):
        ids[-5:] = -1
        ids[3, 0], ids[4, 1] = 40, -7            # beyond the experts
        logits[0, :3] = -math.inf
        logits[1, 2] = math.nan
        logits[2, 4] = math.inf
        logits[6] = -500.0                       # logistics that vanish in f32
        logits[7] = -math.inf                    # no expert left, though it has ids
        logits[8] = 200.0
        logits[-1] = math.nan                    # a padding token's logits do not count
    run_balance(tokens, 24, 2, "f32", sigmoid, 1, edit)


def test_balance_loss_without_pairs(gpu):
    def none(logits, ids):
        ids[:] = -1
    for tokens in (0, 9, 100):
        run_balance(tokens, 16, 2, "f32", False, 0, none)


def test_balance_loss_outputs_are_optional(gpu):
    tokens, experts = 200, 16
    logits = matrix(tokens, experts, 0, "f32", 1)
    ids = torch.randint(0, experts, (tokens, 2), dtype=torch.int32, device="cuda")
    counts, loss, d = torch.zeros((experts,), dtype=torch.int32, device="cuda"), torch.zeros((1,), device="cuda"), torch.zeros_like(logits)
    op = c.BalanceLoss()
    size = c.RouteCoord(tokens, experts, 2)
    ok(op(op.Arguments(size, ref(logits), ids, counts, loss, ref(d))))
    assert torch.equal(counts.cpu(), torch.bincount(ids.flatten().cpu().long(), minlength=experts).int())
    other, alone = torch.zeros_like(counts), torch.zeros_like(loss)
    ok(op(op.Arguments(size, ref(logits), ids, counts=other)))
    ok(op(op.Arguments(size, ref(logits), ids, loss=alone)))
    assert torch.equal(other, counts) and torch.equal(alone, loss)
    ok(op(op.Arguments(size, ref(logits), ids, ref_dLogits=ref(logits))))   # in place
    assert torch.equal(logits, d)


def shifted(rows, cols, pad, kind, seed, by, sigma=1.0):
    """A matrix that begins `by` elements behind an aligned address; -> the view and its TensorRef."""
    flat = torch.full((rows * (cols + pad) + by + 8,), GUARD, dtype=H.TYPES[kind], device="cuda")
    view = flat[by:by + rows * (cols + pad)].view(rows, cols + pad)
    if seed is not None:
        view[:, :cols] = matrix(rows, cols, 0, kind, seed, sigma)
    return view, c.TensorRef(view, cols + pad)


@pytest.mark.parametrize("m,n", [(40, 600), (650, 1200), (650, 200)])
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("offsets", [(1, 0, 1, 0), (0, 1, 0, 1), (3, 3, 2, 5)])
def test_operands_that_begin_anywhere(gpu, m, n, pad, offsets):
    """Every operand at its own distance from an aligned address: rows of different shifts in one call."""
    (x, rx), (dy, rdy), (dr, rdr) = (shifted(m, n, pad, "bf16", i, by) for i, by in enumerate(offsets[:3]))
    out, rout = shifted(m, n, pad, "bf16", None, offsets[3])
    x64, dy64, dr64 = (v[:, :n].double().cpu() for v in (x, dy, dr))
    gamma = matrix(1, n, 0, "f32", 7)[0]
    mean, rstd = torch.zeros((m,), device="cuda"), torch.zeros((m,), device="cuda")
    op = c.LayerNorm(c.bf16_t)
    ok(op(op.Arguments(c.RowsCoord(m, n), rx, gamma, None, rout, mean, rstd, 1e-5)))
    for got, want in zip((out[:, :n], mean, rstd), H.layer_norm(x64, gamma.double().cpu(), None, 1e-5, "bf16")):
        assert H.worst(got, want) <= 1
    dgamma, dbeta, dbias = (torch.zeros((n,), device="cuda") for _ in range(3))
    op = c.LayerNormGrad(c.bf16_t)
    ok(op(op.Arguments(c.RowsCoord(m, n), rdy, rx, gamma, mean, rstd, rout, dgamma, dbeta, rdr)))
    want = H.layer_norm_grad(dy64, x64, gamma.double().cpu(), mean.double().cpu(), rstd.double().cpu(), dr64, "bf16")
    for got, w in zip((out[:, :n], dgamma, dbeta), want):
        assert H.worst(got, w) <= 1
    op = c.BiasActivationGrad(c.bf16_t, c.Gelu())
    ok(op(op.Arguments(c.RowsCoord(m, n), rdy, rx, rout, dbias)))
    want, sums = H.epilogue_grad(dy64, x64, "gelu", "bf16")
    assert H.worst(out[:, :n], want) <= 1 and H.worst(dbias, sums) <= 1
    w, rw = shifted(n, 72, pad, "bf16", 9, offsets[1], n ** -0.5)
    d, rd = shifted(m, 72, pad, "bf16", None, offsets[3])
    r, rr = shifted(m, 72, pad, "bf16", 10, offsets[2])
    op = c.GemmBF16(c.RowMajor, c.RowMajor)
    ok(op(op.Arguments(c.GemmCoord(m, 72, n), rx, rw, rr, rd, c.BiasActivation(beta=1.0))))
    want, _ = H.product(x64, w[:, :72].double().cpu(), None, "none", r[:, :72].double().cpu(), 1.0, 1.0, "bf16")
    assert H.worst(d[:, :72], want) <= 1
    for v, cols in ((out, n), (d, 72)):
        assert pad == 0 or bool((v[:, cols:] == GUARD).all())
