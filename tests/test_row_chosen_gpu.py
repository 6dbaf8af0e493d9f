"""Routing, row plans, the experts' products and low-rank adapters against plain 64-bit forms, at
the sizes and masks where they can go wrong."""
import numpy as np
import pytest
import torch

import cpu_ops_b200 as c
from cpu_ops_b200 import _capi, workloads as W
from tests import row_chosen_helpers as H

pytestmark = pytest.mark.gpu

STORAGE = {_capi.FMT_E4M3: c.fp8e4m3_t, _capi.FMT_E5M2: c.fp8e5m2_t, _capi.FMT_E2M1: c.fp4e2m1_t}
E4, E5, F4 = _capi.FMT_E4M3, _capi.FMT_E5M2, _capi.FMT_E2M1
FLOATS = {"f32": (torch.float32, c.f32_t), "f16": (torch.float16, c.f16_t), "bf16": (torch.bfloat16, c.bf16_t)}
OK = c.Status.kSuccess


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def check(status):
    assert status == OK, (status, _capi.last_error())


# ---- routing ---------------------------------------------------------------------------------


def run_route(logits, kind, top_k, bias=None, sigmoid=False, n_groups=1, top_groups=1, group_best=1, renormalize=True,
              scale=1.0, ld=None, plan=True, **op_args):
    tokens, experts = logits.shape
    ids = torch.full((tokens, top_k), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((tokens, top_k), float("nan"), device="cuda")
    offsets = torch.full((experts + 1,), -7, dtype=torch.int32, device="cuda")
    order = torch.full((tokens * top_k,), -7, dtype=torch.int32, device="cuda")
    op = c.RouteExperts(FLOATS[kind][1], **op_args)
    check(op(op.Arguments(c.RouteCoord(tokens, experts, top_k), c.TensorRef(logits, ld or experts), ids, weights,
                          c.RowPlan(offsets, order) if plan else None,
                          c.Scoring.kSigmoid if sigmoid else c.Scoring.kSoftmax, bias,
                          c.ExpertGroups(n_groups, top_groups, group_best), renormalize, scale)))
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in (ids, weights, offsets, order)]


def check_route(logits, kind, top_k, bias=None, **kw):
    got = run_route(logits, kind, top_k, bias=None if bias is None else dev(bias), **kw)
    options = {"sigmoid": False, "n_groups": 1, "top_groups": 1, "group_best": 1, "renormalize": True, "scale": 1.0}
    options.update({k: v for k, v in kw.items() if k in options})
    ids, weights = H.route(logits.double().cpu().numpy(), bias, top_k, **options)
    assert np.array_equal(got[0], ids)
    # formed in 64 bits, rounded once: half a step of f32, and as much for the 64-bit roundings
    assert np.all(np.abs(got[1] - weights) <= np.finfo(np.float32).eps * np.abs(weights) + 1e-45)
    offsets, order = H.plan_of(ids, logits.shape[1])
    assert np.array_equal(got[2], offsets) and np.array_equal(got[3], order)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 2, 2), (3, 31, 5), (7, 32, 32), (33, 33, 2),
                                                  (64, 64, 8), (5, 100, 7), (9, 256, 8), (17, 257, 6), (4, 1000, 32),
                                                  (2, 1024, 10), (700, 60, 6)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_sizes(gpu, tokens, experts, top_k, sigmoid):
    rng = W.rng_for(tokens * 1000 + experts, 3)
    logits = dev((2 * rng.standard_normal((tokens, experts))).astype(np.float32))
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    check_route(logits, "f32", top_k, sigmoid=sigmoid)
    check_route(logits, "f32", top_k, bias=bias, sigmoid=sigmoid, renormalize=False, scale=2.5)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("experts,n_groups,top_groups,best", [(16, 4, 2, 1), (64, 8, 3, 2), (256, 8, 4, 2), (12, 12, 5, 2),
                                                              (6, 2, 1, 2), (96, 3, 3, 1), (1024, 64, 7, 2)])
def test_route_groups_and_types(gpu, kind, experts, n_groups, top_groups, best):
    rng = W.rng_for(experts, 4)
    logits = dev((2 * rng.standard_normal((37, experts))).astype(np.float32)).to(FLOATS[kind][0])
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
    for sigmoid in (False, True):
        check_route(logits, kind, min(8, experts), bias=bias, sigmoid=sigmoid, n_groups=n_groups,
                    top_groups=top_groups, group_best=best)


def test_route_ties_go_to_the_lowest_index(gpu):
    rng = W.rng_for(5, 5)
    logits = dev(rng.integers(-2, 3, (200, 70)).astype(np.float32))
    check_route(logits, "f32", 9)
    check_route(logits, "f32", 9, sigmoid=True, n_groups=7, top_groups=3)
    check_route(torch.zeros((5, 40), device="cuda"), "f32", 32)


def test_route_masks_infinities_and_nan(gpu):
    rng = W.rng_for(6, 5)
    x = rng.standard_normal((12, 48)).astype(np.float32)
    x[0] = -np.inf                     # nothing left
    x[1] = np.nan
    x[2, 3:] = -np.inf                 # fewer than top_k left
    x[3, ::2] = np.finfo(np.float32).min
    x[4, 5] = np.inf
    x[5, [5, 9]] = np.inf              # two share
    x[6] = np.finfo(np.float32).min
    x[7, 10] = np.nan
    x[8, :16] = -np.inf                # a whole group of three
    x[9] = 1e4 * x[9]
    bias = (0.1 * rng.standard_normal(48)).astype(np.float32)
    bias[[1, 20]] = -np.inf
    bias[2] = np.nan
    for sigmoid in (False, True):
        for b in (None, bias):
            check_route(dev(x), "f32", 5, bias=b, sigmoid=sigmoid)
            check_route(dev(x), "f32", 5, bias=b, sigmoid=sigmoid, n_groups=3, top_groups=2, group_best=2)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_choices_that_f32_cannot_settle(gpu, sigmoid):
    """Scores a rounding of f32 apart, saturated ones, zeros of either sign, numbers below every digit."""
    rng = W.rng_for(10, 5)
    x = np.zeros((24, 64), np.float32)
    base = rng.standard_normal(24).astype(np.float32)
    for t in range(24):   # neighbours one or two steps of f32 apart, shuffled
        steps = rng.permutation(64) % 13
        v = np.full(64, base[t], np.float32)
        for j in range(64):
            for _ in range(int(steps[j])):
                v[j] = np.nextafter(v[j], np.float32(np.inf))
        x[t] = v
    x[4] = rng.permutation(np.concatenate((np.float32([20, 25, 28, 30]).repeat(8), np.arange(45, 77)))).astype(np.float32)
    x[5] = -x[4]
    x[6] = np.where(np.arange(64) % 3 == 0, -0.0, 0.0)
    x[7] = rng.permutation(64).astype(np.float32) * np.float32(1e-30)
    x[8] = rng.permutation(64).astype(np.float32) * np.float32(-1000)
    x[9] = rng.permutation(64).astype(np.float32) * np.float32(40)
    bias = rng.permutation((np.float32(0.25) + np.arange(64) * np.float32(2.0 ** -24))).astype(np.float32)
    for b in (None, bias):
        for kw in ({}, {"n_groups": 8, "top_groups": 3, "group_best": 2}, {"n_groups": 64, "top_groups": 20}):
            check_route(dev(x), "f32", 7, bias=b, sigmoid=sigmoid, **kw)


def test_route_padded_rows_and_no_plan(gpu):
    rng = W.rng_for(8, 5)
    wide = dev(rng.standard_normal((19, 45)).astype(np.float32))
    check_route(wide[:, :40], "f32", 3, ld=45)
    ids, weights, offsets, order = run_route(wide[:, :40], "f32", 3, ld=45, plan=False)
    assert (offsets == -7).all() and (order == -7).all() and (ids >= 0).all()
    run_route(torch.zeros((0, 8), device="cuda"), "f32", 2)


@pytest.mark.parametrize("rows,groups", [(0, 5), (1, 1), (31, 3), (1000, 64), (4096, 1024), (4097, 7), (30000, 255),
                                         (70000, 1023), (131072, 3), (131073, 37)])
def test_group_rows(gpu, rows, groups):
    ids = W.rng_for(rows, 6).integers(-2, groups + 2, rows).astype(np.int32)
    offsets = torch.full((groups + 1,), -7, dtype=torch.int32, device="cuda")
    order = torch.full((max(rows, 1),), -7, dtype=torch.int32, device="cuda")
    op = c.GroupRows()
    check(op(op.Arguments(rows, groups, dev(ids), c.RowPlan(offsets, order))))
    want = H.plan_of(ids, groups)
    assert np.array_equal(offsets.cpu().numpy(), want[0])
    assert np.array_equal(order.cpu().numpy()[:rows], want[1])


# ---- the experts' products -----------------------------------------------------------------------


class Experts:
    """Operands of one call: `pairs_per_a_row` pairs share a row of A."""

    def __init__(self, fa, fb, rows, n, k, groups, gated=False, share=1, seed=0, pad=0, lds=None, gap=0, ids=None,
                 offset=0):
        rng = W.rng_for(seed, 7)
        self.fa, self.fb, self.rows, self.n, self.k, self.groups = fa, fb, rows, n, k, groups
        self.gated, self.share = gated, share
        n_b = 2 * n if gated else n
        self.a_rows, self.group_rows = -(-rows // share), n_b + gap
        mixed = fb == F4 and fa != F4
        step = 64 if mixed else 32
        self.ld = -(-k // step) * step + pad
        self.lds = lds or -(-k // 32)
        b_rows = groups * self.group_rows
        self.A = W.mx_elements(fa, self.a_rows, k, self.ld, rng).reshape(self.a_rows, -1)
        self.B = W.mx_elements(fb, b_rows, k, self.ld, rng).reshape(b_rows, -1)
        self.SA = W.mx_scales(self.a_rows, self.lds, 120, 126, rng)
        self.SB = W.mx_scales(b_rows, self.lds, 117, 123, rng)
        self.ids = rng.integers(0, groups, rows).astype(np.int32) if ids is None else np.asarray(ids, np.int32)
        self.weights = rng.random(rows).astype(np.float32)
        self.offset = offset  # bytes by which the scale arrays are moved off their alignment

    def dense(self):
        A = H.decode_mx(self.A, self.SA.reshape(-1, self.lds), self.fa, self.k)
        B = H.decode_mx(self.B, self.SB.reshape(-1, self.lds), self.fb, self.k)
        B = B.reshape(self.groups, self.group_rows, self.k)[:, :2 * self.n if self.gated else self.n]
        return A, B

    def moved(self, x):
        buf = torch.zeros(x.size + self.offset, dtype=torch.uint8, device="cuda")
        buf[self.offset:] = dev(x)
        return buf[self.offset:]

    def run(self, weighted=False, summed=1, plan=None, D=None, ldd=None, **op_args):
        d_rows = self.rows // summed
        ldd = ldd or self.n
        if D is None:
            D = torch.full((d_rows, ldd), 7.5, device="cuda")
        offsets, order = plan or H.plan_of(self.ids, self.groups)
        self.keep = [dev(self.A), dev(self.B), self.moved(self.SA), self.moved(self.SB), dev(offsets), dev(order),
                     dev(self.weights), dev(self.ids)]
        A, B, SA, SB, off, ordr, weights, ids = self.keep
        op = c.GemmMxGrouped(STORAGE[self.fa], STORAGE[self.fb], gated=self.gated, **op_args)
        self.args = op.Arguments(
            c.GroupedCoord(self.rows, self.n, self.k, self.groups), c.MxTensorRef(A, SA, self.ld, self.lds),
            c.MxTensorRef(B, SB, self.ld, self.lds), c.RowPlan(off, ordr), c.TensorRef(D, ldd),
            pairs_per_a_row=self.share, row_weights=weights if weighted else None, pairs_per_d_row=summed,
            ids=ids if summed > 1 else None, b_group_rows=self.group_rows)
        check(op(self.args))
        return D

    def check(self, weighted=False, summed=1, ldd=None):
        D = self.run(weighted, summed, ldd=ldd).cpu().numpy()
        A, B = self.dense()
        want, err = H.grouped(A, B, self.ids, self.n, self.gated, self.share, self.weights if weighted else None, summed,
                              np.full((self.rows // summed, self.n), 7.5))
        got = D[:, :self.n].astype(np.float64)
        assert np.isfinite(got).all()
        assert np.all(np.abs(got - want) <= err), np.max(np.abs(got - want) / np.maximum(err, 1e-300))
        assert (D[:, self.n:] == 7.5).all()
        # far closer than the worst case allows, taken together
        assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want) + 1e-30


PAIRS = [(E4, E4), (E5, E5), (E4, E5), (F4, F4), (E4, F4), (E5, F4)]


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_formats(gpu, fa, fb, gated):
    Experts(fa, fb, 70, 200, 640, 5, gated=gated, share=2, seed=1).check()


# Many pairs per group: A is copied in plan order first.  Narrow outputs take one tile per CTA, wide ones two.
MANY = [(260, 200, 640, 3), (400, 6000, 96, 4), (777, 1000, 320, 2), (650, 5000, 224, 13)]


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,n,k,groups", MANY)
def test_grouped_many_pairs(gpu, fa, fb, gated, rows, n, k, groups):
    if fb == F4 and fa != F4:
        k = 128 * (-(-k // 128))
    before = c.launch_count()
    Experts(fa, fb, rows, n // 2 if gated else n, k, groups, gated=gated, share=2, seed=rows).check()
    assert c.launch_count() - before == 2


@pytest.mark.parametrize("rows,n,k,groups", MANY[:2])
@pytest.mark.parametrize("summed,share", [(1, 1), (2, 1), (4, 4)])
def test_grouped_many_pairs_weights_and_sums(gpu, rows, n, k, groups, summed, share):
    rng = W.rng_for(rows, 7)
    ids = rng.integers(-1, groups, rows)
    ids[:20] = -1
    e = Experts(E4, E4, rows, n, k, groups, share=share, ids=ids, seed=3, gap=5, pad=64)
    e.check(True, summed, ldd=n + 3)
    Experts(F4, F4, rows, n // 3, k, groups, gated=True, share=share, ids=ids, seed=4).check(True, summed)


@pytest.mark.parametrize("rows,n,k,groups", MANY[:2])
@pytest.mark.parametrize("lds,offset", [(32, 0), (32, 4), (21, 3)])
def test_grouped_many_pairs_scales_anywhere(gpu, rows, n, k, groups, lds, offset):
    for fmt, gated in ((E4, True), (F4, False)):
        Experts(fmt, fmt, rows, n, k, groups, gated=gated, share=2, lds=lds, offset=offset, seed=lds).check()


@pytest.mark.parametrize("k", [2, 34, 130, 258, 1002])
def test_grouped_many_pairs_k_inside_a_block(gpu, k):
    for fmt in (E5, F4):
        Experts(fmt, fmt, 200, 5000, k, 2, seed=k).check()


def test_grouped_many_pairs_of_a_plan_that_lies(gpu):
    e = Experts(E4, E4, 300, 72, 128, 4, share=3, seed=8)
    offsets, order = H.plan_of(e.ids, 4)
    bad = order.copy()
    bad[::5] = np.array([1 << 30, -5, 300, -(1 << 31)], np.int64)[np.arange(bad[::5].size) % 4]
    D = e.run(plan=(offsets, bad)).cpu().numpy()
    left = np.setdiff1d(np.arange(300), order[np.arange(300) % 5 != 0])
    assert (D[left] == 7.5).all()
    A, B = e.dense()
    want, err = H.grouped(A, B, np.where(np.isin(np.arange(300), left), -1, e.ids), 72, False, 3, None, 1, np.full((300, 72), 7.5))
    assert np.all(np.abs(D - want) <= err)


def test_grouped_one_large_group_among_many(gpu):
    """Far more pairs in one group than the average the call is planned for."""
    ids = np.where(np.arange(2000) % 50 == 0, np.arange(2000) % 7, 5)
    Experts(E4, E4, 2000, 300, 256, 40, ids=ids, seed=5).check()
    Experts(E4, E4, 2000, 300, 256, 20, gated=True, ids=ids, seed=5).check()


@pytest.mark.parametrize("rows,n,k,groups", [(1, 1, 32, 1), (1, 128, 128, 4), (2, 129, 4096, 3), (16, 64, 96, 1),
                                             (17, 300, 1056, 2), (193, 130, 256, 1), (385, 65, 544, 2),
                                             (1000, 40, 64, 300), (64, 127, 8192, 2), (5, 257, 288, 1024)])
@pytest.mark.parametrize("fmt", [E4, F4])
def test_grouped_sizes(gpu, rows, n, k, groups, fmt):
    Experts(fmt, fmt, rows, n, k, groups, seed=rows).check()


@pytest.mark.parametrize("k", [1, 2, 30, 34, 130, 258, 1002])
def test_grouped_k_inside_a_block(gpu, k):
    Experts(E4, E4, 40, 150, k, 3, seed=k).check()
    if k % 2 == 0:
        Experts(F4, F4, 40, 150, k, 3, gated=True, seed=k).check()


@pytest.mark.parametrize("summed,share", [(1, 1), (2, 1), (3, 3), (8, 1), (8, 8)])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_weights_and_sums(gpu, summed, share, weighted, gated):
    Experts(E4, E4, 24 * 3, 100, 320, 6, gated=gated, share=share, seed=summed).check(weighted, summed, ldd=103)


@pytest.mark.parametrize("lds,offset", [(16, 0), (16, 4), (20, 0), (17, 0), (16, 3), (19, 1)])
@pytest.mark.parametrize("fmt", [E4, F4])
def test_grouped_scales_anywhere(gpu, lds, offset, fmt):
    Experts(fmt, fmt, 90, 140, 480, 3, gated=True, share=2, lds=lds, offset=offset, seed=lds).check()


def test_grouped_strides_between_groups(gpu):
    Experts(E5, E5, 64, 72, 256, 4, gap=9, pad=64, seed=2).check(ldd=80)
    Experts(E4, F4, 64, 72, 256, 4, gated=True, gap=5, pad=64, seed=3).check()


def test_grouped_pairs_in_no_group(gpu):
    rng = W.rng_for(9, 7)
    ids = rng.integers(-1, 5, 60)
    ids[:12] = -1                    # whole rows without any
    for summed in (1, 4):
        Experts(E4, E4, 60, 96, 128, 5, share=2, ids=ids, seed=4).check(summed=summed)
    Experts(E4, E4, 60, 96, 128, 5, ids=np.full(60, -1), seed=4).check()
    Experts(E4, E4, 60, 96, 128, 5, ids=np.full(60, -1), seed=4).check(summed=4)


def test_grouped_all_pairs_in_one_group(gpu):
    Experts(E4, E4, 500, 96, 256, 64, ids=np.full(500, 63), seed=5).check()
    Experts(F4, F4, 500, 96, 256, 64, gated=True, ids=np.full(500, 0), seed=5).check()


def test_grouped_rows_of_others_do_not_leak(gpu):
    """NaN weights of a group without pairs, NaN rows without a group, NaN behind n and k."""
    e = Experts(E4, E4, 50, 72, 200, 4, gap=8, seed=6)
    e.ids[e.ids == 2] = 1
    e.ids[::7] = -1
    e.A[::7] = 0x7F
    e.A[:, 200:] = 0x7F
    B = e.B.reshape(4, 80, -1)
    B[2] = 0x7F
    B[:, 72:] = 0x7F
    B[..., 200:] = 0x7F
    e.check()


def test_grouped_nan_stays_in_its_row_and_column(gpu):
    e = Experts(E4, E4, 40, 72, 256, 2, seed=7)
    e.A[3, 5] = 0x7F
    e.B[int(e.ids[0]) * 72 + 11, 100] = 0x7F
    D = e.run().cpu().numpy()
    nan = np.isnan(D)
    want = np.zeros_like(nan)
    want[3] = True
    want[e.ids == e.ids[0], 11] = True
    assert np.array_equal(nan, want)


def test_grouped_keeps_within_a_plan_that_lies(gpu):
    """Entries of a plan outside the pairs are passed over; nothing else is written."""
    e = Experts(E4, E4, 64, 72, 128, 4, seed=8)
    offsets, order = H.plan_of(e.ids, 4)
    bad = order.copy()
    bad[::5] = np.array([1 << 30, -5, 64, -(1 << 31)], np.int64)[np.arange(bad[::5].size) % 4]
    D = e.run(plan=(offsets, bad)).cpu().numpy()
    left = np.setdiff1d(np.arange(64), order[np.arange(64) % 5 != 0])
    assert (D[left] == 7.5).all()
    A, B = e.dense()
    want, err = H.grouped(A, B, np.where(np.isin(np.arange(64), left), -1, e.ids), 72, False, 1, None, 1, np.full((64, 72), 7.5))
    assert np.all(np.abs(D - want) <= err)
    for lie in ([5, 90, -3, 1 << 30, 64], [64, 0, 64, 0, 64], [-(1 << 31)] * 5, [0, 1 << 30, 7, 2, 3]):
        assert np.isfinite(e.run(plan=(np.array(lie, np.int32), order)).cpu().numpy()).all()


def test_grouped_no_group_has_no_work(gpu):
    e = Experts(E4, E4, 8, 32, 64, 1, seed=9)
    e.groups = 0
    D = e.run(plan=(np.zeros(1, np.int32), np.full(8, -1, np.int32)))
    assert (D.cpu().numpy() == 7.5).all()


# ---- adapters ------------------------------------------------------------------------------------


def run_adapters(kx, kw, m, n, k, rank, count, ids=None, scaled=True, in_place=False, pad=(0, 0, 0), gap=0, seed=0,
                 spoil=None, **op_args):
    rng = W.rng_for(seed, 8)
    x = dev(rng.standard_normal((m, k + pad[0])).astype(np.float32)).to(FLOATS[kx][0])
    A = dev((rng.standard_normal((count, rank + gap, k + pad[0])) / np.sqrt(max(k, 1))).astype(np.float32)).to(FLOATS[kw][0])
    B = dev(rng.standard_normal((count, n + gap, rank + pad[1])).astype(np.float32)).to(FLOATS[kw][0])
    scales = (rng.random(count) + 0.5).astype(np.float32)
    C = dev(rng.standard_normal((m, n + pad[2])).astype(np.float32))
    ids = rng.integers(-1, count + 1, m).astype(np.int32) if ids is None else np.asarray(ids, np.int32)
    if spoil:
        spoil(x, A, B, C)
    before = C.cpu().numpy().copy()
    D = C if in_place else torch.full_like(C, 3.25)
    op = c.LowRankAdapters(FLOATS[kx][1], FLOATS[kw][1], **op_args)
    check(op(op.Arguments(c.AdapterCoord(m, n, k, rank, count), c.TensorRef(x, k + pad[0]),
                          c.AdapterRef(A, k + pad[0], (rank + gap) * (k + pad[0])),
                          c.AdapterRef(B, rank + pad[1], (n + gap) * (rank + pad[1])), dev(ids), c.TensorRef(C, n + pad[2]),
                          c.TensorRef(D, n + pad[2]), dev(scales) if scaled else None)))
    torch.cuda.synchronize()
    got = D.cpu().numpy().astype(np.float64)
    want, err = H.adapters(x[:, :k].double().cpu().numpy(), A[:, :rank, :k].double().cpu().numpy(),
                           B[:, :n, :rank].double().cpu().numpy(), ids, scales if scaled else None, before[:, :n])
    return got, want, err, before


def check_adapters(*args, **kw):
    n = args[3]
    got, want, err, before = run_adapters(*args, **kw)
    assert np.isfinite(got[:, :n]).all()
    assert np.all(np.abs(got[:, :n] - want) <= err), np.max(np.abs(got[:, :n] - want) / np.maximum(err, 1e-300))
    rest = before[:, n:] if kw.get("in_place") else np.full_like(before[:, n:], 3.25)
    assert np.array_equal(got[:, n:], rest)
    moved = np.abs(want - before[:, :n])
    assert np.linalg.norm(got[:, :n] - want) <= 4e-6 * np.linalg.norm(moved) + 1e-6 * np.linalg.norm(want)


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")]
ROWS = [1, 5, 64, 300, 1111]


@pytest.mark.parametrize("kx,kw", TYPES)
@pytest.mark.parametrize("m", ROWS)
def test_adapters_types(gpu, kx, kw, m):
    check_adapters(kx, kw, m, 264, 520, 16, 5, seed=m)


@pytest.mark.parametrize("m", [1, 50, 700])
@pytest.mark.parametrize("n,k,rank,count", [(1, 1, 1, 1), (7, 9, 3, 2), (64, 64, 8, 4), (130, 100, 17, 3),
                                            (300, 2048, 64, 6), (65, 33, 256, 2), (512, 4096, 33, 40)])
def test_adapters_sizes(gpu, m, n, k, rank, count):
    check_adapters("bf16", "bf16", m, n, k, rank, count, seed=n + m)


@pytest.mark.parametrize("m", [3, 600])
@pytest.mark.parametrize("pad", [(0, 0, 0), (3, 0, 1), (8, 8, 4), (0, 5, 3), (1, 1, 0)])
def test_adapters_strides(gpu, m, pad):
    for kx, kw in TYPES:
        check_adapters(kx, kw, m, 97, 168, 24, 4, pad=pad, gap=2, scaled=False, seed=m)


@pytest.mark.parametrize("m", [4, 900])
def test_adapters_in_place(gpu, m):
    check_adapters("bf16", "bf16", m, 200, 256, 16, 3, in_place=True, seed=m)
    check_adapters("f32", "bf16", m, 199, 255, 15, 3, in_place=True, pad=(1, 0, 2), seed=m)


@pytest.mark.parametrize("m", [6, 520])
def test_adapters_rows_without(gpu, m):
    """A row without an adapter is C, bit for bit, whatever its x holds."""
    ids = np.where(np.arange(m) % 3 == 0, -1, np.arange(m) % 2)
    ids[1] = 1 << 30

    def spoil(x, A, B, C):
        x[::3] = float("nan")
        x[1] = float("inf")
        A[2] = float("nan")
        B[2] = float("nan")

    for in_place in (False, True):
        got, want, err, before = run_adapters("bf16", "bf16", m, 96, 128, 8, 3, ids=ids, in_place=in_place, spoil=spoil)
        none = (ids < 0) | (ids >= 3)
        assert np.array_equal(got[none], before[none])
        assert np.all(np.abs(got - want)[~none] <= err[~none])
    check_adapters("bf16", "bf16", m, 96, 128, 8, 3, ids=np.full(m, -1))
    check_adapters("bf16", "bf16", m, 96, 128, 8, 3, ids=np.full(m, 2), in_place=True)


@pytest.mark.parametrize("m", [2, 400])
def test_adapters_empty_products(gpu, m):
    for k, rank, count in ((0, 4, 2), (16, 0, 2)):
        got, want, err, before = run_adapters("bf16", "bf16", m, 40, k, rank, count)
        assert np.array_equal(got, before)


def test_adapters_keep_f32_accuracy(gpu):
    """The product between the two factors is not rounded to 16 bits: large and small parts of it
    cancel in the second product."""
    for m in (2, 640):
        k, rank, n = 64, 2, 32
        x = torch.ones((m, k), dtype=torch.bfloat16, device="cuda")
        A = torch.zeros((1, rank, k), dtype=torch.bfloat16, device="cuda")
        A[0, 0, 0], A[0, 0, 1], A[0, 1, 0] = 256.0, 2.0 ** -12, 256.0   # u = (256 + 2^-12, 256): 21 bits
        B = torch.zeros((1, n, rank), dtype=torch.bfloat16, device="cuda")
        B[0, :, 0], B[0, :, 1] = 1.0, -1.0
        C = torch.zeros((m, n), device="cuda")
        D = torch.empty_like(C)
        op = c.LowRankAdapters(c.bf16_t)
        check(op(op.Arguments(c.AdapterCoord(m, n, k, rank, 1), c.TensorRef(x, k), c.AdapterRef(A, k, rank * k),
                              c.AdapterRef(B, rank, n * rank), torch.zeros(m, dtype=torch.int32, device="cuda"),
                              c.TensorRef(C, n), c.TensorRef(D, n))))
        assert (D == 2.0 ** -12).all()


# Many rows go tile by tile: several launches instead of one.


def check_many_rows(*args, **kw):
    before = c.launch_count()
    check_adapters(*args, **kw)
    assert c.launch_count() - before >= 3, "these rows were to go tile by tile"


@pytest.mark.parametrize("kx,kw", TYPES)
def test_adapters_many_rows_types(gpu, kx, kw):
    check_many_rows(kx, kw, 2500, 264, 520, 16, 5, seed=1)
    check_many_rows(kx, kw, 4200, 260, 500, 15, 5, seed=2)


@pytest.mark.parametrize("m,n,k,rank,count", [(1500, 300, 2048, 64, 6), (4000, 65, 33, 256, 2), (6000, 130, 100, 17, 3),
                                              (2048, 1024, 64, 48, 1), (5000, 64, 1000, 8, 9), (3000, 128, 256, 129, 30),
                                              (4097, 500, 300, 65, 1000)])
def test_adapters_many_rows_sizes(gpu, m, n, k, rank, count):
    if count == 1000:   # (a plan of nearly as many groups as there may be; the rows all in a few of them)
        ids = W.rng_for(3, 8).integers(0, 1000, 12)[W.rng_for(4, 8).integers(0, 12, m)]
        got, want, err, _ = run_adapters("bf16", "bf16", m, n, k, rank, count, ids=ids)
        assert np.all(np.abs(got - want) <= err)
    else:
        check_many_rows("bf16", "bf16", m, n, k, rank, count, seed=n)
        check_many_rows("f32", "f16", m, n, k, rank, count, seed=k)


@pytest.mark.parametrize("pad", [(3, 0, 1), (8, 8, 4), (0, 5, 3), (1, 1, 0), (2, 2, 2)])
def test_adapters_many_rows_strides(gpu, pad):
    for kx, kw in TYPES:
        check_many_rows(kx, kw, 4000, 97, 168, 24, 4, pad=pad, gap=2, scaled=False, seed=5)
        check_many_rows(kx, kw, 4000, 96, 168, 24, 4, pad=pad, in_place=True, seed=6)


def test_adapters_many_rows_without(gpu):
    m = 4000
    ids = np.where(np.arange(m) % 3 == 0, -1, np.arange(m) % 2)
    ids[1] = 1 << 30

    def spoil(x, A, B, C):
        x[::3] = float("nan")
        x[1] = float("inf")
        A[2] = float("nan")
        B[2] = float("nan")

    for in_place in (False, True):
        before = c.launch_count()
        got, want, err, C = run_adapters("bf16", "bf16", m, 256, 256, 16, 3, ids=ids, in_place=in_place, spoil=spoil)
        assert c.launch_count() - before >= 3
        none = (ids < 0) | (ids >= 3)
        assert np.array_equal(got[none], C[none])
        assert np.all(np.abs(got - want)[~none] <= err[~none])
    check_many_rows("bf16", "bf16", m, 256, 256, 16, 3, ids=np.full(m, -1))
    check_many_rows("f16", "f16", m, 256, 256, 16, 3, ids=np.full(m, 2), in_place=True)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_adapters_many_rows_keep_f32_accuracy(gpu, kind):
    """As above: 256 + 2^-12 and 256 cancel in the second product; in f16 also beside a number near the
    top of u's range, and with all of u tiny."""
    m, k, rank, n = 4000, 256, 16, 256
    t, storage = FLOATS[kind]
    for size in (1.0, 2.0 ** -40, 2.0 ** 30):
        x = torch.full((m, k), size, dtype=torch.float32, device="cuda")
        A = torch.zeros((1, rank, k), dtype=t, device="cuda")
        A[0, 0, 0], A[0, 0, 1], A[0, 1, 0] = 256.0, 2.0 ** -12, 256.0
        B = torch.zeros((1, n, rank), dtype=t, device="cuda")
        B[0, :, 0], B[0, :, 1] = 1.0, -1.0
        C = torch.zeros((m, n), device="cuda")
        D = torch.empty_like(C)
        op = c.LowRankAdapters(c.f32_t, storage)
        before = c.launch_count()
        check(op(op.Arguments(c.AdapterCoord(m, n, k, rank, 1), c.TensorRef(x, k), c.AdapterRef(A, k, rank * k),
                              c.AdapterRef(B, rank, n * rank), torch.zeros(m, dtype=torch.int32, device="cuda"),
                              c.TensorRef(C, n), c.TensorRef(D, n))))
        assert c.launch_count() - before >= 3
        assert (D == size * 2.0 ** -12).all()


# ---- together, on streams and in graphs ------------------------------------------------------------


def layer(stream, tokens=48, experts=12, top_k=3, width=256, inner=192, rank=8):
    """Routing, the gated products, the summed products, and an adapter on the result."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    x = randn(tokens, width)
    logits = randn(tokens, experts)
    A, SA = H.quantise_e4m3(x)
    W1, S1 = H.quantise_e4m3(randn(experts * 2 * inner, width) / 16)
    W2, S2 = H.quantise_e4m3(randn(experts * width, inner) / 14)
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device="cuda")
    weights = torch.empty((tokens, top_k), device="cuda")
    plan = c.RowPlan(torch.empty(experts + 1, dtype=torch.int32, device="cuda"),
                     torch.empty(tokens * top_k, dtype=torch.int32, device="cuda"))
    pairs = tokens * top_k
    h = torch.zeros((pairs, inner), device="cuda")
    y = torch.empty((tokens, width), device="cuda")
    la, lb = (randn(2, rank, width) / 16).bfloat16(), randn(2, width, rank).bfloat16()
    lora = (torch.arange(tokens, device="cuda") % 3 - 1).int()
    xb = x.bfloat16()
    torch.cuda.synchronize()
    kw = {"stream": stream.cuda_stream, "asynchronous": True}
    route, up, down = c.RouteExperts(c.f32_t, **kw), c.GemmMxGrouped(gated=True, **kw), c.GemmMxGrouped(**kw)
    low = c.LowRankAdapters(c.bf16_t, **kw)

    def run():
        check(route(route.Arguments(c.RouteCoord(tokens, experts, top_k), c.TensorRef(logits, experts), ids, weights, plan)))
        check(up(up.Arguments(c.GroupedCoord(pairs, inner, width, experts), c.MxTensorRef(A, SA, width, width // 32),
                              c.MxTensorRef(W1, S1, width, width // 32), plan, c.TensorRef(h, inner), pairs_per_a_row=top_k)))
        with torch.cuda.stream(stream):
            hq, hs = H.quantise_e4m3(h)
        check(down(down.Arguments(c.GroupedCoord(pairs, width, inner, experts), c.MxTensorRef(hq, hs, inner, inner // 32),
                                  c.MxTensorRef(W2, S2, inner, inner // 32), plan, c.TensorRef(y, width),
                                  row_weights=weights, pairs_per_d_row=top_k, ids=ids)))
        check(low(low.Arguments(c.AdapterCoord(tokens, width, width, rank, 2), c.TensorRef(xb, width),
                                c.AdapterRef(la, width, rank * width), c.AdapterRef(lb, rank, width * rank), lora,
                                c.TensorRef(y, width), c.TensorRef(y, width))))
        return hq, hs

    hq, hs = run()
    torch.cuda.synchronize()
    n = lambda t: t.cpu().numpy()  # noqa: E731
    want_ids, want_w = H.route(n(logits), None, top_k, False, 1, 1, 1, True, 1.0)
    assert np.array_equal(n(ids), want_ids)
    eh, _ = H.grouped(H.decode_mx(n(A), n(SA), E4, width), H.decode_mx(n(W1), n(S1), E4, width).reshape(experts, -1, width),
                      want_ids, inner, True, top_k, None, 1, np.zeros((pairs, inner)))
    assert np.linalg.norm(n(h) - eh) <= 1e-5 * np.linalg.norm(eh)
    ey, _ = H.grouped(H.decode_mx(n(hq), n(hs), E4, inner), H.decode_mx(n(W2), n(S2), E4, inner).reshape(experts, -1, inner),
                      want_ids, width, False, 1, want_w, top_k, None)
    ey, _ = H.adapters(xb.double().cpu().numpy(), la.double().cpu().numpy(), lb.double().cpu().numpy(), n(lora), None, ey)
    assert np.linalg.norm(n(y) - ey) <= 1e-5 * np.linalg.norm(ey)
    return run, (logits, y)


def test_layer_of_experts(gpu):
    layer(torch.cuda.current_stream())


def test_layer_on_a_side_stream_captured_and_replayed(gpu):
    stream = torch.cuda.Stream()
    run, (logits, y) = layer(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        keep = run()
    first = y.clone()
    y.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, y)
    logits.copy_(-logits)            # other experts: the graph reads the arrays anew
    graph.replay()
    torch.cuda.synchronize()
    replayed = y.clone()
    run()
    torch.cuda.synchronize()
    assert torch.equal(replayed, y) and not torch.equal(first, y)
    del keep


def test_results_are_the_same_every_time(gpu):
    e = Experts(E4, E4, 600, 320, 512, 9, share=3, seed=11)
    first = e.run(weighted=True, summed=3).clone()
    for _ in range(5):
        assert torch.equal(first, e.run(weighted=True, summed=3))


def test_host_memory_is_refused(gpu):
    op = c.GroupRows()
    ids = np.zeros(4, np.int32)
    out = torch.zeros(4, dtype=torch.int32, device="cuda")
    st = op(op.Arguments(4, 2, ids, c.RowPlan(out, out)))
    assert st == c.Status.kErrorInvalidArguments and "device memory" in _capi.last_error()


def test_synchronous_call_under_capture_is_refused(gpu):
    """... and leaves the capture as it is."""
    stream = torch.cuda.Stream()
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    order = torch.zeros(4, dtype=torch.int32, device="cuda")
    sync = c.GroupRows(stream=stream.cuda_stream)
    queued = c.GroupRows(stream=stream.cuda_stream, asynchronous=True)
    args = sync.Arguments(4, 2, ids, c.RowPlan(offsets, order))
    check(sync(args))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert sync(args) == c.Status.kErrorInvalidArguments
        check(queued(args))
    ids.fill_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert offsets.tolist() == [0, 0, 4] and order.tolist() == [0, 1, 2, 3]


def test_calls_from_threads_on_their_own_streams(gpu):
    """Workspaces belong to streams: calls of several threads do not meet in one."""
    import threading
    jobs = []
    for t in range(4):
        e = Experts(E4, E4, 600 + 30 * t, 200 + 64 * t, 256, 3 + t, share=3, seed=20 + t)
        stream = torch.cuda.Stream()
        want = e.run(weighted=True, summed=3).clone()
        jobs.append((e, stream, want, torch.empty_like(want)))
    torch.cuda.synchronize()
    bad = []

    def work(e, stream, want, D):
        op = c.GemmMxGrouped(stream=stream.cuda_stream, asynchronous=True)
        e.args.ref_D = c.TensorRef(D, e.n)
        desc = op.describe(e.args)
        for _ in range(50):
            if op.run(desc) != OK:
                bad.append(_capi.last_error())
        if c.stream_status(stream.cuda_stream) != OK:
            bad.append("stream status")

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad
    for e, stream, want, D in jobs:
        assert torch.equal(want, D)


def test_memory_space_given(gpu):
    """With MEM_DEVICE the pointers are taken as they are."""
    ids = dev(np.array([1, 0, 1, -1], np.int32))
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    order = torch.zeros(4, dtype=torch.int32, device="cuda")
    op = c.GroupRows(memory_space=_capi.MEM_DEVICE, device=0)
    check(op(op.Arguments(4, 2, ids, c.RowPlan(offsets, order))))
    assert offsets.tolist() == [0, 1, 3] and order.tolist() == [1, 0, 2, -1]


@pytest.mark.parametrize("budget", [1000])
def test_waits_have_time_in_a_long_call(gpu, lib, budget):
    """The bounded waits of the experts' kernel are for a stage, not for the call: a budget of a
    millisecond is enough for one that takes longer."""
    e = Experts(E4, E4, 3000, 2048, 2048, 24, seed=30)
    want = e.run().clone()
    try:
        lib.cpuops_b200_set_wait_budget_us(budget)
        assert torch.equal(want, e.run())
    finally:
        lib.cpuops_b200_set_wait_budget_us(0)
