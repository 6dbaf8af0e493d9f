"""Calls of the operators whose weights are chosen per row in which a bound, a mask, an infinity or
the sharing of a stream decides the result."""
import math

import numpy as np
import pytest
import torch

import cpu_ops_b200 as c
from cpu_ops_b200 import workloads as W
from tests import row_chosen_helpers as H
from tests.test_row_chosen_gpu import E4, Experts, check, check_route, dev

pytestmark = pytest.mark.gpu


def run_with_ids(e, weighted, D, ldd):
    """The call of `e` once more, its ids given beside one pair per row of D."""
    e.run(weighted, D=D, ldd=ldd)
    D.fill_(float("nan"))
    e.args.ids = e.keep[-1]
    check(c.GemmMxGrouped()(e.args))
    return D.cpu().numpy()


# ---- routing: choices that f32 scores leave open ----------------------------------------------


def test_route_softmax_sum_that_loses_its_small_terms(gpu):
    """1024 experts: 36 scores of 5.9e-8 are each less than half a step of a running f32 sum of 1, so that
    the sum stays 1 and the first score is 2.1e-6 too large, more than the second choice is behind."""
    x = np.full((2, 1024), -200, np.float32)
    bias = np.full(1024, -1, np.float32)
    x[:, 0] = 0
    x[0, list(range(32, 1024, 32)) + [1, 2, 4, 8, 16]] = np.float32(math.log(5.9e-8))
    # the same with a score near half a step in every place of the first lane, others small
    x[1, 1:] = -20 + 4 * W.rng_for(1024, 9).random(1023).astype(np.float32)
    x[1, list(range(32, 1024, 32))] = np.float32(math.log(5.9e-8))
    bias[37] = np.float32(-2.08e-6)
    check_route(dev(x), "f32", 1, bias=bias)
    check_route(dev(x), "f32", 2, bias=bias, n_groups=16, top_groups=2)


def test_route_groups_whose_two_best_cancel(gpu):
    """A group's two best choices are +100 and -100 and a little: each is rounded to 8e-6 in f32, their sum is
    below one."""
    rng = W.rng_for(2000, 9)
    x = rng.standard_normal((2000, 8)).astype(np.float32)
    x[:, 4:] = x[:, :4]
    x[:, 4:6] += (4e-5 * (2 * rng.random((2000, 2)) - 1)).astype(np.float32)
    bias = np.array([100, -100, -np.inf, -np.inf] * 2, np.float32)
    for sigmoid in (False, True):
        check_route(dev(x), "f32", 1, bias=bias, sigmoid=sigmoid, n_groups=2, top_groups=1, group_best=2)


# ---- the experts' products ---------------------------------------------------------------------


@pytest.mark.parametrize("rows,n,k,groups", [(5, 96, 128, 3), (64, 1003, 96, 4), (600, 1000, 320, 2), (9, 40, 64, 0)])
@pytest.mark.parametrize("weighted", [False, True])
def test_grouped_one_pair_per_row_with_ids_writes_every_row(gpu, rows, n, k, groups, weighted):
    """With ids, rows of D without a group are zeros for one pair per row as for several."""
    rng = W.rng_for(rows, 9)
    ids = rng.integers(-1, max(groups, 1) + 1, rows)
    ids[-3:] = -1
    e = Experts(E4, E4, rows, n, k, max(groups, 1), ids=ids, seed=rows)
    if groups == 0:
        e.groups, e.ids = 0, np.full(rows, -1, np.int32)
    for ldd in (n, n + 3):
        D = torch.full((rows, ldd), float("nan"), device="cuda")
        got = run_with_ids(e, weighted, D, ldd)
        if groups == 0:
            want, err = np.zeros((rows, n)), np.zeros((rows, n))
        else:
            A, B = e.dense()
            want, err = H.grouped(A, B, e.ids, n, False, 1, e.weights if weighted else None, 1, np.zeros((rows, n)))
        assert np.all(np.abs(got[:, :n] - want) <= err)
        none = (e.ids < 0) | (e.ids >= groups)
        assert none.any() and not got[none, :n].view(np.int32).any()     # (+0, bit for bit)
        assert np.isnan(got[:, n:]).all()
    # without ids they are left as they were
    D = torch.full((rows, n), 7.5, device="cuda")
    assert (e.run(weighted, D=D).cpu().numpy()[none] == 7.5).all()
