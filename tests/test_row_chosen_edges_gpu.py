"""Calls of the operators whose weights are chosen per row in which a bound, a mask, an infinity or
the sharing of a stream decides the result."""
import math

import numpy as np
import pytest

from cpu_ops_b200 import workloads as W
from tests.test_row_chosen_gpu import check_route, dev

pytestmark = pytest.mark.gpu


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
