"""Calls of the operators whose weights are chosen per row in which a bound, a mask, an infinity or
the sharing of a stream decides the result."""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import cpu_ops_b200 as c
from cpu_ops_b200 import _capi, workloads as W
from tests import row_chosen_helpers as H
from tests.gpu_helpers import MX_TOL, gather, normwise, run_mx_gpu
from tests.test_row_chosen_gpu import E4, Experts, check, check_route, dev, run_adapters

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


def test_waits_are_for_a_stage_not_for_the_call(gpu, lib):
    """A budget for the bounded waits of 400 us is enough for a call that takes several times as long."""
    budget = 400
    e = Experts(E4, E4, 131072, 4096, 4096, 8, share=512, seed=31)
    want = e.run()
    D = torch.full_like(want, float("nan"))
    e.args.ref_D = c.TensorRef(D, e.n)
    op = c.GemmMxGrouped(stream=torch.cuda.current_stream().cuda_stream, asynchronous=True)
    desc = op.describe(e.args)
    check(op.run(desc))   # (this stream's workspace is in place)
    D.fill_(float("nan"))
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    try:
        lib.cpuops_b200_set_wait_budget_us(budget)
        start.record()
        check(op.run(desc))
        end.record()
        check(c.stream_status(torch.cuda.current_stream().cuda_stream))
    finally:
        lib.cpuops_b200_set_wait_budget_us(0)
    assert start.elapsed_time(end) * 1000 > 3 * budget
    assert torch.equal(want, D)


def test_a_call_after_one_without_memory(gpu):
    """A workspace that does not fit the device fails its call, and only that one."""
    rows, n, k = 1 << 16, 1 << 20, 32          # the pairs' rows: 275 GB
    A = torch.zeros((1, k), dtype=torch.uint8, device="cuda")
    B = torch.zeros((n, k), dtype=torch.uint8, device="cuda")
    ones = torch.full((n, 1), 127, dtype=torch.uint8, device="cuda")
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    order = torch.arange(rows, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    D = torch.full((rows // 32, n), 7.5, device="cuda")
    op = c.GemmMxGrouped()
    st = op(op.Arguments(c.GroupedCoord(rows, n, k, 1), c.MxTensorRef(A, ones, k, 1), c.MxTensorRef(B, ones, k, 1),
                         c.RowPlan(offsets, order), c.TensorRef(D, n), pairs_per_a_row=rows, pairs_per_d_row=32, ids=ids))
    assert st not in (c.Status.kSuccess, c.Status.kErrorInvalidArguments) and "memory" in _capi.last_error()
    assert (D == 7.5).all()
    del D
    Experts(E4, E4, 40, 96, 128, 5, seed=32).check(summed=2)


def test_a_call_after_an_error_of_the_program(gpu):
    """An error that the program's own runtime call left behind is not this call's."""
    e = Experts(E4, E4, 40, 96, 128, 5, seed=33)
    e.check(summed=2)
    runtime = ctypes.CDLL("libcudart.so.12")
    pointer = ctypes.c_void_p()
    assert runtime.cudaMalloc(ctypes.byref(pointer), ctypes.c_size_t(1 << 50)) != 0
    try:
        status = c.GemmMxGrouped(memory_space=_capi.MEM_DEVICE)(e.args)
    finally:
        runtime.cudaGetLastError()
    check(status)


# ---- adapters: infinities ----------------------------------------------------------------------


@pytest.mark.parametrize("kx,kw", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("m", [6, 4000])
@pytest.mark.parametrize("where", ["x", "a", "b"])
def test_adapters_infinities(gpu, kx, kw, m, where):
    """An infinity reaches what it is multiplied with as the formula says, in few rows as in many (whose factors are
    multiplied in parts, one of which may be zero or of the other sign)."""

    def spoil(x, A, B, C):
        if kx == "f32":
            x *= 1e6            # u beyond f16's range
            x[:, ::2] = x[:, ::2].bfloat16().float()      # (whose second part is zero)
        if where == "x":
            x[2::5, 3] = float("inf")
            x[1, 7] = -float("inf")
        elif where == "a":
            A[1, 2, 5] = float("inf")
            A[0, 0, 100] = -float("inf")
        else:
            B[1, 9, 3] = float("inf")
            B[0, 130, 0] = -float("inf")
            B[2, 64:, 7] = float("inf")

    ids = np.arange(m) % 4 - 1
    before = c.launch_count()
    with np.errstate(invalid="ignore"):
        got, want, err, _ = run_adapters(kx, kw, m, 200, 160, 16, 3, ids=ids, spoil=spoil, seed=m)
    assert (c.launch_count() - before >= 3) == (m > 100)
    assert not np.isfinite(want).all()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    finite = np.isfinite(want)
    assert np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)])
    assert np.all(np.abs(got[finite] - want[finite]) <= err[finite])


# ---- workspaces belong to streams, whatever their handles say ------------------------------------


PER_THREAD = 2   # cudaStreamPerThread


def many_async(jobs, turns, results):
    """Runs every job's call `turns` times, asynchronously, and its stream's status at the end."""
    for e, stream, D, op in jobs:
        e.args.ref_D = c.TensorRef(D, e.n)
        desc = op.describe(e.args)
        for _ in range(turns):
            if op.run(desc) != c.Status.kSuccess:
                results.append(_capi.last_error())
        if c.stream_status(stream) != c.Status.kSuccess:
            results.append("stream status")


def expert_job(t, stream):
    e = Experts(E4, E4, 600 + 30 * t, 200 + 64 * t, 256, 3 + t, share=3, seed=20 + t)
    want = e.run(weighted=True, summed=3).clone()
    return e, stream, torch.empty_like(want), c.GemmMxGrouped(stream=stream, asynchronous=True), want


def test_the_per_thread_stream_is_another_in_every_thread(gpu):
    """Threads that all pass cudaStreamPerThread run side by side, each in a workspace of its own."""
    jobs = [expert_job(t, PER_THREAD) for t in range(4)]
    torch.cuda.synchronize()
    for generation in range(3):    # (workspaces of threads that have ended are taken over)
        for job in jobs:
            job[2].fill_(float("nan"))
        torch.cuda.synchronize()
        bad = []
        threads = [threading.Thread(target=many_async, args=([job[:4]], 50, bad)) for job in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not bad
        for job in jobs:
            assert torch.equal(job[2], job[4])


def test_a_gemm_on_the_per_thread_stream(gpu):
    """The GEMMs' workspaces are found the same way."""
    P = W.mx_problem(_capi.FMT_E4M3, 512, 384, 4096, True, seed=3)
    status, want = run_mx_gpu(P, 1.0, 0.5)
    assert status == c.Status.kSuccess
    found = [None] * 4

    def work(i):
        op = c.GemmMxE4M3(stream=PER_THREAD, asynchronous=True)
        A, B, SA, SB, C = (dev(x) for x in (P.A, P.B, P.SA, P.SB, P.C))
        D = torch.empty_like(C)
        torch.cuda.synchronize()
        desc = op.describe(op.Arguments(c.GemmCoord(P.m, P.n, P.k), c.MxTensorRef(A, SA, P.lda, P.ldsa),
                                        c.MxTensorRef(B, SB, P.ldb, P.ldsb), c.TensorRef(C, P.ldc), c.TensorRef(D, P.ldc),
                                        c.LinearCombination(1.0, 0.5)))
        ok = all(op.run(desc) == c.Status.kSuccess for _ in range(40)) and c.stream_status(PER_THREAD) == c.Status.kSuccess
        found[i] = (ok, D.cpu().numpy())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for ok, D in found:
        assert ok and normwise(*(gather(x, P.m, P.n, P.ldc, P.c_row_major) for x in (D, want))) <= MX_TOL


def test_a_stream_with_a_destroyed_streams_handle(gpu):
    """Work of a destroyed stream may still run when a new stream has its handle."""
    runtime = pytest.importorskip("cuda.bindings.runtime")
    jobs = [expert_job(t, None) for t in range(2)]
    torch.cuda.synchronize()
    for turn in range(6):
        for e, _, D, _, _ in jobs:
            D.fill_(float("nan"))
        torch.cuda.synchronize()
        bad = []
        for e, _, D, _, _ in jobs:
            status, stream = runtime.cudaStreamCreateWithFlags(runtime.cudaStreamNonBlocking)
            assert int(status) == 0
            op = c.GemmMxGrouped(stream=int(stream), asynchronous=True)
            e.args.ref_D = c.TensorRef(D, e.n)
            desc = op.describe(e.args)
            bad += [_capi.last_error() for _ in range(30) if op.run(desc) != c.Status.kSuccess]
            assert int(runtime.cudaStreamDestroy(stream)[0]) == 0
        torch.cuda.synchronize()
        assert not bad
        for job in jobs:
            assert torch.equal(job[2], job[4])


def test_capture_on_the_per_thread_stream(gpu):
    """A captured call keeps its workspace for the graph, and one that has none is refused."""
    runtime = pytest.importorskip("cuda.bindings.runtime")
    e, stream, D, op, want = expert_job(1, PER_THREAD)
    e.args.ref_D = c.TensorRef(D, e.n)
    desc = op.describe(e.args)
    torch.cuda.synchronize()
    seen = {}

    def capture(warm):
        handle = runtime.cudaStream_t(PER_THREAD)
        if warm:
            seen["warm"] = op.run(desc)
        mode = runtime.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal
        seen["begin"] = int(runtime.cudaStreamBeginCapture(handle, mode)[0])
        seen["call"] = op.run(desc)
        status, seen["graph"] = runtime.cudaStreamEndCapture(handle)
        seen["end"] = int(status)

    for warm in (False, True):
        t = threading.Thread(target=capture, args=(warm,))
        t.start()
        t.join()
        assert seen["begin"] == 0 and seen["end"] == 0
        if not warm:
            assert seen["call"] == c.Status.kErrorInvalidArguments
    assert seen["warm"] == seen["call"] == c.Status.kSuccess
    status, graph = runtime.cudaGraphInstantiate(seen["graph"], 0)
    assert int(status) == 0
    # the capturing thread has ended: another one must not take the graph's workspace over
    other = expert_job(2, PER_THREAD)
    bad = []
    D.fill_(float("nan"))
    other[2].fill_(float("nan"))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    t = threading.Thread(target=many_async, args=([other[:4]], 100, bad))
    t.start()
    for _ in range(100):
        assert int(runtime.cudaGraphLaunch(graph, runtime.cudaStream_t(side.cuda_stream))[0]) == 0
    t.join()
    torch.cuda.synchronize()
    assert not bad and torch.equal(D, want) and torch.equal(other[2], other[4])
