"""The 16-bit layers' operators together: a sparse layer's norm, router and shared expert, forward and backward,
each step against its formula in 64 bits on the tensors that the step before left; and the calls around them
(graphs, streams, threads, far offsets, few SMs)."""
import threading

import pytest
import torch

import cpu_ops_b200 as c
from cpu_ops_b200 import _capi
from tests import dense_helpers as H
from tests.test_dense_gpu import held, matrix, ok, ref, unguarded

pytestmark = pytest.mark.gpu
TOKENS, WIDTH, INNER, EXPERTS, TOP_K = 300, 264, 520, 24, 3
BF16, F32 = torch.bfloat16, torch.float32


class Layer:
    """y = x + W2 gelu(W1 norm(x) + b1) + b2, and a router on norm(x): parameters, buffers and calls."""

    def __init__(self, stream=None, seed=1, tokens=TOKENS):
        def w(rows, cols, seed_):
            return matrix(rows, cols, 0, "bf16", seed + seed_, cols ** -0.5)
        self.tokens = tokens
        self.x = matrix(tokens, WIDTH, 0, "f32", seed, 1.5)
        self.gamma, self.beta = (matrix(1, WIDTH, 0, "f32", seed + i)[0] for i in (20, 21))
        self.w1, self.w2, self.wr = w(INNER, WIDTH, 30), w(WIDTH, INNER, 31), w(EXPERTS, WIDTH, 32)
        self.b1, self.b2 = matrix(1, INNER, 0, "f32", seed + 33)[0], matrix(1, WIDTH, 0, "f32", seed + 34)[0]
        self.dy = matrix(tokens, WIDTH, 0, "f32", seed + 40, 0.1)     # what comes back from the layers above
        self.upstream = torch.tensor([0.5], device="cuda")

        def z(*shape, kind=F32):
            return torch.zeros(shape, dtype=kind, device="cuda")
        self.h, self.mean, self.rstd = z(tokens, WIDTH, kind=BF16), z(tokens), z(tokens)
        self.logits, self.ids, self.weights = z(tokens, EXPERTS), z(tokens, TOP_K, kind=torch.int32), z(tokens, TOP_K)
        self.counts, self.loss, self.dlogits = z(EXPERTS, kind=torch.int32), z(1), z(tokens, EXPERTS)
        self.z1, self.a1, self.y = z(tokens, INNER, kind=BF16), z(tokens, INNER, kind=BF16), z(tokens, WIDTH)
        self.dy16, self.dlogits16 = z(tokens, WIDTH, kind=BF16), z(tokens, EXPERTS, kind=BF16)
        self.db1, self.db2, self.da1, self.dz1 = z(INNER), z(WIDTH), z(tokens, INNER, kind=BF16), z(tokens, INNER, kind=BF16)
        self.dw1, self.dw2, self.dwr = z(INNER, WIDTH), z(WIDTH, INNER), z(EXPERTS, WIDTH)
        self.dh0, self.dh = z(tokens, WIDTH, kind=BF16), z(tokens, WIDTH, kind=BF16)
        self.dx, self.dgamma, self.dbeta = z(tokens, WIDTH), z(WIDTH), z(WIDTH)
        self.place = {} if stream is None else {"stream": stream, "asynchronous": True}

    def gemm(self, m, n, k, a, b, d, la=c.RowMajor, lb=c.RowMajor, epilogue=None, residual=None, z=None, storage=None):
        op = c.GemmBF16(la, lb, storage_d=storage or c.bf16_t, **self.place)
        ok(op(op.Arguments(c.GemmCoord(m, n, k), ref(a), ref(b), ref(residual), ref(d), epilogue or c.BiasActivation(), ref(z))))

    def forward(self):
        t, place = self.tokens, self.place
        norm = c.LayerNorm(c.f32_t, c.bf16_t, **place)
        ok(norm(norm.Arguments(c.RowsCoord(t, WIDTH), ref(self.x), self.gamma, self.beta, ref(self.h), self.mean, self.rstd, 1e-5)))
        self.gemm(t, EXPERTS, WIDTH, self.h, self.wr, self.logits, lb=c.ColumnMajor, storage=c.f32_t)
        route = c.RouteExperts(c.f32_t, **place)
        ok(route(route.Arguments(c.RouteCoord(t, EXPERTS, TOP_K), ref(self.logits), self.ids, self.weights)))
        balance = c.BalanceLoss(c.f32_t, **place)
        ok(balance(balance.Arguments(c.RouteCoord(t, EXPERTS, TOP_K), ref(self.logits), self.ids, self.counts, self.loss,
                                     ref(self.dlogits), c.Scoring.kSoftmax, 0.01, self.upstream)))
        self.gemm(t, INNER, WIDTH, self.h, self.w1, self.a1, lb=c.ColumnMajor, epilogue=c.BiasActivation(self.b1, c.Gelu()), z=self.z1)
        self.gemm(t, WIDTH, INNER, self.a1, self.w2, self.y, lb=c.ColumnMajor, epilogue=c.BiasActivation(self.b2, beta=1.0),
                  residual=self.x, storage=c.f32_t)

    def backward(self):
        t, place = self.tokens, self.place
        self.dy16.copy_(self.dy)
        self.dlogits16.copy_(self.dlogits)
        grad = c.BiasActivationGrad(c.bf16_t, **place)
        ok(grad(grad.Arguments(c.RowsCoord(t, WIDTH), ref(self.dy16), dbias=self.db2)))
        self.gemm(t, INNER, WIDTH, self.dy16, self.w2, self.da1)
        self.gemm(WIDTH, INNER, t, self.dy16, self.a1, self.dw2, la=c.ColumnMajor, storage=c.f32_t)
        grad = c.BiasActivationGrad(c.bf16_t, c.Gelu(), **place)
        ok(grad(grad.Arguments(c.RowsCoord(t, INNER), ref(self.da1), ref(self.z1), ref(self.dz1), self.db1)))
        self.gemm(INNER, WIDTH, t, self.dz1, self.h, self.dw1, la=c.ColumnMajor, storage=c.f32_t)
        self.gemm(EXPERTS, WIDTH, t, self.dlogits16, self.h, self.dwr, la=c.ColumnMajor, storage=c.f32_t)
        self.gemm(t, WIDTH, EXPERTS, self.dlogits16, self.wr, self.dh0)
        self.gemm(t, WIDTH, INNER, self.dz1, self.w1, self.dh, epilogue=c.BiasActivation(beta=1.0), residual=self.dh0)
        norm = c.LayerNormGrad(c.f32_t, c.bf16_t, **place)
        ok(norm(norm.Arguments(c.RowsCoord(t, WIDTH), ref(self.dh), ref(self.x), self.gamma, self.mean, self.rstd, ref(self.dx),
                               self.dgamma, self.dbeta, ref_dR=ref(self.dy))))

    def results(self):
        return {k: v for k, v in vars(self).items() if isinstance(v, torch.Tensor)}


def d(x):
    return x.double().cpu()


def check(layer):
    """Every step against its formula, on what the step before stored."""
    s = layer
    h, mean, rstd = H.layer_norm(d(s.x), d(s.gamma), d(s.beta), 1e-5, "bf16")
    steps = [(s.h, h), (s.mean, mean), (s.rstd, rstd)]
    steps.append((s.logits, H.product(d(s.h), d(s.wr).t(), None, "none", None, 1.0, 0.0, "f32")[0]))
    counts, loss, dlogits = H.balance(d(s.logits), s.ids.cpu(), False, float(torch.tensor(0.01)), 0.5, "f32")
    assert torch.equal(counts.int(), s.counts.cpu())
    steps += [(s.loss, (loss[0].reshape(1), loss[1].reshape(1))), (s.dlogits, (dlogits[0], dlogits[1] + 1e-37))]
    a1, z1 = H.product(d(s.h), d(s.w1).t(), d(s.b1), "gelu", None, 1.0, 0.0, "bf16")
    steps += [(s.a1, a1), (s.z1, z1), (s.y, H.product(d(s.a1), d(s.w2).t(), d(s.b2), "none", d(s.x), 1.0, 1.0, "f32")[0])]
    steps.append((s.db2, H.epilogue_grad(d(s.dy16), None, "none", "bf16")[1]))
    steps.append((s.da1, H.product(d(s.dy16), d(s.w2), None, "none", None, 1.0, 0.0, "bf16")[0]))
    steps.append((s.dw2, H.product(d(s.dy16).t(), d(s.a1), None, "none", None, 1.0, 0.0, "f32")[0]))
    dz1, db1 = H.epilogue_grad(d(s.da1), d(s.z1), "gelu", "bf16")
    steps += [(s.dz1, dz1), (s.db1, db1)]
    steps.append((s.dw1, H.product(d(s.dz1).t(), d(s.h), None, "none", None, 1.0, 0.0, "f32")[0]))
    steps.append((s.dwr, H.product(d(s.dlogits16).t(), d(s.h), None, "none", None, 1.0, 0.0, "f32")[0]))
    steps.append((s.dh0, H.product(d(s.dlogits16), d(s.wr), None, "none", None, 1.0, 0.0, "bf16")[0]))
    steps.append((s.dh, H.product(d(s.dz1), d(s.w1), None, "none", d(s.dh0), 1.0, 1.0, "bf16")[0]))
    steps += list(zip((s.dx, s.dgamma, s.dbeta),
                      H.layer_norm_grad(d(s.dh), d(s.x), d(s.gamma), d(s.mean), d(s.rstd), d(s.dy), "f32")))
    for i, (got, want) in enumerate(steps):
        assert H.worst(got, want) <= 1, i


def test_a_sparse_layers_step(gpu):
    layer = Layer()
    layer.forward()
    layer.backward()
    torch.cuda.synchronize()
    check(layer)


def test_the_step_captured_and_replayed(gpu):
    """Eager calls on a stream, then the same step as a graph on other inputs: the bits of an eager step on them."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer = Layer(stream.cuda_stream)
        layer.forward()
        layer.backward()
    stream.synchronize()
    first = {k: v.clone() for k, v in layer.results().items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        layer.forward()
        layer.backward()
    other = Layer(seed=50)
    layer.x.copy_(other.x)
    layer.dy.copy_(other.dy)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    check(layer)
    replayed = {k: v.clone() for k, v in layer.results().items()}
    with torch.cuda.stream(stream):
        layer.forward()
        layer.backward()
    stream.synchronize()
    for name, value in layer.results().items():
        assert torch.equal(value, replayed[name]), name
    assert not torch.equal(first["dx"], replayed["dx"])


def test_a_first_call_under_capture_is_refused_or_needs_nothing(gpu):
    """A capture that would have to allocate is told so, and stays intact; calls without a workspace are captured."""
    stream = torch.cuda.Stream()
    dy, dbias = matrix(5000, 512, 0, "bf16", 1), torch.zeros((512,), device="cuda")
    x, y = matrix(20, 512, 0, "bf16", 2), torch.zeros((20, 512), dtype=BF16, device="cuda")
    place = {"stream": stream.cuda_stream, "asynchronous": True}
    warm = c.LayerNorm(c.bf16_t)
    ok(warm(warm.Arguments(c.RowsCoord(20, 512), ref(x), ref_Y=ref(y))))
    y.zero_()
    torch.cuda.synchronize()
    grad, norm = c.BiasActivationGrad(c.bf16_t, **place), c.LayerNorm(c.bf16_t, **place)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert grad(grad.Arguments(c.RowsCoord(5000, 512), ref(dy), dbias=dbias)) == c.Status.kErrorInvalidArguments
        assert "capture" in _capi.last_error()
        ok(norm(norm.Arguments(c.RowsCoord(20, 512), ref(x), ref_Y=ref(y))))
        sync = c.LayerNorm(c.bf16_t, stream=stream.cuda_stream)
        assert sync(sync.Arguments(c.RowsCoord(20, 512), ref(x), ref_Y=ref(y))) == c.Status.kErrorInvalidArguments
    graph.replay()
    torch.cuda.synchronize()
    assert H.worst(y, H.layer_norm(d(x), None, None, 1e-5, "bf16")[0]) <= 1


def test_steps_on_two_streams_and_threads(gpu):
    """Steps that run side by side give each its own result."""
    layers, errors = [], []
    for i in range(2):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            layers.append((stream, Layer(stream.cuda_stream, seed=10 + i, tokens=TOKENS + 97 * i)))
        stream.synchronize()

    def work(stream, layer):
        try:
            with torch.cuda.stream(stream):
                for _ in range(5):
                    layer.forward()
                    layer.backward()
        except BaseException as e:  # noqa: B902 (shown by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=pair) for pair in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for stream, layer in layers:
        check(layer)
        assert c.stream_status(stream.cuda_stream) == c.Status.kSuccess


def test_few_sms(gpu, lib):
    """A limit on the SMs changes parts and grids, not what is computed."""
    layer = Layer()
    try:
        for sms in (3, 40):
            assert lib.cpuops_b200_set_sm_limit(-1, sms) == 0
            layer.forward()
            layer.backward()
            torch.cuda.synchronize()
            check(layer)
            for m, n in ((3, 9000), (100, 300), (500, 900)):
                a, w, out = matrix(m, 512, 0, "bf16", 1), matrix(n, 512, 0, "bf16", 2, 0.05), held(m, n, 0, "bf16")
                layer.gemm(m, n, 512, a, w, out, lb=c.ColumnMajor)
                assert _capi.last_plan().grid <= sms
                assert H.worst(out[:m], H.product(d(a), d(w).t(), None, "none", None, 1.0, 0.0, "bf16")[0]) <= 1
    finally:
        lib.cpuops_b200_set_sm_limit(-1, 0)


def test_far_rows(gpu):
    """Rows whose offsets pass 2^31 elements."""
    m, n, ld = 700, 72, 4_000_000
    base = torch.zeros((m * ld,), dtype=BF16, device="cuda")
    x = base.view(m, ld)
    x[:, :n] = matrix(m, n, 0, "bf16", 1)
    x[:, n] = 77.0
    x64 = d(x[:, :n])
    far = c.TensorRef(x, ld)
    y = held(m, n, 0, "bf16")
    norm = c.LayerNorm(c.bf16_t)
    ok(norm(norm.Arguments(c.RowsCoord(m, n), far, ref_Y=ref(y))))
    assert H.worst(y[:m], H.layer_norm(x64, None, None, 1e-5, "bf16")[0]) <= 1 and unguarded(y, m, n)
    dbias = torch.zeros((n,), device="cuda")
    grad = c.BiasActivationGrad(c.bf16_t, c.Silu())
    ok(grad(grad.Arguments(c.RowsCoord(m, n), far, far, ref(y), dbias)))
    want, sums = H.epilogue_grad(x64, x64, "silu", "bf16")
    assert H.worst(y[:m], want) <= 1 and H.worst(dbias, sums) <= 1
    w = matrix(40, n, 0, "bf16", 2, 0.2)
    out = held(m, 40, 0, "f32")
    gemm = c.GemmBF16(c.RowMajor, c.ColumnMajor, storage_d=c.f32_t)
    ok(gemm(gemm.Arguments(c.GemmCoord(m, 40, n), far, ref(w), c.TensorRef(), ref(out))))
    assert H.worst(out[:m], H.product(x64, d(w).t(), None, "none", None, 1.0, 0.0, "f32")[0]) <= 1
    # ... written there: a residual and its sum, in place
    gemm = c.GemmBF16(c.RowMajor, c.ColumnMajor)
    a = matrix(m, 32, 0, "bf16", 3)
    w = matrix(n, 32, 0, "bf16", 4, 0.2)
    ok(gemm(gemm.Arguments(c.GemmCoord(m, n, 32), ref(a), ref(w), far, far, c.BiasActivation(beta=1.0))))
    assert H.worst(x[:, :n], H.product(d(a), d(w).t(), None, "none", x64, 1.0, 1.0, "bf16")[0]) <= 1
    assert bool((x[:, n] == 77.0).all()) and bool((x[:, n + 1] == 0).all())


def test_host_and_foreign_pointers_are_refused(gpu):
    x = torch.zeros((4, 8), dtype=BF16)
    y = torch.zeros((4, 8), dtype=BF16, device="cuda")
    norm = c.LayerNorm(c.bf16_t)
    assert norm(norm.Arguments(c.RowsCoord(4, 8), ref(x), ref_Y=ref(y))) == c.Status.kErrorInvalidArguments
    assert "not memory of device" in _capi.last_error()
    gemm = c.GemmBF16(c.RowMajor, c.ColumnMajor)
    assert gemm(gemm.Arguments(c.GemmCoord(4, 4, 8), ref(y), ref(x), c.TensorRef(), c.TensorRef(y, 8))) == c.Status.kErrorInvalidArguments


def test_a_shorter_wait_budget_changes_nothing(gpu, lib):
    """The waits' budget bounds a wait, not a call's work."""
    try:
        assert lib.cpuops_b200_set_wait_budget_us(200000) == 0
        layer = Layer()
        layer.forward()
        layer.backward()
        torch.cuda.synchronize()
        check(layer)
    finally:
        lib.cpuops_b200_set_wait_budget_us(0)
