"""The bounded waits of a call begin when the call before it on the stream has ended, not when its kernel is resident:
kernels of this library start beside the one before, as far as there is room on the SMs, and wait for its end."""
import pytest
import torch

import cpu_ops_b200 as c
from cpu_ops_b200 import _capi

pytestmark = pytest.mark.gpu
S = c.Status
BUDGET_US = 1000


class Long:
    """A call of this library that takes several milliseconds and leaves nearly all SMs free: two very long rows."""

    def __init__(self, place):
        n = 1 << 25
        self.x, self.y = torch.ones((2, n), device="cuda"), torch.full((2, n), 7.0, device="cuda")
        self.op = c.LayerNorm(c.f32_t, **place)
        self.desc = self.op.describe(self.op.Arguments(c.RowsCoord(2, n), c.TensorRef(self.x, n), ref_Y=c.TensorRef(self.y, n)))

    def __call__(self):
        assert self.op.run(self.desc) == S.kSuccess, _capi.last_error()


def behind_a_long_call(lib, make):
    """make(place) -> (operator, descriptor, output, the value of its every element)."""
    stream = torch.cuda.Stream()
    place = {"stream": stream.cuda_stream, "asynchronous": True}
    with torch.cuda.stream(stream):
        long = Long(place)
        op, desc, D, want = make(place)
        assert op.run(desc) == S.kSuccess, _capi.last_error()   # (this stream's workspace is in place)
        long()
        D.fill_(0)
        stream.synchronize()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        try:
            assert lib.cpuops_b200_set_wait_budget_us(BUDGET_US) == 0
            start.record()
            long()
            assert op.run(desc) == S.kSuccess, _capi.last_error()
            end.record()
            assert c.stream_status(stream.cuda_stream) == S.kSuccess, _capi.last_error()
        finally:
            lib.cpuops_b200_set_wait_budget_us(0)
    assert start.elapsed_time(end) * 1000 > 3 * BUDGET_US
    assert bool((D == want).all()) and bool((long.y == 0).all())


@pytest.mark.parametrize("d", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k,slices,pair", [(300, 256, 1024, 1, False), (300, 256, 1024, 1, True), (8, 512, 2048, 4, False)])
def test_a_16_bit_product(gpu, lib, m, n, k, slices, pair, d):
    kind = {"bf16": (c.bf16_t, torch.bfloat16), "f32": (c.f32_t, torch.float32)}[d]

    def make(place):
        a, b = (torch.ones(s, dtype=torch.bfloat16, device="cuda") for s in ((m, k), (n, k)))
        D = torch.zeros((m, n), dtype=kind[1], device="cuda")
        op = c.GemmBF16(c.RowMajor, c.ColumnMajor, storage_d=kind[0], pair=pair, **place)
        desc = op.describe(op.Arguments(c.GemmCoord(m, n, k), c.TensorRef(a, k), c.TensorRef(b, k), c.TensorRef(), c.TensorRef(D, n),
                                        split_k_slices=slices))
        op.held = (a, b)
        return op, desc, D, float(k)
    behind_a_long_call(lib, make)


@pytest.mark.parametrize("m,n,k,pair", [(300, 256, 1024, False), (300, 256, 1024, True)])
def test_an_int8_product(gpu, lib, m, n, k, pair):
    def make(place):
        a, b = torch.ones((m, k), dtype=torch.uint8, device="cuda"), torch.ones((k, n), dtype=torch.int8, device="cuda")
        D = torch.zeros((m, n), dtype=torch.int32, device="cuda")
        op = c.GemmU8S8S32(c.RowMajor, c.RowMajor, c.RowMajor, pair=pair, **place)
        desc = op.describe(op.Arguments(c.GemmCoord(m, n, k), c.TensorRef(a, k), c.TensorRef(b, n), c.TensorRef(D, n), c.TensorRef(D, n),
                                        c.LinearCombination(1, 0)))
        op.held = (a, b)
        return op, desc, D, k
    behind_a_long_call(lib, make)


@pytest.mark.parametrize("m,n,k,pair", [(300, 256, 1024, False), (300, 256, 1024, True), (8, 512, 2048, None)])
def test_an_mx_product(gpu, lib, m, n, k, pair):
    def make(place):
        a, b = (torch.full(s, 0x38, dtype=torch.uint8, device="cuda") for s in ((m, k), (n, k)))   # e4m3's 1
        sa, sb = (torch.full((rows, k // 32), 127, dtype=torch.uint8, device="cuda") for rows in (m, n))
        D = torch.zeros((m, n), device="cuda")
        op = c.GemmMxE4M3(c.RowMajor, pair=pair, **place)
        desc = op.describe(op.Arguments(c.GemmCoord(m, n, k), c.MxTensorRef(a, sa, k, k // 32), c.MxTensorRef(b, sb, k, k // 32),
                                        c.TensorRef(D, n), c.TensorRef(D, n), c.LinearCombination(1.0, 0.0)))
        op.held = (a, b, sa, sb)
        return op, desc, D, float(k)
    behind_a_long_call(lib, make)
