"""What the operators whose weights are chosen per row refuse, before they touch a device."""
import ctypes as C

import numpy as np
import pytest

import cpu_ops_b200 as c
from cpu_ops_b200 import _capi

S = c.Status
BUF = np.zeros(1 << 16, np.uint8)
BASE = (BUF.ctypes.data + 255) // 256 * 256


def route(**kw):
    d = _capi.RouteDesc(struct_size=C.sizeof(_capi.RouteDesc), tokens=4, experts=8, top_k=2, scoring=0, n_groups=1,
                        top_groups=1, group_best=1, logits_type=0, ld_logits=8, logits=BASE, ids=BASE, weights=BASE,
                        offsets=BASE, order=BASE, device=-1)
    for k, v in kw.items():
        setattr(d, k, v)
    return S(_capi.load().cpuops_b200_route(C.byref(d)))


def grouped(**kw):
    d = _capi.GemmGroupedDesc(struct_size=C.sizeof(_capi.GemmGroupedDesc), a_format=_capi.FMT_E4M3, b_format=_capi.FMT_E4M3,
                              rows=8, n=16, k=64, groups=4, a_rows=8, pairs_per_a_row=1, pairs_per_d_row=1, b_group_rows=16,
                              lda=64, ldb=64, ld_scales_a=2, ld_scales_b=2, ldd=16, device=-1)
    for name in ("a", "b", "a_scales", "b_scales", "offsets", "order", "ids", "d"):
        setattr(d, name, BASE)
    for k, v in kw.items():
        setattr(d, k, v)
    return S(_capi.load().cpuops_b200_gemm_grouped(C.byref(d)))


def adapters(**kw):
    d = _capi.AdaptersDesc(struct_size=C.sizeof(_capi.AdaptersDesc), m=4, n=16, k=32, rank=8, adapters=2, x_type=2, w_type=2,
                           ldx=32, lda=32, ldb=8, ldc=16, ldd=16, a_stride=256, b_stride=128, x=BASE, a=BASE, b=BASE, ids=BASE,
                           c=BASE, d=BASE + 4096, device=-1)
    for k, v in kw.items():
        setattr(d, k, v)
    return S(_capi.load().cpuops_b200_adapters(C.byref(d)))


def group_rows(**kw):
    d = _capi.GroupRowsDesc(struct_size=C.sizeof(_capi.GroupRowsDesc), rows=4, groups=2, ids=BASE, offsets=BASE, order=BASE,
                            device=-1)
    for k, v in kw.items():
        setattr(d, k, v)
    return S(_capi.load().cpuops_b200_group_rows(C.byref(d)))


@pytest.mark.parametrize("call", [route, grouped, adapters, group_rows])
def test_descriptor_size_is_checked(lib, call):
    assert call(struct_size=8) == S.kErrorBadDescriptor


@pytest.mark.parametrize("change,status", [
    (dict(scoring=2), S.kErrorBadDescriptor), (dict(logits_type=3), S.kErrorBadDescriptor),
    (dict(tokens=-1), S.kErrorInvalidProblem), (dict(experts=0), S.kErrorInvalidProblem),
    (dict(top_k=0), S.kErrorInvalidProblem), (dict(top_k=9), S.kErrorInvalidArguments),
    (dict(n_groups=3), S.kErrorInvalidArguments), (dict(n_groups=0), S.kErrorInvalidArguments),
    (dict(n_groups=2, top_groups=3), S.kErrorInvalidArguments), (dict(top_groups=0), S.kErrorInvalidArguments),
    (dict(group_best=3), S.kErrorInvalidArguments), (dict(experts=1025, ld_logits=1025), S.kErrorUnsupported),
    (dict(experts=64, ld_logits=64, top_k=33), S.kErrorUnsupported), (dict(logits=None), S.kErrorInvalidArguments),
    (dict(ids=None), S.kErrorInvalidArguments), (dict(weights=None), S.kErrorInvalidArguments),
    (dict(order=None), S.kErrorInvalidArguments), (dict(offsets=None), S.kErrorInvalidArguments),
    (dict(ld_logits=7), S.kErrorInvalidArguments),
    (dict(tokens=1 << 30, top_k=4), S.kErrorInvalidArguments)])
def test_route_refuses(lib, change, status):
    assert route(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(a_format=0), S.kErrorBadDescriptor), (dict(b_format=9), S.kErrorBadDescriptor),
    (dict(a_format=_capi.FMT_E2M1), S.kErrorUnsupported), (dict(rows=-1), S.kErrorInvalidProblem),
    (dict(n=-1), S.kErrorInvalidProblem), (dict(k=-1), S.kErrorInvalidProblem), (dict(groups=-1), S.kErrorInvalidProblem),
    (dict(rows=0, a=None), S.kSuccess), (dict(n=0, d=None), S.kSuccess), (dict(k=0), S.kErrorInvalidArguments),
    (dict(groups=1025), S.kErrorUnsupported), (dict(pairs_per_a_row=0), S.kErrorInvalidArguments),
    (dict(pairs_per_d_row=0), S.kErrorInvalidArguments), (dict(pairs_per_d_row=3), S.kErrorInvalidArguments),
    (dict(a_rows=7), S.kErrorInvalidArguments), (dict(a_rows=0), S.kErrorInvalidArguments),
    (dict(pairs_per_d_row=2, ids=None), S.kErrorInvalidArguments), (dict(a=None), S.kErrorInvalidArguments),
    (dict(b=None), S.kErrorInvalidArguments), (dict(a_scales=None), S.kErrorInvalidArguments),
    (dict(b_scales=None), S.kErrorInvalidArguments), (dict(offsets=None), S.kErrorInvalidArguments),
    (dict(order=None), S.kErrorInvalidArguments), (dict(d=None), S.kErrorInvalidArguments),
    (dict(lda=63), S.kErrorInvalidArguments), (dict(ldb=48), S.kErrorInvalidArguments),
    (dict(ld_scales_a=1), S.kErrorInvalidArguments), (dict(ld_scales_b=1), S.kErrorInvalidArguments),
    (dict(ldd=15), S.kErrorInvalidArguments), (dict(b_group_rows=15), S.kErrorInvalidArguments),
    (dict(gated=1), S.kErrorInvalidArguments),              # b_group_rows covers half of 2 n
    (dict(lda=72), S.kErrorInvalidArguments), (dict(a=BASE + 8), S.kErrorInvalidArguments),
    (dict(ldb=72), S.kErrorInvalidArguments), (dict(b=BASE + 4), S.kErrorInvalidArguments),
    (dict(b_group_rows=1 << 30), S.kErrorInvalidArguments),
    (dict(a_format=_capi.FMT_E2M1, b_format=_capi.FMT_E2M1, k=63), S.kErrorInvalidArguments),
    (dict(b_format=_capi.FMT_E2M1), S.kErrorInvalidArguments),   # k is no multiple of 128
    (dict(b_format=_capi.FMT_E2M1, k=128, lda=128, ldb=160, ld_scales_a=4, ld_scales_b=4), S.kErrorInvalidArguments)])
def test_grouped_refuses(lib, change, status):
    assert grouped(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(x_type=3), S.kErrorBadDescriptor), (dict(w_type=-1), S.kErrorBadDescriptor), (dict(w_type=0), S.kErrorUnsupported),
    (dict(x_type=1), S.kErrorUnsupported), (dict(m=-1), S.kErrorInvalidProblem), (dict(rank=-1), S.kErrorInvalidProblem),
    (dict(m=0, x=None), S.kSuccess), (dict(n=0, d=None), S.kSuccess), (dict(rank=257, ldb=257), S.kErrorUnsupported),
    (dict(x=None), S.kErrorInvalidArguments), (dict(a=None), S.kErrorInvalidArguments), (dict(b=None), S.kErrorInvalidArguments),
    (dict(ids=None), S.kErrorInvalidArguments), (dict(c=None), S.kErrorInvalidArguments), (dict(d=None), S.kErrorInvalidArguments),
    (dict(ldx=31), S.kErrorInvalidArguments), (dict(lda=31), S.kErrorInvalidArguments), (dict(ldb=7), S.kErrorInvalidArguments),
    (dict(ldc=15), S.kErrorInvalidArguments), (dict(ldd=15), S.kErrorInvalidArguments), (dict(a_stride=-1), S.kErrorInvalidArguments),
    (dict(k=(1 << 30) + 1, ldx=(1 << 30) + 1, lda=(1 << 30) + 1), S.kErrorInvalidArguments),
    (dict(d=BASE, ldd=20), S.kErrorInvalidArguments)])
def test_adapters_refuse(lib, change, status):
    assert adapters(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), S.kErrorInvalidProblem), (dict(groups=-1), S.kErrorInvalidProblem), (dict(ids=None), S.kErrorInvalidArguments),
    (dict(offsets=None), S.kErrorInvalidArguments), (dict(order=None), S.kErrorInvalidArguments),
    (dict(groups=1025), S.kErrorUnsupported)])
def test_group_rows_refuse(lib, change, status):
    assert group_rows(**change) == status


def test_valid_calls_reach_the_device(lib):
    """Every refusal above is one field away from a call that only lacks a GPU here."""
    if lib.cpuops_b200_device_count() > 0:
        pytest.skip("a GPU is present: the same calls run in the gpu tests")
    for call in (route, grouped, adapters, group_rows):
        assert call() == S.kErrorNoDevice


def test_descriptors_of_operators(lib):
    op = c.GemmMxGrouped(c.fp8e4m3_t, c.fp4e2m1_t, gated=True, device=3)
    d = op.describe(op.Arguments(c.GroupedCoord(24, 96, 128, 5), c.MxTensorRef(16, 32, 128, 4), c.MxTensorRef(48, 64, 128, 4),
                                 c.RowPlan(80, 96), c.TensorRef(112, 100), pairs_per_a_row=3))
    assert (d.a_rows, d.b_group_rows, d.gated, d.device, d.pairs_per_d_row) == (8, 192, 1, 3, 1)
    assert (d.a_format, d.b_format) == (_capi.FMT_E4M3, _capi.FMT_E2M1)
    assert (d.offsets, d.order, d.d, d.ldd) == (80, 96, 112, 100)
