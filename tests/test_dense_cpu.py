"""What the 16-bit layers' operators refuse, before they touch a device."""
import ctypes as C

import numpy as np
import pytest

import cpu_ops_b200 as c
from cpu_ops_b200 import _capi

S = c.Status
BUF = np.zeros(1 << 16, np.uint8)
BASE = (BUF.ctypes.data + 255) // 256 * 256
F32, F16, BF16 = _capi.TYPE_F32, _capi.TYPE_F16, _capi.TYPE_BF16
BIG = (1 << 30) + 1


def _call(entry, kind, fields, change):
    d = kind(struct_size=C.sizeof(kind), device=-1, **fields)
    for k, v in change.items():
        setattr(d, k, v)
    return S(getattr(_capi.load(), "cpuops_b200_" + entry)(C.byref(d)))


def gemm16(**kw):
    return _call("gemm16", _capi.Gemm16Desc, dict(
        type=BF16, c_type=BF16, d_type=BF16, m=4, n=16, k=32, a_row_major=1, b_row_major=0, lda=32, ldb=32, ldc=16, ldd=16, ldz=16,
        alpha=1.0, beta=1.0, a=BASE, b=BASE, c=BASE, d=BASE + 4096, z=BASE + 8192, bias=BASE), kw)


def epilogue_grad(**kw):
    return _call("epilogue_grad", _capi.EpilogueGradDesc, dict(
        type=BF16, m=4, n=16, activation=_capi.OP_GELU, lddy=16, ldz=16, lddz=16, dy=BASE, z=BASE + 4096, dz=BASE + 8192,
        dbias=BASE + 12288), kw)


def layer_norm(**kw):
    return _call("layer_norm", _capi.LayerNormDesc, dict(
        x_type=F32, y_type=BF16, m=4, n=16, ldx=16, ldy=16, eps=1e-5, x=BASE, gamma=BASE, beta=BASE, y=BASE + 4096,
        mean=BASE + 8192, rstd=BASE + 12288), kw)


def layer_norm_grad(**kw):
    return _call("layer_norm_grad", _capi.LayerNormGradDesc, dict(
        x_type=F32, y_type=BF16, m=4, n=16, lddy=16, ldx=16, lddr=16, lddx=16, dy=BASE, x=BASE, dr=BASE, gamma=BASE, mean=BASE,
        rstd=BASE, dx=BASE + 4096, dgamma=BASE + 8192, dbeta=BASE + 12288), kw)


def balance_loss(**kw):
    return _call("balance_loss", _capi.BalanceLossDesc, dict(
        tokens=4, experts=8, top_k=2, coefficient=1.0, ld_logits=8, ld_dlogits=8, logits=BASE, ids=BASE, counts=BASE + 4096,
        loss=BASE + 8192, dlogits=BASE + 12288), kw)


CALLS = [gemm16, epilogue_grad, layer_norm, layer_norm_grad, balance_loss]


@pytest.mark.parametrize("call", CALLS)
def test_descriptor_size_is_checked(lib, call):
    assert call(struct_size=8) == S.kErrorBadDescriptor


@pytest.mark.parametrize("change,status", [
    (dict(type=3), S.kErrorBadDescriptor), (dict(c_type=-1), S.kErrorBadDescriptor), (dict(d_type=9), S.kErrorBadDescriptor),
    (dict(activation=_capi.OP_CLAMP), S.kErrorBadDescriptor), (dict(activation=-1), S.kErrorBadDescriptor),
    (dict(type=F32), S.kErrorUnsupported), (dict(d_type=F16), S.kErrorUnsupported), (dict(c_type=F16), S.kErrorUnsupported),
    (dict(m=-1), S.kErrorInvalidProblem), (dict(n=-1), S.kErrorInvalidProblem), (dict(k=-1), S.kErrorInvalidProblem),
    (dict(m=0, a=None), S.kSuccess), (dict(n=0, d=None), S.kSuccess),
    (dict(m=BIG), S.kErrorInvalidArguments), (dict(n=BIG), S.kErrorInvalidArguments), (dict(k=BIG), S.kErrorInvalidArguments),
    (dict(a=None), S.kErrorInvalidArguments), (dict(b=None), S.kErrorInvalidArguments), (dict(c=None), S.kErrorInvalidArguments),
    (dict(d=None), S.kErrorInvalidArguments),
    (dict(lda=31), S.kErrorInvalidArguments), (dict(ldb=31), S.kErrorInvalidArguments), (dict(ldc=15), S.kErrorInvalidArguments),
    (dict(ldd=15), S.kErrorInvalidArguments), (dict(ldz=15), S.kErrorInvalidArguments),
    (dict(a_row_major=0, lda=3), S.kErrorInvalidArguments), (dict(b_row_major=1, ldb=15), S.kErrorInvalidArguments),
    (dict(c=BASE + 4096, ldc=20), S.kErrorInvalidArguments), (dict(c=BASE + 4096, c_type=F32), S.kErrorInvalidArguments),
    (dict(z=BASE + 4096), S.kErrorInvalidArguments), (dict(z=BASE), S.kErrorInvalidArguments),
    (dict(split_k_slices=3), S.kErrorInvalidArguments), (dict(split_k_slices=16), S.kErrorInvalidArguments),
    (dict(split_k_slices=-1), S.kErrorInvalidArguments), (dict(tile_n=24), S.kErrorInvalidArguments), (dict(tile_n=512), S.kErrorInvalidArguments),
    (dict(a=BASE + 1), S.kErrorInvalidArguments), (dict(b=BASE + 1), S.kErrorInvalidArguments), (dict(c=BASE + 1), S.kErrorInvalidArguments),
    (dict(d=BASE + 4097), S.kErrorInvalidArguments), (dict(z=BASE + 8193), S.kErrorInvalidArguments),
    (dict(bias=BASE + 2), S.kErrorInvalidArguments)])
def test_gemm16_refuses(lib, change, status):
    assert gemm16(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(type=3), S.kErrorBadDescriptor), (dict(activation=2), S.kErrorBadDescriptor), (dict(m=-1), S.kErrorInvalidProblem),
    (dict(n=-1), S.kErrorInvalidProblem), (dict(n=0, dy=None), S.kSuccess), (dict(m=0, dbias=None, dy=None), S.kSuccess),
    (dict(m=BIG), S.kErrorInvalidArguments), (dict(n=BIG), S.kErrorInvalidArguments), (dict(dy=None), S.kErrorInvalidArguments),
    (dict(z=None), S.kErrorInvalidArguments), (dict(dz=None), S.kErrorInvalidArguments),
    (dict(activation=0, dz=None, dbias=None), S.kErrorInvalidArguments), (dict(lddy=15), S.kErrorInvalidArguments),
    (dict(ldz=15), S.kErrorInvalidArguments), (dict(lddz=15), S.kErrorInvalidArguments), (dict(dz=BASE, lddz=20), S.kErrorInvalidArguments),
    (dict(dz=BASE + 4096, lddz=20), S.kErrorInvalidArguments), (dict(dy=BASE + 1), S.kErrorInvalidArguments),
    (dict(z=BASE + 4097), S.kErrorInvalidArguments), (dict(dz=BASE + 8193), S.kErrorInvalidArguments), (dict(dbias=BASE + 2), S.kErrorInvalidArguments)])
def test_epilogue_grad_refuses(lib, change, status):
    assert epilogue_grad(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(x_type=3), S.kErrorBadDescriptor), (dict(y_type=-1), S.kErrorBadDescriptor), (dict(x_type=F16), S.kErrorUnsupported),
    (dict(x_type=BF16, y_type=F32), S.kErrorUnsupported), (dict(m=-1), S.kErrorInvalidProblem), (dict(n=-1), S.kErrorInvalidProblem),
    (dict(m=0, x=None), S.kSuccess), (dict(n=0, y=None), S.kSuccess), (dict(m=BIG), S.kErrorInvalidArguments),
    (dict(n=BIG), S.kErrorInvalidArguments), (dict(eps=-1e-5), S.kErrorInvalidArguments), (dict(eps=float("nan")), S.kErrorInvalidArguments),
    (dict(x=None), S.kErrorInvalidArguments), (dict(y=None), S.kErrorInvalidArguments), (dict(ldx=15), S.kErrorInvalidArguments),
    (dict(ldy=15), S.kErrorInvalidArguments), (dict(y=BASE), S.kErrorInvalidArguments), (dict(x=BASE + 2), S.kErrorInvalidArguments),
    (dict(y=BASE + 4097), S.kErrorInvalidArguments), (dict(gamma=BASE + 2), S.kErrorInvalidArguments),
    (dict(y_type=F32, y=BASE, ldy=20), S.kErrorInvalidArguments)])
def test_layer_norm_refuses(lib, change, status):
    assert layer_norm(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(x_type=3), S.kErrorBadDescriptor), (dict(x_type=F16), S.kErrorUnsupported), (dict(m=-1), S.kErrorInvalidProblem),
    (dict(n=-1), S.kErrorInvalidProblem), (dict(n=0, x=None), S.kSuccess), (dict(m=0, dgamma=None, dbeta=None, x=None), S.kSuccess),
    (dict(m=BIG), S.kErrorInvalidArguments), (dict(n=BIG), S.kErrorInvalidArguments),
    (dict(dy=None), S.kErrorInvalidArguments), (dict(x=None), S.kErrorInvalidArguments), (dict(mean=None), S.kErrorInvalidArguments),
    (dict(rstd=None), S.kErrorInvalidArguments), (dict(dx=None), S.kErrorInvalidArguments), (dict(lddy=15), S.kErrorInvalidArguments),
    (dict(ldx=15), S.kErrorInvalidArguments), (dict(lddr=15), S.kErrorInvalidArguments), (dict(lddx=15), S.kErrorInvalidArguments),
    (dict(dx=BASE), S.kErrorInvalidArguments),                                      # dY is of another type
    (dict(dy=BASE + 16384, dx=BASE, lddx=20), S.kErrorInvalidArguments), (dict(dx=BASE + 4098), S.kErrorInvalidArguments),
    (dict(dr=BASE + 2), S.kErrorInvalidArguments), (dict(dbeta=BASE + 12290), S.kErrorInvalidArguments)])
def test_layer_norm_grad_refuses(lib, change, status):
    assert layer_norm_grad(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(scoring=2), S.kErrorBadDescriptor), (dict(logits_type=5), S.kErrorBadDescriptor), (dict(tokens=-1), S.kErrorInvalidProblem),
    (dict(experts=0), S.kErrorInvalidProblem), (dict(top_k=0), S.kErrorInvalidProblem), (dict(experts=1025), S.kErrorUnsupported),
    (dict(top_k=33), S.kErrorUnsupported), (dict(tokens=1 << 30, top_k=4), S.kErrorInvalidArguments),
    (dict(logits=None), S.kErrorInvalidArguments), (dict(ids=None), S.kErrorInvalidArguments), (dict(ld_logits=7), S.kErrorInvalidArguments),
    (dict(ld_dlogits=7), S.kErrorInvalidArguments), (dict(dlogits=BASE, ld_dlogits=9), S.kErrorInvalidArguments),
    (dict(counts=None, loss=None, dlogits=None), S.kSuccess), (dict(logits=BASE + 2), S.kErrorInvalidArguments),
    (dict(ids=BASE + 2), S.kErrorInvalidArguments), (dict(upstream=BASE + 1), S.kErrorInvalidArguments)])
def test_balance_loss_refuses(lib, change, status):
    assert balance_loss(**change) == status


def test_valid_calls_reach_the_device(lib):
    """Every refusal above is one field away from a call that only lacks a GPU here."""
    if lib.cpuops_b200_device_count() > 0:
        pytest.skip("a GPU is present: the same calls run in the gpu tests")
    for call in CALLS:
        assert call() == S.kErrorNoDevice
    assert gemm16(beta=0.0, c=None, ldc=0, z=None, ldz=0, bias=None) == S.kErrorNoDevice
    assert gemm16(k=0, a=None, b=None) == S.kErrorNoDevice
    assert epilogue_grad(activation=0, z=None, ldz=0, dz=None, lddz=0) == S.kErrorNoDevice
    assert layer_norm(gamma=None, beta=None, mean=None, rstd=None) == S.kErrorNoDevice
    assert balance_loss(tokens=0, logits=None, ids=None) == S.kErrorNoDevice


def test_descriptors_of_operators(lib):
    op = c.GemmF16(c.ColumnMajor, c.RowMajor, storage_d=c.f32_t, device=3, pair=False, tile_n=64)
    d = op.describe(op.Arguments(c.GemmCoord(24, 96, 128), c.TensorRef(16, 24), c.TensorRef(32, 96), c.TensorRef(48, 97), c.TensorRef(64, 98),
                                 c.BiasActivation(80, c.Silu(), 0.5, 2.0), c.TensorRef(96, 99), 4))
    assert (d.type, d.c_type, d.d_type, d.activation) == (F16, F32, F32, _capi.OP_SILU)
    assert (d.m, d.n, d.k, d.a_row_major, d.b_row_major) == (24, 96, 128, 0, 1)
    assert (d.lda, d.ldb, d.ldc, d.ldd, d.ldz, d.alpha, d.beta) == (24, 96, 97, 98, 99, 0.5, 2.0)
    assert (d.a, d.b, d.bias, d.c, d.d, d.z) == (16, 32, 80, 48, 64, 96)
    assert (d.split_k_slices, d.tile_n, d.flags, d.device) == (4, 64, _capi.FLAG_PAIR_OFF, 3)
    op = c.LayerNormGrad(c.f32_t, c.f16_t)
    d = op.describe(op.Arguments(c.RowsCoord(5, 7), c.TensorRef(16, 8), c.TensorRef(32, 9), 48, 64, 80, c.TensorRef(96, 10), 112, 128,
                                 c.TensorRef(144, 11)))
    assert (d.x_type, d.y_type, d.m, d.n, d.lddy, d.ldx, d.lddr, d.lddx) == (F32, F16, 5, 7, 8, 9, 11, 10)
    assert (d.dy, d.x, d.dr, d.gamma, d.mean, d.rstd, d.dx, d.dgamma, d.dbeta) == (16, 32, 144, 48, 64, 80, 96, 112, 128)
