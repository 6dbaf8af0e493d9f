"""16-bit layers and their gradients: products with bias, activation and residual in the
epilogue, that epilogue's gradient, layer norm and its gradient, a router's balance loss.

The reference has 16-bit GEMMs (gemm/device/gemm.h) and layer norm (ops/norm.h) on the CPU, and no
gradients.  Names and calls follow ``row_chosen.py``: an operator takes its ``Arguments`` and
returns a ``Status``, ``describe`` / ``run`` keep the descriptor of a repeated call, buffers are
torch CUDA tensors or raw device addresses.  All work is done by ``libcpu_ops_b200.so``.

A layer's backward pass, of Y = act(X W^T + bias) + R with W by rows and Z kept:
    BiasActivationGrad: dZ, dbias of dY and Z (dR is dY itself)
    dX = dZ W           GemmBF16(RowMajor, RowMajor)
    dW = dZ^T X         GemmBF16(ColumnMajor, RowMajor, storage_d=f32_t), beta = 1 to add up
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Any

from . import _capi
from .gemm import GemmCoord, RowMajor, TensorRef, data_ptr
from .row_chosen import RouteCoord, Scoring, _RowOperator, bf16_t, f16_t, f32_t


@dataclass
class RowsCoord:
    """``rows`` rows of ``n`` elements."""
    rows: int = 0
    n: int = 0


@dataclass
class BiasActivation:
    """z = alpha * A B + bias, D = activation(z) + beta * C; ``activation`` is None, Relu(), Gelu()
    or Silu(), ``bias`` n floats or None."""
    bias: Any = None
    activation: Any = None
    alpha: float = 1.0
    beta: float = 0.0


@dataclass
class Gemm16Arguments:
    """``ref_Z`` without data: z is not kept.  ``split_k_slices`` 0: automatic."""
    problem_size: GemmCoord = field(default_factory=GemmCoord)
    ref_A: TensorRef = field(default_factory=TensorRef)
    ref_B: TensorRef = field(default_factory=TensorRef)
    ref_C: TensorRef = field(default_factory=TensorRef)
    ref_D: TensorRef = field(default_factory=TensorRef)
    epilogue: BiasActivation = field(default_factory=BiasActivation)
    ref_Z: TensorRef = field(default_factory=TensorRef)
    split_k_slices: int = 0


@dataclass
class BiasActivationGradArguments:
    """``ref_Z`` is not read without an activation; ``ref_dZ`` may then be left out."""
    problem_size: RowsCoord = field(default_factory=RowsCoord)
    ref_dY: TensorRef = field(default_factory=TensorRef)
    ref_Z: TensorRef = field(default_factory=TensorRef)
    ref_dZ: TensorRef = field(default_factory=TensorRef)
    dbias: Any = None


@dataclass
class LayerNormArguments:
    problem_size: RowsCoord = field(default_factory=RowsCoord)
    ref_X: TensorRef = field(default_factory=TensorRef)
    gamma: Any = None
    beta: Any = None
    ref_Y: TensorRef = field(default_factory=TensorRef)
    mean: Any = None
    rstd: Any = None
    eps: float = 1e-5


@dataclass
class LayerNormGradArguments:
    """``ref_dR``: a gradient that is added to dX (the residual stream's), or none."""
    problem_size: RowsCoord = field(default_factory=RowsCoord)
    ref_dY: TensorRef = field(default_factory=TensorRef)
    ref_X: TensorRef = field(default_factory=TensorRef)
    gamma: Any = None
    mean: Any = None
    rstd: Any = None
    ref_dX: TensorRef = field(default_factory=TensorRef)
    dgamma: Any = None
    dbeta: Any = None
    ref_dR: TensorRef = field(default_factory=TensorRef)


@dataclass
class BalanceLossArguments:
    """``upstream``: the loss's own gradient, one float on the device (None: 1)."""
    problem_size: RouteCoord = field(default_factory=RouteCoord)
    ref_logits: TensorRef = field(default_factory=TensorRef)
    ids: Any = None
    counts: Any = None
    loss: Any = None
    ref_dLogits: TensorRef = field(default_factory=TensorRef)
    scoring: Scoring = Scoring.kSoftmax
    coefficient: float = 1.0
    upstream: Any = None


def _opcode(activation) -> int:
    return 0 if activation is None else int(activation.opcode)


class _Gemm16(_RowOperator):
    Arguments = Gemm16Arguments
    _entry = "cpuops_b200_gemm16"
    Storage = bf16_t

    def __init__(self, layout_a=RowMajor, layout_b=RowMajor, *, storage_c=None, storage_d=None, tile_n: int = 0,
                 pair=None, **kw):
        super().__init__(**kw)
        self.LayoutA, self.LayoutB = layout_a, layout_b
        self.StorageD = storage_d or self.Storage
        self.StorageC = storage_c or self.StorageD
        # testing/tuning, as for the quantised GEMMs
        self._tile_n = tile_n
        self._pair_flag = 0 if pair is None else (_capi.FLAG_PAIR_ON if pair else _capi.FLAG_PAIR_OFF)

    def describe(self, args: Gemm16Arguments) -> _capi.Gemm16Desc:
        desc = _capi.Gemm16Desc()
        ps, epilogue = args.problem_size, args.epilogue
        desc.type, desc.c_type, desc.d_type = self.Storage.type, self.StorageC.type, self.StorageD.type
        desc.m, desc.n, desc.k = int(ps.m), int(ps.n), int(ps.k)
        desc.a_row_major, desc.b_row_major = int(self.LayoutA.kIsRowMajor), int(self.LayoutB.kIsRowMajor)
        desc.activation = _opcode(epilogue.activation)
        desc.alpha, desc.beta = float(epilogue.alpha), float(epilogue.beta)
        desc.bias = data_ptr(epilogue.bias)
        desc.a, desc.lda = data_ptr(args.ref_A.data), int(args.ref_A.ld)
        desc.b, desc.ldb = data_ptr(args.ref_B.data), int(args.ref_B.ld)
        desc.c, desc.ldc = data_ptr(args.ref_C.data), int(args.ref_C.ld)
        desc.d, desc.ldd = data_ptr(args.ref_D.data), int(args.ref_D.ld)
        desc.z, desc.ldz = data_ptr(args.ref_Z.data), int(args.ref_Z.ld)
        desc.split_k_slices, desc.tile_n = int(args.split_k_slices), int(self._tile_n)
        self._place(desc)
        desc.flags |= self._pair_flag
        return desc


class GemmBF16(_Gemm16):
    """D = activation(alpha * A B + bias) + beta * C of bf16 matrices; C and D bf16 or f32."""
    Storage = bf16_t


class GemmF16(_Gemm16):
    """The same of f16 matrices; C and D f16 or f32."""
    Storage = f16_t


class BiasActivationGrad(_RowOperator):
    """dZ = dY * activation'(Z) and dbias, the column sums of dZ."""

    Arguments = BiasActivationGradArguments
    _entry = "cpuops_b200_epilogue_grad"

    def __init__(self, storage=bf16_t, activation=None, **kw):
        super().__init__(**kw)
        self.Storage, self.activation = storage, activation

    def describe(self, args: BiasActivationGradArguments) -> _capi.EpilogueGradDesc:
        desc = _capi.EpilogueGradDesc()
        ps = args.problem_size
        desc.type, desc.activation = self.Storage.type, _opcode(self.activation)
        desc.m, desc.n = int(ps.rows), int(ps.n)
        desc.dy, desc.lddy = data_ptr(args.ref_dY.data), int(args.ref_dY.ld)
        desc.z, desc.ldz = data_ptr(args.ref_Z.data), int(args.ref_Z.ld)
        desc.dz, desc.lddz = data_ptr(args.ref_dZ.data), int(args.ref_dZ.ld)
        desc.dbias = data_ptr(args.dbias)
        return self._place(desc)


class LayerNorm(_RowOperator):
    """Y = (X - mean) * rstd * gamma + beta, row by row, with mean and rstd for the gradient."""

    Arguments = LayerNormArguments
    _entry = "cpuops_b200_layer_norm"

    def __init__(self, storage_x=bf16_t, storage_y=None, **kw):
        super().__init__(**kw)
        self.StorageX, self.StorageY = storage_x, storage_y or storage_x

    def describe(self, args: LayerNormArguments) -> _capi.LayerNormDesc:
        desc = _capi.LayerNormDesc()
        ps = args.problem_size
        desc.x_type, desc.y_type = self.StorageX.type, self.StorageY.type
        desc.m, desc.n, desc.eps = int(ps.rows), int(ps.n), float(args.eps)
        desc.x, desc.ldx = data_ptr(args.ref_X.data), int(args.ref_X.ld)
        desc.y, desc.ldy = data_ptr(args.ref_Y.data), int(args.ref_Y.ld)
        desc.gamma, desc.beta = data_ptr(args.gamma), data_ptr(args.beta)
        desc.mean, desc.rstd = data_ptr(args.mean), data_ptr(args.rstd)
        return self._place(desc)


class LayerNormGrad(_RowOperator):
    """dX, dgamma and dbeta of LayerNorm; ``storage_x`` is X's, dX's and dR's, ``storage_y`` dY's."""

    Arguments = LayerNormGradArguments
    _entry = "cpuops_b200_layer_norm_grad"

    def __init__(self, storage_x=bf16_t, storage_y=None, **kw):
        super().__init__(**kw)
        self.StorageX, self.StorageY = storage_x, storage_y or storage_x

    def describe(self, args: LayerNormGradArguments) -> _capi.LayerNormGradDesc:
        desc = _capi.LayerNormGradDesc()
        ps = args.problem_size
        desc.x_type, desc.y_type = self.StorageX.type, self.StorageY.type
        desc.m, desc.n = int(ps.rows), int(ps.n)
        desc.dy, desc.lddy = data_ptr(args.ref_dY.data), int(args.ref_dY.ld)
        desc.x, desc.ldx = data_ptr(args.ref_X.data), int(args.ref_X.ld)
        desc.dr, desc.lddr = data_ptr(args.ref_dR.data), int(args.ref_dR.ld)
        desc.dx, desc.lddx = data_ptr(args.ref_dX.data), int(args.ref_dX.ld)
        desc.gamma, desc.mean, desc.rstd = data_ptr(args.gamma), data_ptr(args.mean), data_ptr(args.rstd)
        desc.dgamma, desc.dbeta = data_ptr(args.dgamma), data_ptr(args.dbeta)
        return self._place(desc)


class BalanceLoss(_RowOperator):
    """Counts per expert, the loss coefficient * experts * sum_e f_e P_e, and its gradient by the
    logits: beside RouteExperts, on its ids."""

    Arguments = BalanceLossArguments
    _entry = "cpuops_b200_balance_loss"

    def __init__(self, storage=f32_t, **kw):
        super().__init__(**kw)
        self.Storage = storage

    def describe(self, args: BalanceLossArguments) -> _capi.BalanceLossDesc:
        desc = _capi.BalanceLossDesc()
        ps = args.problem_size
        desc.tokens, desc.experts, desc.top_k = int(ps.tokens), int(ps.experts), int(ps.top_k)
        desc.scoring, desc.coefficient = int(args.scoring), float(args.coefficient)
        desc.logits_type = self.Storage.type
        desc.logits, desc.ld_logits = data_ptr(args.ref_logits.data), int(args.ref_logits.ld)
        desc.dlogits, desc.ld_dlogits = data_ptr(args.ref_dLogits.data), int(args.ref_dLogits.ld)
        desc.ids, desc.upstream = data_ptr(args.ids), data_ptr(args.upstream)
        desc.counts, desc.loss = data_ptr(args.counts), data_ptr(args.loss)
        return self._place(desc)
