"""Projections whose weights are chosen per row: routing to experts, the experts' products on
MX operands, low-rank adapters beside a shared projection.

The reference has no counterpart.  Names and calls follow ``gemm.py``: an operator takes its
``Arguments`` and returns a ``Status``, ``describe`` / ``run`` keep the descriptor of a
repeated call, buffers are torch CUDA tensors or raw device addresses (the index arrays that
choose the weights stay on the device: host memory is refused).  All work is done by
``libcpu_ops_b200.so``.
"""
from __future__ import annotations

import ctypes as C
import enum
from dataclasses import dataclass, field
from typing import Any, Optional

from . import _capi
from .gemm import MxTensorRef, Status, TensorRef, _Operator, data_ptr, fp8e4m3_t


class f32_t:
    type = _capi.TYPE_F32


class f16_t:
    type = _capi.TYPE_F16


class bf16_t:
    type = _capi.TYPE_BF16


class Scoring(enum.IntEnum):
    kSoftmax = _capi.SCORE_SOFTMAX
    kSigmoid = _capi.SCORE_SIGMOID


@dataclass
class RowPlan:
    """Pairs (a row and one of its groups) sorted by group, int32: ``order`` holds pair numbers,
    ``offsets[g]:offsets[g + 1]`` those of group g; -1 behind the last."""
    offsets: Any = None
    order: Any = None


@dataclass
class RouteCoord:
    tokens: int = 0
    experts: int = 0
    top_k: int = 0


@dataclass
class ExpertGroups:
    """Only experts of the ``top`` best of ``count`` equal runs are chosen; a run counts as the
    sum of its ``best`` (1 or 2) best experts."""
    count: int = 1
    top: int = 1
    best: int = 1


@dataclass
class GroupedCoord:
    """``rows`` pairs, each times its group's n x k matrix (gated: 2n x k)."""
    rows: int = 0
    n: int = 0
    k: int = 0
    groups: int = 0


@dataclass
class AdapterCoord:
    m: int = 0
    n: int = 0
    k: int = 0
    rank: int = 0
    adapters: int = 0


@dataclass
class AdapterRef:
    """One factor of every adapter: rows ``ld`` elements apart, adapters ``stride``."""
    data: Any = None
    ld: int = 0
    stride: int = 0


@dataclass
class RouteArguments:
    problem_size: RouteCoord = field(default_factory=RouteCoord)
    ref_logits: TensorRef = field(default_factory=TensorRef)
    ids: Any = None
    weights: Any = None
    plan: Optional[RowPlan] = None
    scoring: Scoring = Scoring.kSoftmax
    bias: Any = None
    groups: ExpertGroups = field(default_factory=ExpertGroups)
    renormalize: bool = True
    scale: float = 1.0


@dataclass
class GroupRowsArguments:
    rows: int = 0
    groups: int = 0
    ids: Any = None
    plan: RowPlan = field(default_factory=RowPlan)


@dataclass
class GemmGroupedArguments:
    """``ref_B`` covers all groups; group g starts at its row ``g * b_group_rows`` (0: the rows
    of one group).  ``a_rows`` 0: as many as the pairs need.  With ``ids`` (those of the plan; needed
    where ``pairs_per_d_row`` > 1) rows of D without a group become zeros, without they are left."""
    problem_size: GroupedCoord = field(default_factory=GroupedCoord)
    ref_A: MxTensorRef = field(default_factory=MxTensorRef)
    ref_B: MxTensorRef = field(default_factory=MxTensorRef)
    plan: RowPlan = field(default_factory=RowPlan)
    ref_D: TensorRef = field(default_factory=TensorRef)
    pairs_per_a_row: int = 1
    row_weights: Any = None
    pairs_per_d_row: int = 1
    ids: Any = None
    a_rows: int = 0
    b_group_rows: int = 0


@dataclass
class AdaptersArguments:
    problem_size: AdapterCoord = field(default_factory=AdapterCoord)
    ref_X: TensorRef = field(default_factory=TensorRef)
    ref_A: AdapterRef = field(default_factory=AdapterRef)
    ref_B: AdapterRef = field(default_factory=AdapterRef)
    ids: Any = None
    ref_C: TensorRef = field(default_factory=TensorRef)
    ref_D: TensorRef = field(default_factory=TensorRef)
    scales: Any = None


class _RowOperator(_Operator):
    """Stream, device and error plumbing as for the GEMM operators."""

    _entry = ""

    def __init__(self, *, stream: Optional[int] = None, asynchronous: bool = False,
                 memory_space: int = _capi.MEM_AUTO, device: int = -1):
        super().__init__(stream=stream, asynchronous=asynchronous, memory_space=memory_space, device=device)
        self._call = getattr(_capi.load(), self._entry)

    def run(self, desc) -> Status:
        return Status(self._call(C.byref(desc)))

    def __call__(self, args) -> Status:
        desc = self.describe(args)
        if self._stream is None:
            _settle(args)
        return self.run(desc)

    def _place(self, desc):
        desc.struct_size = C.sizeof(type(desc))
        desc.stream = self._stream
        desc.flags = _capi.FLAG_ASYNC if self._async else 0
        desc.device = self._device
        desc.memory_space = self._memory_space
        return desc


def _settle(args) -> None:
    """The library's own stream is not ordered after torch's: wait for torch's current stream of
    the first CUDA tensor's device, so that what was enqueued there has landed."""
    for value in vars(args).values():
        for buf in (value, getattr(value, "data", None), getattr(value, "order", None)):
            if getattr(buf, "is_cuda", False):
                import torch
                torch.cuda.current_stream(buf.device).synchronize()
                return


class RouteExperts(_RowOperator):
    """Scores of logits, the best experts of every token with their weights, and the row plan."""

    Arguments = RouteArguments
    _entry = "cpuops_b200_route"

    def __init__(self, storage=f32_t, **kw):
        super().__init__(**kw)
        self.Storage = storage

    def describe(self, args: RouteArguments) -> _capi.RouteDesc:
        desc = _capi.RouteDesc()
        ps, groups, plan = args.problem_size, args.groups, args.plan or RowPlan()
        desc.tokens, desc.experts, desc.top_k = int(ps.tokens), int(ps.experts), int(ps.top_k)
        desc.scoring = int(args.scoring)
        desc.n_groups, desc.top_groups, desc.group_best = int(groups.count), int(groups.top), int(groups.best)
        desc.renormalize, desc.scale = int(bool(args.renormalize)), float(args.scale)
        desc.logits_type, desc.ld_logits = self.Storage.type, int(args.ref_logits.ld)
        desc.logits, desc.bias = data_ptr(args.ref_logits.data), data_ptr(args.bias)
        desc.ids, desc.weights = data_ptr(args.ids), data_ptr(args.weights)
        desc.offsets, desc.order = data_ptr(plan.offsets), data_ptr(plan.order)
        return self._place(desc)


class GroupRows(_RowOperator):
    """The row plan of ids that come from elsewhere."""

    Arguments = GroupRowsArguments
    _entry = "cpuops_b200_group_rows"

    def describe(self, args: GroupRowsArguments) -> _capi.GroupRowsDesc:
        desc = _capi.GroupRowsDesc()
        desc.rows, desc.groups = int(args.rows), int(args.groups)
        desc.ids = data_ptr(args.ids)
        desc.offsets, desc.order = data_ptr(args.plan.offsets), data_ptr(args.plan.order)
        return self._place(desc)


class GemmMxGrouped(_RowOperator):
    """The experts' products: MX rows of A, gathered by the plan, times each group's MX matrix.
    ``gated``: a group's matrix holds n gate rows, then n up rows, and a pair's result is
    silu(gate) * up."""

    Arguments = GemmGroupedArguments
    _entry = "cpuops_b200_gemm_grouped"

    def __init__(self, storage_a=fp8e4m3_t, storage_b=None, gated: bool = False, **kw):
        super().__init__(**kw)
        self.StorageA, self.StorageB = storage_a, storage_b or storage_a
        self.gated = bool(gated)

    def describe(self, args: GemmGroupedArguments) -> _capi.GemmGroupedDesc:
        desc = _capi.GemmGroupedDesc()
        ps, a, b = args.problem_size, args.ref_A, args.ref_B
        desc.a_format, desc.b_format = self.StorageA.fmt, self.StorageB.fmt
        desc.rows, desc.n, desc.k, desc.groups = int(ps.rows), int(ps.n), int(ps.k), int(ps.groups)
        desc.gated = int(self.gated)
        desc.pairs_per_a_row, desc.pairs_per_d_row = int(args.pairs_per_a_row), int(args.pairs_per_d_row)
        desc.a_rows = int(args.a_rows) or -(-desc.rows // max(1, desc.pairs_per_a_row))
        desc.b_group_rows = int(args.b_group_rows) or desc.n * (2 if self.gated else 1)
        desc.a, desc.a_scales = data_ptr(a.data), data_ptr(a.scales)
        desc.lda, desc.ld_scales_a = int(a.ld), int(a.ld_scales)
        desc.b, desc.b_scales = data_ptr(b.data), data_ptr(b.scales)
        desc.ldb, desc.ld_scales_b = int(b.ld), int(b.ld_scales)
        desc.offsets, desc.order = data_ptr(args.plan.offsets), data_ptr(args.plan.order)
        desc.ids, desc.row_weights = data_ptr(args.ids), data_ptr(args.row_weights)
        desc.d, desc.ldd = data_ptr(args.ref_D.data), int(args.ref_D.ld)
        return self._place(desc)


class LowRankAdapters(_RowOperator):
    """D = C + scale * (X A^T) B^T with one adapter (A, B, scale) per row, or none."""

    Arguments = AdaptersArguments
    _entry = "cpuops_b200_adapters"

    def __init__(self, storage_x=bf16_t, storage_w=None, **kw):
        super().__init__(**kw)
        self.StorageX, self.StorageW = storage_x, storage_w or storage_x

    def describe(self, args: AdaptersArguments) -> _capi.AdaptersDesc:
        desc = _capi.AdaptersDesc()
        ps = args.problem_size
        desc.m, desc.n, desc.k = int(ps.m), int(ps.n), int(ps.k)
        desc.rank, desc.adapters = int(ps.rank), int(ps.adapters)
        desc.x_type, desc.w_type = self.StorageX.type, self.StorageW.type
        desc.x, desc.ldx = data_ptr(args.ref_X.data), int(args.ref_X.ld)
        desc.a, desc.lda, desc.a_stride = data_ptr(args.ref_A.data), int(args.ref_A.ld), int(args.ref_A.stride)
        desc.b, desc.ldb, desc.b_stride = data_ptr(args.ref_B.data), int(args.ref_B.ld), int(args.ref_B.stride)
        desc.ids, desc.scales = data_ptr(args.ids), data_ptr(args.scales)
        desc.c, desc.ldc = data_ptr(args.ref_C.data), int(args.ref_C.ld)
        desc.d, desc.ldd = data_ptr(args.ref_D.data), int(args.ref_D.ld)
        return self._place(desc)
