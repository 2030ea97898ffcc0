"""Products with weights held in 4 bits under group scales.

  W4WeightsPlan     weights quantized and laid out for the products, and read back
  W4LinearPlan      x W^T for one token, a few or a prompt
  MoeW4GroupedPlan  the same by expert, for the pairs of a mixture

No counterpart in the reference; beside the int8 weight-only GEMV and the grouped
int8 products of ``plans``, in their manner: ``select`` a plan for a descriptor,
``run`` it on a stream (torch's current one by default); ``run`` neither allocates
nor synchronises, so it can be captured into a graph, and errors are the exceptions
of ``plans``.  Operands are checked against the descriptor in the binding
(csrc/w4_binding.cpp), before any launch.

A weight is a code (sign, two exponent bits, one mantissa bit) times a power of two
that 32 consecutive weights of a row share; include/baracuda_kernels.h describes the
packed bytes.
"""
from __future__ import annotations

import struct
from dataclasses import dataclass

import torch

from .ffi import lib
from .plans import ElementKind, InvalidProblem, Unsupported, check

try:
    from . import _w4
except ImportError as e:      # no fallback: the operands' checks and the calls are in it
    raise RuntimeError("baracuda_amd/_w4.so is missing or does not fit: build it with "
                       "`python -m baracuda_amd.build`") from e


def _raw_stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# torch's own lookup by device index where it has one: no Stream object for each call
_w4.connect(InvalidProblem, getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream))

_TAG = {ElementKind.F32: 0, ElementKind.F16: 1, ElementKind.Bf16: 2}


def packed_bytes(n: int, k: int) -> int:
    """Bytes of one packed matrix [N, K]."""
    if not (1 <= n < 2 ** 31 and 1 <= k < 2 ** 31):
        raise InvalidProblem(f"packed_bytes({n}, {k})")
    return int(lib().w4_packed_bytes_gfx950(n, k))


def _element(desc) -> int:
    if desc.element not in _TAG:
        raise Unsupported(f"element {desc.element}: F32, F16 or Bf16")
    return _TAG[desc.element]


def _sizes_fit(desc) -> None:
    """Sizes as the C entries take them."""
    for name, value in vars(desc).items():
        if isinstance(value, int) and not -2 ** 31 <= value < 2 ** 31:
            raise Unsupported(f"{name} = {value}")


def _pack(element, n, k, rows=0, matrices=1, topk=1, gated=False, bytes_of=0) -> bytes:
    """A plan's sizes as the binding reads them (struct Sizes)."""
    return struct.pack("8q", element, n, k, rows, matrices, topk, gated, bytes_of)


# ---- weights -------------------------------------------------------------------
@dataclass(frozen=True)
class W4WeightsDescriptor:
    n: int
    k: int
    matrices: int = 1
    element: ElementKind = ElementKind.Bf16


class W4WeightsPlan:
    """Matrices [N, K] (or [matrices, N, K]) and their packed form, uint8 [matrices,
    packed_bytes(N, K)]."""

    def __init__(self, desc: W4WeightsDescriptor):
        d = self.desc = desc
        self._packed = _pack(_element(d), d.n, d.k, matrices=d.matrices, bytes_of=packed_bytes(d.n, d.k))

    @classmethod
    def select(cls, desc: W4WeightsDescriptor) -> "W4WeightsPlan":
        _sizes_fit(desc)
        check(lib().w4_weights_gfx950_can_implement(desc.matrices, desc.n, desc.k, _element(desc)), "W4WeightsPlan::select")
        return cls(desc)

    def workspace_size(self) -> int:
        return 0

    def quantize(self, weights, packed, stream=None) -> None:
        """Each group's scale is the smallest power of two under which no magnitude of
        it reaches 7, codes are the nearest, ties to the even one."""
        st = _w4.quantize(self._packed, stream, weights, packed)
        if st:
            check(st, "W4WeightsPlan::quantize")

    def pack(self, codes, scales, packed, stream=None) -> None:
        """From codes uint8 [.., N, K / 2] and scales uint8 [.., N, K / 32], as a
        checkpoint holds them; the descriptor's element has no part in it, and no scale is
        refused: what a product's element cannot hold is rounded there (W4LinearPlan)."""
        st = _w4.pack(self._packed, stream, codes, scales, packed)
        if st:
            check(st, "W4WeightsPlan::pack")

    def read(self, packed, weights, stream=None) -> None:
        """The values that packed weights stand for, rounded to the element."""
        st = _w4.read(self._packed, stream, packed, weights)
        if st:
            check(st, "W4WeightsPlan::read")


# ---- products --------------------------------------------------------------------
@dataclass(frozen=True)
class W4LinearDescriptor:
    m: int                             # tokens
    n: int                             # rows of the weights
    k: int
    element: ElementKind = ElementKind.Bf16
    gated: bool = False                # out = silu(y[:, :n / 2]) * y[:, n / 2:]


class W4LinearPlan:
    """out [M, N] (gated: [M, N / 2]) = x [M, K] W^T + bias, f32 [N].  Sums, bias and
    gate are held in 32 bits and rounded once.  Weights enter as elements: in bf16 as
    they are (scales of 2^-125 to 2^125), in f16 with scales of 2^-23 to 2^13; beyond
    these they are rounded to the element, in f16 to infinity from 65520 on.  ``quantize``
    keeps scales of f16 weights below that, a checkpoint in bf16 or f32 need not."""

    def __init__(self, desc: W4LinearDescriptor):
        d = self.desc = desc
        self._packed = _pack(_element(d), d.n, d.k, rows=d.m, gated=d.gated, bytes_of=packed_bytes(d.n, d.k))

    @classmethod
    def select(cls, desc: W4LinearDescriptor) -> "W4LinearPlan":
        _sizes_fit(desc)
        check(lib().w4_linear_gfx950_can_implement(*cls._sizes(desc)), "W4LinearPlan::select")
        return cls(desc)

    @staticmethod
    def _sizes(d) -> list:
        return [d.m, d.n, d.k, _element(d), int(d.gated)]

    def workspace_size(self) -> int:
        """Bytes that `run` needs beside its operands; what they hold does not matter."""
        return int(lib().w4_linear_gfx950_workspace_size(*self._sizes(self.desc)))

    def run(self, x, packed, out, bias=None, workspace=None, stream=None) -> None:
        st = _w4.linear(self._packed, stream, x, packed, out, bias, workspace)
        if st:
            check(st, "W4LinearPlan::run")


@dataclass(frozen=True)
class MoeW4GroupedDescriptor:
    num_experts: int
    topk: int
    size_m: int                        # token-expert pairs
    n: int
    k: int
    element: ElementKind = ElementKind.Bf16
    gated: bool = False


class MoeW4GroupedPlan:
    """W4LinearPlan's product by expert, with the routing contract of
    ``plans.MoeS8GroupedPlan``: position p of the pairs sorted by expert is pair
    sorted_token_ids[p] of expert expert_ids[p]; a pair's input row is pair / topk
    (the pair's own with topk_weights, which scale its output), its output row the
    pair's own.  Positions of no expert (num_experts, all of them last) are left out.

    The rows of x times K are less than 2^30.  ``select`` refuses what passes it with
    ceil(size_m / topk) rows; with topk_weights x has size_m rows, and ``run`` refuses
    those that pass it."""

    def __init__(self, desc: MoeW4GroupedDescriptor):
        d = self.desc = desc
        self._packed = _pack(_element(d), d.n, d.k, rows=d.size_m, matrices=d.num_experts, topk=d.topk, gated=d.gated,
                             bytes_of=packed_bytes(d.n, d.k))

    @classmethod
    def select(cls, desc: MoeW4GroupedDescriptor) -> "MoeW4GroupedPlan":
        _sizes_fit(desc)
        check(lib().moe_w4_grouped_gfx950_can_implement(*cls._sizes(desc)), "MoeW4GroupedPlan::select")
        return cls(desc)

    @staticmethod
    def _sizes(d) -> list:
        return [d.num_experts, d.topk, d.size_m, d.n, d.k, _element(d), int(d.gated)]

    def workspace_size(self) -> int:
        """Bytes that `run` needs beside its operands; what they hold does not matter."""
        return int(lib().moe_w4_grouped_gfx950_workspace_size(*self._sizes(self.desc)))

    def run(self, x, packed, sorted_token_ids, expert_ids, out, expert_counts, expert_offsets, bias=None,
            topk_weights=None, workspace=None, stream=None) -> None:
        st = _w4.grouped(self._packed, stream, x, packed, sorted_token_ids, expert_ids, out, expert_counts,
                         expert_offsets, bias, topk_weights, workspace)
        if st:
            check(st, "MoeW4GroupedPlan::run")


__all__ = ["W4WeightsDescriptor", "W4WeightsPlan", "W4LinearDescriptor", "W4LinearPlan", "MoeW4GroupedDescriptor",
           "MoeW4GroupedPlan", "packed_bytes", "InvalidProblem", "Unsupported"]
