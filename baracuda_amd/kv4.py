"""A key-value cache held in 4 bits: what fills it, attention over it, its pages.

  QkNormRopePlan    RMS norm of each head of Q and K and the position rotation
  Kv4AppendPlan     the same, and K and V quantized into pages of the cache
  Kv4ReadPlan       the values that slots of the cache stand for
  Kv4AttentionPlan  attention of a ragged batch over its pages
  KvPagesPlan       copying, forking, releasing and compacting pages

No counterpart in the reference.  The manner is that of ``plans``: ``select`` a
plan for a descriptor, ``run`` it on a stream (torch's current one by default);
``run`` neither allocates nor synchronises, so it can be captured into a graph,
and errors are the exceptions of ``plans``.  Operands are checked
against the descriptor in the binding (csrc/kv4_binding.cpp), before any launch.

The cache is a uint8 tensor [pages, kv heads, kv4.head_bytes(page size, D)], two
codes a byte (sign, two exponent bits, one mantissa bit); 32 values share a
power of two.  include/baracuda_kernels.h describes its bytes.
"""
from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Optional

import torch

from .ffi import lib
from .plans import ElementKind, InvalidProblem, Unsupported, _need, check

try:
    from . import _kv4
except ImportError as e:      # no fallback: the operands' checks and the calls are in it
    raise RuntimeError("baracuda_amd/_kv4.so is missing or does not fit: build it with "
                       "`python -m baracuda_amd.build`") from e


def _raw_stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# torch's own lookup by device index where it has one: no Stream object for each call
_kv4.connect(InvalidProblem, getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream))

_TAG = {ElementKind.F32: 0, ElementKind.F16: 1, ElementKind.Bf16: 2}


def head_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one head of one page."""
    return page_size * (head_dim + head_dim // 16)


def _element(desc) -> int:
    if desc.element not in _TAG:
        raise Unsupported(f"element {desc.element}: F32, F16 or Bf16")
    return _TAG[desc.element]


_INT64 = ("tokens", "num_pages", "max_kv", "page_bytes")


def _sizes_fit(desc) -> None:
    """Sizes as the C entries take them: 64 bits for the long ones, 32 for the others."""
    for name, value in vars(desc).items():
        if isinstance(value, int) and not -2 ** 31 <= value < 2 ** (63 if name in _INT64 else 31):
            raise Unsupported(f"{name} = {value}")


def _pack(tokens=0, hq=0, hk=0, dim=0, rope=0, axes=1, interleaved=False, element=0, norm=False, eps=0.0, ps=0, pages=0,
          seqs=0, max_q=0, max_kv=0, max_pages=0, causal=False, window=0, scale=0.0, layers=0, page_bytes=0, rows=0) -> bytes:
    """A plan's sizes as the binding reads them (struct Sizes)."""
    return struct.pack("9qd8qd3q", tokens, hq, hk, dim, rope, axes, interleaved, element, norm, eps, ps, pages, seqs, max_q,
                       max_kv, max_pages, causal, window, scale, layers, page_bytes, rows)


# ---- norm and rotation -------------------------------------------------------
@dataclass(frozen=True)
class QkNormRopeDescriptor:
    tokens: int
    num_heads: int
    num_kv_heads: int
    head_dim: int
    rope_dim: int                      # the first values of a head, rotated; 0: none
    element: ElementKind = ElementKind.Bf16
    axes: int = 1                      # position axes
    interleaved: bool = False          # pairs (2i, 2i + 1) in place of (i, i + rope_dim / 2)
    eps: float = 1e-6
    norm: bool = True


class QkNormRopePlan:
    """q_out, k_out = rotate(x * w / sqrt(mean(x^2) + eps)) of each head, in one
    pass.  Statistics and products are held in 32 bits (in 64 for heads that leave
    their range) and rounded once; the outputs may be the inputs."""

    def __init__(self, desc: QkNormRopeDescriptor):
        d = self.desc = desc
        self._packed = _pack(d.tokens, d.num_heads, d.num_kv_heads, d.head_dim, d.rope_dim, d.axes, d.interleaved,
                             _element(d), d.norm, d.eps)

    @classmethod
    def select(cls, desc: QkNormRopeDescriptor) -> "QkNormRopePlan":
        _sizes_fit(desc)
        check(lib().qk_norm_rope_gfx950_can_implement(desc.tokens, desc.num_heads, desc.num_kv_heads, desc.head_dim,
                                                      desc.rope_dim, desc.axes, _element(desc)),
              "QkNormRopePlan::select")
        _need(desc.eps >= 0, "eps must not be negative")
        return cls(desc)

    def workspace_size(self) -> int:
        return 0

    def run(self, q, k, q_out, k_out, q_weight=None, k_weight=None, positions=None, cos=None, sin=None,
            pair_axis=None, stream=None) -> None:
        st = _kv4.qk_norm_rope(self._packed, stream, q, k, q_out, k_out, q_weight, k_weight, positions, cos, sin, pair_axis)
        if st:
            check(st, "QkNormRopePlan::run")


# ---- into the cache and back -------------------------------------------------
@dataclass(frozen=True)
class Kv4AppendDescriptor:
    tokens: int
    num_heads: int                     # of Q; 0: there is no Q
    num_kv_heads: int
    head_dim: int
    page_size: int
    num_pages: int
    rope_dim: int = 0
    element: ElementKind = ElementKind.Bf16
    axes: int = 1
    interleaved: bool = False
    eps: float = 1e-6
    norm: bool = True


class Kv4AppendPlan:
    """K (norm and rotation, rounded to the element) and V of new tokens into
    their slots of the cache, and Q's norm and rotation, in one pass.  K is
    computed in 64 bits, so that the codes are those of the exact values."""

    def __init__(self, desc: Kv4AppendDescriptor):
        d = self.desc = desc
        self._packed = _pack(d.tokens, d.num_heads, d.num_kv_heads, d.head_dim, d.rope_dim, d.axes, d.interleaved,
                             _element(d), d.norm, d.eps, ps=d.page_size, pages=d.num_pages)

    @classmethod
    def select(cls, desc: Kv4AppendDescriptor) -> "Kv4AppendPlan":
        _sizes_fit(desc)
        check(lib().kv4_append_gfx950_can_implement(desc.tokens, desc.num_heads, desc.num_kv_heads, desc.head_dim,
                                                    desc.rope_dim, desc.axes, _element(desc), desc.page_size,
                                                    desc.num_pages), "Kv4AppendPlan::select")
        _need(desc.eps >= 0, "eps must not be negative")
        return cls(desc)

    def workspace_size(self) -> int:
        return 0

    def run(self, k, v, cache, slots, q=None, q_out=None, q_weight=None, k_weight=None, positions=None, cos=None,
            sin=None, pair_axis=None, stream=None) -> None:
        st = _kv4.append(self._packed, stream, k, v, cache, slots, q, q_out, q_weight, k_weight, positions, cos, sin,
                         pair_axis)
        if st:
            check(st, "Kv4AppendPlan::run")


@dataclass(frozen=True)
class Kv4ReadDescriptor:
    tokens: int
    num_kv_heads: int
    head_dim: int
    page_size: int
    num_pages: int
    element: ElementKind = ElementKind.Bf16


class Kv4ReadPlan:
    """k_out, v_out [tokens, kv heads, D] = the values in the tokens' slots."""

    def __init__(self, desc: Kv4ReadDescriptor):
        d = self.desc = desc
        self._packed = _pack(d.tokens, 0, d.num_kv_heads, d.head_dim, element=_element(d), ps=d.page_size, pages=d.num_pages)

    @classmethod
    def select(cls, desc: Kv4ReadDescriptor) -> "Kv4ReadPlan":
        _sizes_fit(desc)
        check(lib().kv4_read_gfx950_can_implement(desc.tokens, desc.num_kv_heads, desc.head_dim, _element(desc),
                                                  desc.page_size, desc.num_pages), "Kv4ReadPlan::select")
        return cls(desc)

    def workspace_size(self) -> int:
        return 0

    def run(self, cache, slots, k_out, v_out, stream=None) -> None:
        st = _kv4.read(self._packed, stream, cache, slots, k_out, v_out)
        if st:
            check(st, "Kv4ReadPlan::run")


# ---- attention -----------------------------------------------------------------
@dataclass(frozen=True)
class Kv4AttentionDescriptor:
    num_seqs: int
    total_q: int                       # new tokens of all sequences
    max_q: int                         # ... of one at most
    max_kv: int                        # tokens of a sequence at most
    num_heads: int
    num_kv_heads: int
    head_dim: int
    page_size: int
    num_pages: int
    max_pages: int                     # columns of the tables
    element: ElementKind = ElementKind.Bf16
    causal: bool = True
    window: int = 0                    # positions that a row sees up to its own; 0: all
    scale: Optional[float] = None      # 1 / sqrt(head_dim)


class Kv4AttentionPlan:
    """softmax(scale q K^T + mask) V over the pages of each sequence, whose new
    tokens are its last ones.  `causal` hides what comes after a row's own
    position, `window` what lies that far or further before it.  A row that sees
    nothing gives zeros."""

    def __init__(self, desc: Kv4AttentionDescriptor):
        d = self.desc = desc
        self._packed = _pack(d.total_q, d.num_heads, d.num_kv_heads, d.head_dim, element=_element(d), ps=d.page_size,
                             pages=d.num_pages, seqs=d.num_seqs, max_q=d.max_q, max_kv=d.max_kv, max_pages=d.max_pages,
                             causal=d.causal, window=d.window, scale=self._sizes(d)[-1])

    @classmethod
    def select(cls, desc: Kv4AttentionDescriptor) -> "Kv4AttentionPlan":
        _sizes_fit(desc)
        check(lib().kv4_attention_gfx950_can_implement(*cls._sizes(desc)), "Kv4AttentionPlan::select")
        return cls(desc)

    @staticmethod
    def _sizes(d) -> list:
        scale = d.scale if d.scale is not None else max(d.head_dim, 1) ** -0.5
        return [d.num_seqs, d.total_q, d.max_q, d.max_kv, d.num_heads, d.num_kv_heads, d.head_dim, d.page_size,
                d.num_pages, d.max_pages, _element(d), int(d.causal), d.window, scale]

    def workspace_size(self) -> int:
        """Bytes that `run` needs beside its operands; what they hold does not matter."""
        d = self.desc
        return int(lib().kv4_attention_gfx950_workspace_size(d.num_seqs, d.max_q, d.max_kv, d.num_heads,
                                                             d.num_kv_heads, d.head_dim, d.window))

    def run(self, q, cache, tables, kv_lens, out, cu_q=None, workspace=None, stream=None) -> None:
        st = _kv4.attention(self._packed, stream, q, cache, tables, kv_lens, out, cu_q, workspace)
        if st:
            check(st, "Kv4AttentionPlan::run")


# ---- pages ---------------------------------------------------------------------
@dataclass(frozen=True)
class KvPagesDescriptor:
    layers: int
    num_pages: int
    page_bytes: int                    # of one layer
    page_size: int                     # tokens
    rows: int                          # sequences that the tables have room for
    max_pages: int                     # columns of the tables


class KvPagesPlan:
    """Pages of a cache [layers, pages, page bytes] whose layers share one table.

    tables int32 [rows, max_pages] holds each row's pages (-1: none), lens int32
    [rows] its tokens, refs int32 [pages] how many rows hold a page (0: free).
    All of it is on the device, and what a call does is decided there."""

    def __init__(self, desc: KvPagesDescriptor):
        d = self.desc = desc
        self._packed = _pack(layers=d.layers, pages=d.num_pages, page_bytes=d.page_bytes, ps=d.page_size, rows=d.rows,
                             max_pages=d.max_pages)

    @classmethod
    def select(cls, desc: KvPagesDescriptor) -> "KvPagesPlan":
        _sizes_fit(desc)
        check(lib().kv_pages_gfx950_can_implement(*cls._sizes(desc)), "KvPagesPlan::select")
        return cls(desc)

    @staticmethod
    def _sizes(d) -> list:
        return [d.layers, d.num_pages, d.page_bytes, d.page_size, d.rows, d.max_pages]

    def workspace_size(self) -> int:
        """Bytes that `compact` needs; the other calls need none."""
        return int(lib().kv_pages_gfx950_workspace_size(*self._sizes(self.desc)))

    def copy(self, cache, src, dst, stream=None) -> None:
        """Page src[i] to page dst[i] in every layer; no destination is a source
        or named twice.  Pairs outside the cache are left out."""
        st = _kv4.pages_copy(self._packed, stream, cache, src, dst)
        if st:
            check(st, "KvPagesPlan::copy")

    def fork(self, cache, tables, lens, refs, parents, children, fresh, stream=None) -> None:
        """Row children[i] becomes what row parents[i] is: full pages are shared, a
        partly filled last one is copied to the lowest free page, fresh[i] (-1:
        none was needed; -2, and an empty row: no page was free, or there is no
        such parent).  No child is a parent or holds pages before."""
        st = _kv4.pages_fork(self._packed, stream, cache, tables, lens, refs, parents, children, fresh)
        if st:
            check(st, "KvPagesPlan::fork")

    def release(self, tables, lens, refs, rows, stream=None) -> None:
        """The rows give their pages back and are empty after."""
        st = _kv4.pages_release(self._packed, stream, tables, lens, refs, rows)
        if st:
            check(st, "KvPagesPlan::release")

    def compact(self, cache, tables, refs, tables_out, refs_out, remap, live, workspace=None, stream=None) -> None:
        """The pages in use move to the front, where live[0] of them lie after:
        the ones past that, lowest first, into the free ones before it, lowest
        first.  remap: each page's new place, -1 for a free one.  tables_out may be
        tables; refs_out is not refs."""
        st = _kv4.pages_compact(self._packed, stream, cache, tables, refs, tables_out, refs_out, remap, live, workspace)
        if st:
            check(st, "KvPagesPlan::compact")


__all__ = ["QkNormRopeDescriptor", "QkNormRopePlan", "Kv4AppendDescriptor", "Kv4AppendPlan", "Kv4ReadDescriptor",
           "Kv4ReadPlan", "Kv4AttentionDescriptor", "Kv4AttentionPlan", "KvPagesDescriptor", "KvPagesPlan", "head_bytes",
           "InvalidProblem", "Unsupported"]
