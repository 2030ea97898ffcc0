"""A key-value cache held in 4 bits: what fills it, attention over it, its pages.

  QkNormRopePlan    RMS norm of each head of Q and K and the position rotation
  Kv4AppendPlan     the same, and K and V quantized into pages of the cache
  Kv4ReadPlan       the values that slots of the cache stand for
  Kv4AttentionPlan  attention of a ragged batch over its pages
  KvPagesPlan       copying, forking, releasing and compacting pages

No counterpart in the reference.  The manner is that of ``plans``: ``select`` a
plan for a descriptor, ``run`` it on a stream (torch's current one by default);
``run`` neither allocates nor synchronises, so it can be captured into a graph,
and errors are the exceptions of ``plans``.

The cache is a uint8 tensor [pages, kv heads, kv4.head_bytes(page size, D)], two
codes a byte (sign, two exponent bits, one mantissa bit); 32 values share a
power of two.  include/baracuda_kernels.h describes its bytes.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .ffi import lib
from .plans import ElementKind, InvalidProblem, Unsupported, _nbytes, _need, _ptr, _stream, check

_TAG = {ElementKind.F32: 0, ElementKind.F16: 1, ElementKind.Bf16: 2}
_DTYPE = {ElementKind.F32: torch.float32, ElementKind.F16: torch.float16, ElementKind.Bf16: torch.bfloat16}


def head_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one head of one page."""
    return page_size * (head_dim + head_dim // 16)


def _element(desc) -> int:
    if desc.element not in _TAG:
        raise Unsupported(f"element {desc.element}: F32, F16 or Bf16")
    return _TAG[desc.element]


def _heads(t: Optional[torch.Tensor], tokens: int, heads: int, dim: int, dtype, what: str) -> None:
    _need(t is not None, f"{what} is required")
    _need(tuple(t.shape) == (tokens, heads, dim) and t.dtype == dtype,
          f"{what} must be {dtype} [{tokens}, {heads}, {dim}]")
    _need(dim <= 1 or t.stride(2) == 1, f"{what}: the values of a head must be dense")


def _out(t: torch.Tensor, what: str) -> None:
    """An output whose elements are all in places of their own."""
    t0, t1, dim = t.stride(0), t.stride(1), t.shape[2]
    dense = (t.shape[1] <= 1 or t1 >= dim) and (t.shape[0] <= 1 or t0 >= (t.shape[1] - 1) * t1 + dim)
    heads_first = t.shape[0] <= 1 or (t0 >= dim and (t.shape[1] <= 1 or t1 >= (t.shape[0] - 1) * t0 + dim))
    _need(t.numel() == 0 or dense or heads_first, f"{what}: rows must not overlap")


def _ints(t: Optional[torch.Tensor], shape: tuple, what: str, dtype=torch.int32) -> None:
    _need(t is not None, f"{what} is required")
    _need(tuple(t.shape) == shape and t.dtype == dtype and t.is_contiguous(),
          f"{what} must be contiguous {dtype} {list(shape)}")


def _row(t: torch.Tensor) -> tuple:
    return t.stride(0), t.stride(1)


def _one_device(*tensors) -> None:
    """All operands on one GPU; the launch goes to that GPU's stream."""
    found = {t.device for t in tensors if t is not None and t.is_cuda}
    _need(len(found) <= 1, "operands must be on one GPU")


def _rotation(d, q_weight, k_weight, positions, cos, sin, pair_axis) -> list:
    """Checks and C arguments of the norms' weights and the rotation's table."""
    dtype = _DTYPE[d.element]
    if d.norm:
        for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            _ints(w, (d.head_dim,), what, dtype)
    else:
        _need(q_weight is None and k_weight is None, "a descriptor without norm takes no weights")
    if not d.rope_dim:
        _need(positions is None and cos is None and sin is None and pair_axis is None,
              "a descriptor without rope_dim takes no rotation")
        return [_ptr(q_weight), _ptr(k_weight), None, None, None, 0, None]
    if positions is not None and positions.dim() == 1 and d.axes == 1:
        positions = positions.unsqueeze(0)
    _ints(positions, (d.axes, d.tokens), "positions")
    for t, what in ((cos, "cos"), (sin, "sin")):
        _need(t is not None, f"{what} is required")
        _need(t.dim() == 2 and t.shape[1] == d.rope_dim // 2 and t.dtype == torch.float32 and t.is_contiguous(),
              f"{what} must be contiguous f32 [positions, rope_dim / 2]")
    _need(cos.shape == sin.shape and cos.shape[0] > 0, "cos and sin must have the same rows")
    if d.axes > 1:
        _ints(pair_axis, (d.rope_dim // 2,), "pair_axis")
    else:
        _need(pair_axis is None, "one axis takes no pair_axis")
    return [_ptr(q_weight), _ptr(k_weight), _ptr(positions), _ptr(cos), _ptr(sin), cos.shape[0], _ptr(pair_axis)]


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
    pass.  Statistics and products are held in 32 bits and rounded once; the
    outputs may be the inputs."""

    def __init__(self, desc: QkNormRopeDescriptor):
        self.desc = desc

    @classmethod
    def select(cls, desc: QkNormRopeDescriptor) -> "QkNormRopePlan":
        check(lib().qk_norm_rope_gfx950_can_implement(desc.tokens, desc.num_heads, desc.num_kv_heads, desc.head_dim,
                                                      desc.rope_dim, desc.axes, _element(desc)),
              "QkNormRopePlan::select")
        _need(desc.eps >= 0, "eps must not be negative")
        return cls(desc)

    def workspace_size(self) -> int:
        return 0

    def run(self, q, k, q_out, k_out, q_weight=None, k_weight=None, positions=None, cos=None, sin=None,
            pair_axis=None, stream=None) -> None:
        d = self.desc
        dtype = _DTYPE[d.element]
        for t, n, what in ((q, d.num_heads, "q"), (q_out, d.num_heads, "q_out"), (k, d.num_kv_heads, "k"),
                           (k_out, d.num_kv_heads, "k_out")):
            _heads(t, d.tokens, n, d.head_dim, dtype, what)
        _out(q_out, "q_out")
        _out(k_out, "k_out")
        _one_device(q, k, q_out, k_out, q_weight, k_weight, positions, cos, sin, pair_axis)
        rot = _rotation(d, q_weight, k_weight, positions, cos, sin, pair_axis)
        check(lib().qk_norm_rope_gfx950_run(
            d.tokens, d.num_heads, d.num_kv_heads, d.head_dim, d.rope_dim, d.axes, int(d.interleaved), _TAG[d.element],
            d.eps, _ptr(q), *_row(q), _ptr(k), *_row(k), _ptr(q_out), *_row(q_out), _ptr(k_out), *_row(k_out), *rot,
            _stream(stream)), "QkNormRopePlan::run")


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


def _check_cache(cache, d) -> None:
    _need(cache is not None and cache.dtype == torch.uint8 and cache.is_contiguous() and tuple(cache.shape) ==
          (d.num_pages, d.num_kv_heads, head_bytes(d.page_size, d.head_dim)),
          f"cache must be contiguous uint8 [{d.num_pages}, {d.num_kv_heads}, {head_bytes(d.page_size, d.head_dim)}]")


class Kv4AppendPlan:
    """K (norm and rotation, rounded to the element) and V of new tokens into
    their slots of the cache, and Q's norm and rotation, in one pass.  K is
    computed in 64 bits, so that the codes are those of the exact values."""

    def __init__(self, desc: Kv4AppendDescriptor):
        self.desc = desc

    @classmethod
    def select(cls, desc: Kv4AppendDescriptor) -> "Kv4AppendPlan":
        check(lib().kv4_append_gfx950_can_implement(desc.tokens, desc.num_heads, desc.num_kv_heads, desc.head_dim,
                                                    desc.rope_dim, desc.axes, _element(desc), desc.page_size,
                                                    desc.num_pages), "Kv4AppendPlan::select")
        _need(desc.eps >= 0, "eps must not be negative")
        return cls(desc)

    def workspace_size(self) -> int:
        return 0

    def run(self, k, v, cache, slots, q=None, q_out=None, q_weight=None, k_weight=None, positions=None, cos=None,
            sin=None, pair_axis=None, stream=None) -> None:
        d = self.desc
        dtype = _DTYPE[d.element]
        _heads(k, d.tokens, d.num_kv_heads, d.head_dim, dtype, "k")
        _heads(v, d.tokens, d.num_kv_heads, d.head_dim, dtype, "v")
        if d.num_heads:
            _heads(q, d.tokens, d.num_heads, d.head_dim, dtype, "q")
            _heads(q_out, d.tokens, d.num_heads, d.head_dim, dtype, "q_out")
            _out(q_out, "q_out")
        else:
            _need(q is None and q_out is None, "a descriptor without query heads takes no q")
        _check_cache(cache, d)
        _ints(slots, (d.tokens,), "slots", torch.int64)
        _one_device(q, k, v, q_out, cache, slots, q_weight, k_weight, positions, cos, sin, pair_axis)
        rot = _rotation(d, q_weight, k_weight, positions, cos, sin, pair_axis)
        none = (0, 0)
        check(lib().kv4_append_gfx950_run(
            d.tokens, d.num_heads, d.num_kv_heads, d.head_dim, d.rope_dim, d.axes, int(d.interleaved), _TAG[d.element],
            d.eps, d.page_size, d.num_pages, _ptr(q), *(none if q is None else _row(q)), _ptr(k), *_row(k), _ptr(v),
            *_row(v), _ptr(q_out), *(none if q_out is None else _row(q_out)), _ptr(cache), _ptr(slots), *rot,
            _stream(stream)), "Kv4AppendPlan::run")


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
        self.desc = desc

    @classmethod
    def select(cls, desc: Kv4ReadDescriptor) -> "Kv4ReadPlan":
        check(lib().kv4_read_gfx950_can_implement(desc.tokens, desc.num_kv_heads, desc.head_dim, _element(desc),
                                                  desc.page_size, desc.num_pages), "Kv4ReadPlan::select")
        return cls(desc)

    def workspace_size(self) -> int:
        return 0

    def run(self, cache, slots, k_out, v_out, stream=None) -> None:
        d = self.desc
        for t, what in ((k_out, "k_out"), (v_out, "v_out")):
            _heads(t, d.tokens, d.num_kv_heads, d.head_dim, _DTYPE[d.element], what)
            _out(t, what)
        _check_cache(cache, d)
        _ints(slots, (d.tokens,), "slots", torch.int64)
        _one_device(cache, slots, k_out, v_out)
        check(lib().kv4_read_gfx950_run(d.tokens, d.num_kv_heads, d.head_dim, _TAG[d.element], d.page_size, d.num_pages,
                                        _ptr(cache), _ptr(slots), _ptr(k_out), *_row(k_out), _ptr(v_out), *_row(v_out),
                                        _stream(stream)), "Kv4ReadPlan::run")


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
    window: int = 0                    # 0: none
    scale: Optional[float] = None      # 1 / sqrt(head_dim)


class Kv4AttentionPlan:
    """softmax(scale q K^T + mask) V over the pages of each sequence, whose new
    tokens are its last ones.  A row that sees nothing gives zeros."""

    def __init__(self, desc: Kv4AttentionDescriptor):
        self.desc = desc

    @classmethod
    def select(cls, desc: Kv4AttentionDescriptor) -> "Kv4AttentionPlan":
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
        d = self.desc
        _heads(q, d.total_q, d.num_heads, d.head_dim, _DTYPE[d.element], "q")
        _heads(out, d.total_q, d.num_heads, d.head_dim, _DTYPE[d.element], "out")
        _out(out, "out")
        _check_cache(cache, d)
        _need(tables is not None and tuple(tables.shape) == (d.num_seqs, d.max_pages) and tables.dtype == torch.int32
              and (d.max_pages <= 1 or tables.stride(1) == 1), f"tables must be int32 [{d.num_seqs}, {d.max_pages}]")
        _ints(kv_lens, (d.num_seqs,), "kv_lens")
        if cu_q is not None:
            _ints(cu_q, (d.num_seqs + 1,), "cu_q")
        else:
            _need(d.max_q == 1 and d.total_q == d.num_seqs, "cu_q is required unless every sequence has one new token")
        _need(workspace is None or workspace.is_contiguous(), "workspace must be contiguous")
        _one_device(q, cache, tables, kv_lens, out, cu_q, workspace)
        check(lib().kv4_attention_gfx950_run(
            *self._sizes(d), _ptr(q), *_row(q), _ptr(cache), _ptr(tables), tables.stride(0), _ptr(kv_lens), _ptr(cu_q),
            _ptr(out), *_row(out), _ptr(workspace), _nbytes(workspace), _stream(stream)), "Kv4AttentionPlan::run")


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
        self.desc = desc

    @classmethod
    def select(cls, desc: KvPagesDescriptor) -> "KvPagesPlan":
        check(lib().kv_pages_gfx950_can_implement(*cls._sizes(desc)), "KvPagesPlan::select")
        return cls(desc)

    @staticmethod
    def _sizes(d) -> list:
        return [d.layers, d.num_pages, d.page_bytes, d.page_size, d.rows, d.max_pages]

    def workspace_size(self) -> int:
        """Bytes that `compact` needs; the other calls need none."""
        return int(lib().kv_pages_gfx950_workspace_size(*self._sizes(self.desc)))

    def _cache(self, cache) -> None:
        d = self.desc
        _need(cache is not None and cache.is_contiguous() and cache.element_size() == 1 and
              tuple(cache.shape) == (d.layers, d.num_pages, d.page_bytes),
              f"cache must be contiguous bytes [{d.layers}, {d.num_pages}, {d.page_bytes}]")

    def _state(self, tables, lens, refs) -> None:
        d = self.desc
        _ints(tables, (d.rows, d.max_pages), "tables")
        if lens is not None:
            _ints(lens, (d.rows,), "lens")
        _ints(refs, (d.num_pages,), "refs")

    def copy(self, cache, src, dst, stream=None) -> None:
        """Page src[i] to page dst[i] in every layer; no destination is a source
        or named twice.  Pairs outside the cache are left out."""
        d = self.desc
        self._cache(cache)
        _need(src is not None and src.dim() == 1, "src must be a vector")
        _ints(src, (src.numel(),), "src")
        _ints(dst, (src.numel(),), "dst")
        _one_device(cache, src, dst)
        check(lib().kv_pages_copy_gfx950_run(d.layers, d.num_pages, d.page_bytes, src.numel(), _ptr(cache), _ptr(src),
                                             _ptr(dst), _stream(stream)), "KvPagesPlan::copy")

    def fork(self, cache, tables, lens, refs, parents, children, fresh, stream=None) -> None:
        """Row children[i] becomes what row parents[i] is: full pages are shared, a
        partly filled last one is copied to the lowest free page, fresh[i] (-1:
        none was needed; -2, and an empty row: no page was free, or there is no
        such parent).  No child is a parent or holds pages before."""
        self._cache(cache)
        self._state(tables, lens, refs)
        _need(lens is not None, "lens is required")
        _need(parents is not None and parents.dim() == 1, "parents must be a vector")
        n = parents.numel()
        for t, what in ((parents, "parents"), (children, "children"), (fresh, "fresh")):
            _ints(t, (n,), what)
        _one_device(cache, tables, lens, refs, parents, children, fresh)
        check(lib().kv_pages_fork_gfx950_run(*self._sizes(self.desc), n, _ptr(cache), _ptr(tables), _ptr(lens), _ptr(refs),
                                             _ptr(parents), _ptr(children), _ptr(fresh), _stream(stream)),
              "KvPagesPlan::fork")

    def release(self, tables, lens, refs, rows, stream=None) -> None:
        """The rows give their pages back and are empty after."""
        d = self.desc
        self._state(tables, lens, refs)
        _need(lens is not None, "lens is required")
        _need(rows is not None and rows.dim() == 1, "rows must be a vector")
        _ints(rows, (rows.numel(),), "rows")
        _one_device(tables, lens, refs, rows)
        check(lib().kv_pages_release_gfx950_run(d.num_pages, d.rows, d.max_pages, rows.numel(), _ptr(tables), _ptr(lens),
                                                _ptr(refs), _ptr(rows), _stream(stream)), "KvPagesPlan::release")

    def compact(self, cache, tables, refs, tables_out, refs_out, remap, live, workspace=None, stream=None) -> None:
        """The pages in use move to the front, where live[0] of them lie after:
        the ones past that, lowest first, into the free ones before it, lowest
        first.  remap: each page's new place, -1 for a free one.  tables_out may be
        tables; refs_out is not refs."""
        d = self.desc
        self._cache(cache)
        self._state(tables, None, refs)
        self._state(tables_out, None, refs_out)
        _ints(remap, (d.num_pages,), "remap")
        _ints(live, (1,), "live")
        _need(refs.data_ptr() != refs_out.data_ptr(), "refs_out must not be refs")
        _need(workspace is None or workspace.is_contiguous(), "workspace must be contiguous")
        _one_device(cache, tables, refs, tables_out, refs_out, remap, live, workspace)
        check(lib().kv_pages_compact_gfx950_run(*self._sizes(d), _ptr(cache), _ptr(tables), _ptr(refs), _ptr(tables_out),
                                                _ptr(refs_out), _ptr(remap), _ptr(live), _ptr(workspace),
                                                _nbytes(workspace), _stream(stream)), "KvPagesPlan::compact")


__all__ = ["QkNormRopeDescriptor", "QkNormRopePlan", "Kv4AppendDescriptor", "Kv4AppendPlan", "Kv4ReadDescriptor",
           "Kv4ReadPlan", "Kv4AttentionDescriptor", "Kv4AttentionPlan", "KvPagesDescriptor", "KvPagesPlan", "head_bytes",
           "InvalidProblem", "Unsupported"]
