"""Host side of the attention between the QKV and the output projection: the
paged key / value cache's writer and its single-token reader (the attention
section of include/lunaflux_fp8.h).

The plan vocabulary's RotaryEmbedding and CausalAttention (lunaflux_amd/plan.py)
cut the work elsewhere: there the attention appends to the cache and takes prompt
rows too, and the catalog has no entry for either. These operations read the same
runtime inputs of a paged step and are bound beside the plan's projections:

  bind_qk_norm_rope   per-head norm of queries and keys, rotary positions of
                      one or several axes, append of the step's keys and values
  bind_paged_decode   attention of one new token per sequence, split over the
                      cache's length and joined

over regions that stay where they are from step to step: `AttentionLayer`
holds the layer's constants, `PagedStep` the step's runtime inputs, which
`stage` rewrites.
"""
from __future__ import annotations

import ctypes
import math
from array import array
from dataclasses import dataclass

import numpy as np

from . import _abi
from .device import Allocation, DeviceError, KernelArgument, KernelArguments, KernelLaunchDimensions
from .fp8 import COUNTS_BYTES, BoundOperation, LaunchStep, ProjectionRuntime, _region

CACHES = {"bf16": _abi.LF_FP8_CACHE_BF16, "e4m3": _abi.LF_FP8_CACHE_E4M3}
PAIRINGS = {"half": _abi.LF_FP8_PAIR_HALF, "neighbour": _abi.LF_FP8_PAIR_NEIGHBOUR}
MAX_SEQUENCES = _abi.LF_FP8_ATTN_MAX_SEQUENCES
AS_THEY_ARE = object()  # PagedStep.stage: the positions that the region holds


class AttentionDescriptor(ctypes.Structure):
    """lf_fp8_attn_desc."""

    _fields_ = [("magic", ctypes.c_uint32), ("query_heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("cache", ctypes.c_int32), ("page_size", ctypes.c_int32),
                ("pages", ctypes.c_int32), ("max_tokens", ctypes.c_int32), ("max_sequences", ctypes.c_int32),
                ("table_entries", ctypes.c_int32), ("window", ctypes.c_int32), ("rotary_dim", ctypes.c_int32),
                ("axes", ctypes.c_int32), ("pairing", ctypes.c_int32), ("norm", ctypes.c_int32),
                ("norm_epsilon", ctypes.c_float), ("softmax_scale", ctypes.c_float), ("reserved", ctypes.c_int32),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("scale_offset", ctypes.c_int64), ("turns_offset", ctypes.c_int64), ("axis_offset", ctypes.c_int64),
                ("region_bytes", ctypes.c_int64), ("padding", ctypes.c_uint8 * 128)]


def _check(operation, status):
    if status != _abi.LF_OK:
        raise DeviceError(operation, status)


def _invalid(what: str):
    return DeviceError(what, _abi.LF_INVALID_ARGUMENT)


@dataclass(frozen=True)
class Rotary:
    """The rotation of a head's first 2 len(turns) values: pair i turns by
    2 pi position[axis[i]] turns[i]. pairing: "half" (i with i + len(turns)) or
    "neighbour" (2 i with 2 i + 1)."""

    turns: np.ndarray
    axis: np.ndarray
    pairing: str = "half"
    axes: int = 0  # positions of a row; 0: as many as `axis` names

    def __post_init__(self):
        turns, given = np.asarray(self.turns, np.float64), np.asarray(self.axis)
        if turns.ndim != 1 or given.shape != turns.shape or self.pairing not in PAIRINGS:
            raise _invalid("rotary pairs")
        if given.dtype.kind not in "iuf" or not (np.abs(given.astype(np.float64)) < 2 ** 31).all() or \
                (given != given.astype(np.int32)).any():
            raise _invalid("axes of rotary pairs are whole numbers")
        axis = given.astype(np.int32)
        object.__setattr__(self, "turns", turns)
        object.__setattr__(self, "axis", axis)
        if self.axes == 0:
            object.__setattr__(self, "axes", int(axis.max(initial=0)) + 1)

    @staticmethod
    def of_theta(theta: float, dim: int, sections=None, pairing: str = "half") -> "Rotary":
        """theta^(-2 i / dim) radians per position for pair i. sections: pairs
        of each axis in turn (time, height, width; they add up to dim / 2)."""
        if not isinstance(dim, (int, np.integer)) or dim < 0 or dim % 2:
            raise _invalid("rotary dimensions")
        dim = int(dim)
        pairs = dim // 2
        sections = [pairs] if sections is None else list(sections)
        if sum(sections) != pairs or min(sections) < 0:
            raise _invalid("rotary sections")
        turns = float(theta) ** (-np.arange(pairs, dtype=np.float64) * 2.0 / dim) / (2.0 * math.pi)
        return Rotary(turns, np.repeat(np.arange(len(sections)), sections), pairing, len(sections))


@dataclass
class AttentionLayer:
    """A layer's constants on the device: the descriptor region."""

    desc: AttentionDescriptor
    allocation: Allocation

    @property
    def region(self) -> KernelArgument:
        return _region(self.allocation, alignment=256)

    @property
    def cache_bytes(self) -> int:
        """Bytes the key cache spans, and the value cache."""
        return _abi.lib().lunaflux_fp8_attn_cache_bytes(ctypes.byref(self.desc))


def attention_descriptor(*, query_heads: int, kv_heads: int, head_dim: int, page_size: int, pages: int,
                         max_tokens: int, max_sequences: int, table_entries: int, cache: str = "bf16",
                         rotary: Rotary | None = None, norm_epsilon: float | None = None,
                         softmax_scale: float | None = None, window: int = 0, strides=None) -> AttentionDescriptor:
    """lunaflux_fp8_attn_descriptor. norm_epsilon None: heads are not
    normalized; softmax_scale None: 1 / sqrt(head_dim); strides: (page, head,
    token) strides of the caches in elements, None: [page][head][token]."""
    if cache not in CACHES:
        raise ValueError(f"unknown cache type {cache!r}; expected one of {tuple(CACHES)}")
    d = AttentionDescriptor()
    try:
        d.query_heads, d.kv_heads, d.head_dim, d.cache = query_heads, kv_heads, head_dim, CACHES[cache]
        d.page_size, d.pages, d.max_tokens, d.max_sequences = page_size, pages, max_tokens, max_sequences
        d.table_entries, d.window = table_entries, window
        for name, value in (("query_heads", query_heads), ("kv_heads", kv_heads), ("head_dim", head_dim),
                            ("page_size", page_size), ("pages", pages), ("max_tokens", max_tokens),
                            ("max_sequences", max_sequences), ("table_entries", table_entries), ("window", window)):
            if getattr(d, name) != value:  # ctypes cuts to 32 bits
                raise _invalid(name)
        d.rotary_dim = 0 if rotary is None else 2 * len(rotary.turns)
        d.axes = 1 if rotary is None else rotary.axes
        if rotary is not None and d.axes != rotary.axes:
            raise _invalid("axes")
        d.pairing = PAIRINGS["half" if rotary is None else rotary.pairing]
        d.norm, d.norm_epsilon = (0, 0.0) if norm_epsilon is None else (1, norm_epsilon)
        d.softmax_scale = 1.0 / math.sqrt(head_dim) if softmax_scale is None and head_dim > 0 else softmax_scale or 0.0
        steps = (0, 0, 0) if strides is None else tuple(strides)
        if len(steps) != 3:
            raise _invalid("strides")
        d.page_stride, d.head_stride, d.token_stride = steps
        if (d.page_stride, d.head_stride, d.token_stride) != steps:
            raise _invalid("strides")
    except TypeError as e:
        raise _invalid(str(e)) from None
    _check("attention_descriptor", _abi.lib().lunaflux_fp8_attn_descriptor(ctypes.byref(d)))
    return d


def descriptor_region(desc: AttentionDescriptor, k_scales=None, v_scales=None, rotary: Rotary | None = None) -> np.ndarray:
    """The bytes of the descriptor region (lunaflux_fp8_attn_region)."""
    scales = None
    if (k_scales is None) != (v_scales is None):
        raise _invalid("cache scales")
    if k_scales is not None:
        scales = np.concatenate([np.asarray(k_scales, np.float32).reshape(-1), np.asarray(v_scales, np.float32).reshape(-1)])
        if np.size(k_scales) != np.size(v_scales):
            raise _invalid("cache scales")
    turns = np.zeros(0, np.float64) if rotary is None else np.ascontiguousarray(rotary.turns)
    axis = np.zeros(0, np.int32) if rotary is None else np.ascontiguousarray(rotary.axis)
    region = np.empty(max(int(desc.region_bytes), 0), np.uint8)
    _check("attention_region", _abi.lib().lunaflux_fp8_attn_region(
        ctypes.byref(desc), None if scales is None else scales.ctypes.data_as(ctypes.POINTER(ctypes.c_float)),
        0 if scales is None else scales.size, turns.ctypes.data_as(ctypes.POINTER(ctypes.c_double)),
        axis.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), turns.size,
        region.ctypes.data_as(ctypes.POINTER(ctypes.c_uint8)), region.size))
    return region


def attention_layer(rt: ProjectionRuntime, *, k_scales=None, v_scales=None, rotary: Rotary | None = None,
                    **fields) -> AttentionLayer:
    """Checks a layer's constants (attention_descriptor) and uploads them. An
    e4m3 cache takes fp32 scales per key head (value = code * scale)."""
    desc = attention_descriptor(rotary=rotary, **fields)
    return AttentionLayer(desc, rt.context.upload(descriptor_region(desc, k_scales, v_scales, rotary)))


def workspace_bytes(entry: int, desc: AttentionDescriptor) -> int:
    n = _abi.lib().lunaflux_fp8_attn_workspace_bytes(entry, ctypes.byref(desc))
    if n < 0:
        raise _invalid("attention_workspace_bytes")
    return n


def launch_geometry(entry: int, desc: AttentionDescriptor):
    dims = (ctypes.c_int32 * 7)()
    symbol = ctypes.create_string_buffer(128)
    _check("attention_launch_geometry", _abi.lib().lunaflux_fp8_attn_launch_geometry(
        entry, ctypes.byref(desc), dims, symbol))
    return (KernelLaunchDimensions.new(tuple(dims[0:3]), tuple(dims[3:6]), dims[6]),
            symbol.value.decode("ascii"))


def _page_table(table) -> np.ndarray:
    if isinstance(table, list):
        try:
            return np.asarray(array("i", table))  # C ints from Python's, the quickest way that changes none
        except (TypeError, OverflowError):
            pass
    return np.asarray(table).reshape(-1)


def _page_tables(page_tables) -> tuple:
    """The number of entries of every sequence's table, and all of them in turn as int32."""
    tables = [_page_table(t) for t in page_tables]
    counts = np.array([t.size for t in tables], np.int64)
    held = [t for t in tables if t.size] or [np.zeros(0, np.int32)]
    kinds = {t.dtype for t in held}
    if any(k.kind not in "iu" for k in kinds):
        raise _invalid("page indices are whole numbers")
    if len(kinds) > 1:  # types that differ may become a float one, or wrap
        held = [t.astype(np.int64) if t.dtype != np.uint64 or t.max() < 2 ** 31 else np.array([2 ** 31]) for t in held]
    indices = np.concatenate(held)
    if indices.dtype != np.int32:
        if indices.min() < -2 ** 31 or indices.max() >= 2 ** 31:
            raise _invalid("page indices are of 32 bits")
        indices = indices.astype(np.int32)
    return counts, indices


class PagedStep:
    """The runtime inputs of a paged step, in regions sized for the layer's
    descriptor (max_tokens rows, max_sequences, table_entries); every layer of
    a model reads the same ones."""

    def __init__(self, rt: ProjectionRuntime, layer: AttentionLayer):
        d = layer.desc
        self.max_tokens, self.max_sequences, self.table_entries = d.max_tokens, d.max_sequences, d.table_entries
        self.axes, self.page_size = d.axes, d.page_size
        self.positioned = True  # the step's rows have positions
        allocate = rt.context.allocate
        self.counts = allocate(COUNTS_BYTES)
        self.positions = allocate(4 * d.max_tokens * d.axes)
        self.row_offsets = allocate(4 * (d.max_sequences + 1))
        self.lengths = allocate(4 * d.max_sequences)
        self.page_offsets = allocate(4 * (d.max_sequences + 1))
        self.page_indices = allocate(4 * d.table_entries)
        self.stage([0], [], [], np.zeros((0, d.axes), np.int32))

    def stage(self, row_offsets, lengths, page_tables, positions=None, prefill_rows: int = 0):
        """Writes a step's inputs. Sequence s has rows row_offsets[s] ..
        row_offsets[s + 1] - 1 and, with them, lengths[s] tokens in the pages
        page_tables[s]; the first prefill_rows sequences are not decoded.
        positions [rows, axes] (or [rows] for one axis); None: the rows have
        none, and appends of layers that rotate refuse to launch; AS_THEY_ARE:
        those that the caller wrote to `positions`, or left there by the step
        before. DeviceError INVALID_ARGUMENT, with nothing written, for a
        step that does not fit or contradicts itself (page indices, of any
        integer type, are the cache owner's and checked on the device). Launches
        that read the step before have to be over: the caller synchronizes their
        streams first. Six copies to the device, one after another: 0.11 ms for
        a few sequences, 0.12 for 32 of 145 pages, 0.7 for 2048 of 16."""
        row_offsets, lengths = np.asarray(row_offsets), np.asarray(lengths)
        n = lengths.size
        for a in (row_offsets, lengths):
            if a.size and (a.ndim != 1 or a.dtype.kind not in "iu"):
                raise _invalid("a step's offsets and lengths are whole numbers in one dimension")
        if row_offsets.size != n + 1 or n > self.max_sequences or len(page_tables) != n or not 0 <= prefill_rows <= n:
            raise _invalid("sequences of a step")
        row_offsets, lengths = row_offsets.astype(np.int64), lengths.astype(np.int64)
        rows = np.diff(row_offsets)
        if row_offsets[0] != 0 or (rows < 0).any() or row_offsets[-1] > self.max_tokens:
            raise _invalid("rows of a step")
        if (rows[prefill_rows:] != 1).any():
            raise _invalid("a decoded sequence has one row")
        if (lengths < rows).any():
            raise _invalid("lengths of a step")
        counts, indices = _page_tables(page_tables)
        if (counts * self.page_size < lengths).any() or counts.sum() > self.table_entries:
            raise _invalid("page tables of a step")
        m = int(row_offsets[-1])
        written = positions is not None and positions is not AS_THEY_ARE
        if written:
            positions = np.asarray(positions)
            if positions.dtype.kind not in "iu" or positions.size != m * self.axes or \
                    positions.shape not in ((m,), (m, self.axes)):
                raise _invalid("positions of a step")
            if positions.size and (positions.min() < -2 ** 31 or positions.max() >= 2 ** 31):
                raise _invalid("positions of a step")
        if lengths.size and lengths.max() >= 2 ** 31:
            raise _invalid("lengths of a step")
        self.counts.copy_from_host(np.array([prefill_rows, n - prefill_rows, n, m, indices.size], np.int32))
        self.row_offsets.copy_from_host(row_offsets.astype(np.int32))
        self.lengths.copy_from_host(lengths.astype(np.int32))
        self.page_offsets.copy_from_host(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        if indices.size:
            self.page_indices.copy_from_host(indices)
        if written:
            self.positions.copy_from_host(positions.astype(np.int32))
        self.positioned = positions is not None or m == 0


@dataclass
class BoundAttention(BoundOperation):
    """check(): DeviceError(INVALID_ARGUMENT) if a launch met offsets, lengths
    or page indices outside the layer's bounds (the rows and keys concerned
    were left out); the error word is cleared. After asynchronous launches the
    caller synchronizes the stream first.

    rotates: the step whose positions the operation turns by, or None."""

    rotates: PagedStep | None = None

    def launch(self, stream, synchronous: bool = True):
        if self.rotates is not None and not self.rotates.positioned:
            raise _invalid("rows of the step have no positions to be rotated by")
        super().launch(stream, synchronous)

    def check(self):
        if self.workspace.read(np.int32, (1,))[0] != 0:
            self.workspace.copy_from_host(np.zeros(1, np.int32))
            raise DeviceError("a paged step left the bounds of its cache or descriptor", _abi.LF_INVALID_ARGUMENT)


def _holds(what: str, region: KernelArgument, byte_count: int):
    if region.byte_count < byte_count or region.alignment < 16:
        raise _invalid(f"{what}: {byte_count} bytes aligned to 16 are wanted")


def _apart(what: str, written, read):
    """Refuses regions of one allocation that overlap, one of them written."""
    for i, p in enumerate(written):
        for q in (*written[:i], *read):
            if p.allocation is q.allocation and p.offset < q.offset + q.byte_count and q.offset < p.offset + p.byte_count:
                raise _invalid(f"{what} overlap")


def _step_fits(layer: AttentionLayer, step: PagedStep):
    d = layer.desc
    if (step.max_tokens, step.max_sequences, step.table_entries, step.page_size) != \
            (d.max_tokens, d.max_sequences, d.table_entries, d.page_size) or step.axes != d.axes:
        raise _invalid("the step was made for another descriptor")


def _workspace(rt: ProjectionRuntime, entry: int, desc: AttentionDescriptor) -> Allocation:
    nbytes = workspace_bytes(entry, desc)
    ws = rt.context.allocate(nbytes)
    ws.copy_from_host(np.zeros(nbytes, np.uint8))
    return ws


def bind_qk_norm_rope(rt: ProjectionRuntime, layer: AttentionLayer, step: PagedStep, qkv: KernelArgument,
                      gq: KernelArgument | None, gk: KernelArgument | None, q: KernelArgument,
                      k_cache: KernelArgument, v_cache: KernelArgument) -> BoundAttention:
    """Packed rows qkv [max_tokens, Hq + 2 Hkv, D] (a QKV projection's output)
    to rotated queries q [max_tokens, Hq, D] and, in the cache, keys and values
    of every row of the step. gq, gk: the norm weights [D], given if and only if
    the layer normalizes its heads. q and the caches may overlap neither each
    other nor what is read."""
    d = layer.desc
    _step_fits(layer, step)
    heads = d.query_heads + 2 * d.kv_heads
    _holds("qkv", qkv, 2 * d.max_tokens * heads * d.head_dim)
    _holds("q", q, 2 * d.max_tokens * d.query_heads * d.head_dim)
    _holds("k_cache", k_cache, layer.cache_bytes)
    _holds("v_cache", v_cache, layer.cache_bytes)
    if (gq is None) != (d.norm == 0) or (gk is None) != (d.norm == 0):
        raise _invalid("norm weights")
    for g in (gq, gk):
        if g is not None:
            _holds("norm weight", g, 2 * d.head_dim)
    unused = layer.region
    dims, symbol = launch_geometry(_abi.ATTN_QK_NORM_ROPE, d)
    ws = _workspace(rt, _abi.ATTN_QK_NORM_ROPE, d)
    args = [_region(step.counts, alignment=4), _region(step.positions, alignment=4),
            _region(step.row_offsets, alignment=4), _region(step.lengths, alignment=4),
            _region(step.page_offsets, alignment=4), _region(step.page_indices, alignment=4), layer.region, qkv,
            unused if gq is None else gq, unused if gk is None else gk, q, k_cache, v_cache, _region(ws, alignment=256)]
    _apart("q, the caches and what is read", args[10:13], args[:10])
    return BoundAttention([LaunchStep(rt.function(symbol), dims, KernelArguments(args), symbol)], workspace=ws,
                          keep=[layer, step], rotates=step if d.rotary_dim else None)


def bind_paged_decode(rt: ProjectionRuntime, layer: AttentionLayer, step: PagedStep, q: KernelArgument,
                      out: KernelArgument, k_cache: KernelArgument, v_cache: KernelArgument) -> BoundAttention:
    """Attention of the step's decoded sequences: q [max_tokens, Hq, D] (bf16,
    rotated) against the cached keys of each, out [max_tokens, Hq D] as the
    output projection reads it. Rows of other sequences stay as they were. out
    may not overlap what is read."""
    d = layer.desc
    _step_fits(layer, step)
    _holds("q", q, 2 * d.max_tokens * d.query_heads * d.head_dim)
    _holds("out", out, 2 * d.max_tokens * d.query_heads * d.head_dim)
    _holds("k_cache", k_cache, layer.cache_bytes)
    _holds("v_cache", v_cache, layer.cache_bytes)
    ws = _workspace(rt, _abi.ATTN_DECODE, d)
    dims, symbol = launch_geometry(_abi.ATTN_DECODE, d)
    args = [_region(step.counts, alignment=4), _region(step.row_offsets, alignment=4), _region(step.lengths, alignment=4),
            _region(step.page_offsets, alignment=4), _region(step.page_indices, alignment=4), layer.region, q, out,
            k_cache, v_cache, _region(ws, alignment=256)]
    _apart("out and what is read", [out], [a for i, a in enumerate(args) if i != 7])
    return BoundAttention([LaunchStep(rt.function(symbol), dims, KernelArguments(args), symbol)], workspace=ws,
                          keep=[layer, step])
