"""Host side of the low-rank adapters beside a projection (the low-rank section
of include/lunaflux_fp8.h).

A projection's weights are shared by every request; what a request's adapter
adds, scaling (x A^T) B^T, goes to the rows of the batch that are its own:

  adapters = LowRankAdapters(rt, hidden=4096, widths=[4096, 1024, 1024], ...)
  qkv = rt.bind_qkv(family, counts, x, wq, wk, wv, y, max_tokens)
  added = bind_low_rank(rt, counts, ids, x, adapters, y, y, max_tokens)

with ids int32 [max_tokens], the adapter of each row of the step (negative:
none). The kernels and their tiles follow from max_tokens, not from the rows of a
step, so steps of few rows want a binding of their own to the same regions: 61 rows
of 16 adapters (columns 4096 + 2 x 1024, hidden 4096) take 13.6 us under up to 256
tokens, 48 under 2048 and 73 under 8192 at rank 16, 32 (57 under 256), 77 and 196
at rank 64. `low_rank` is the numpy-level call for tests and tools.
"""
from __future__ import annotations

import ctypes
import operator
from dataclasses import dataclass

import numpy as np

from . import _abi
from .device import Allocation, DeviceError, KernelArgument, KernelArguments, KernelLaunchDimensions
from .fp8 import COUNTS_BYTES, BoundOperation, LaunchStep, ProjectionRuntime, _region


class LowRankDescriptor(ctypes.Structure):
    """lf_fp8_low_rank_desc."""

    _fields_ = [("magic", ctypes.c_uint32), ("adapters", ctypes.c_int32), ("rank", ctypes.c_int32),
                ("hidden", ctypes.c_int32), ("slices", ctypes.c_int32), ("columns", ctypes.c_int32),
                ("max_tokens", ctypes.c_int32), ("splits", ctypes.c_int32), ("ends", ctypes.c_int32 * 4),
                ("slots", ctypes.c_int32), ("one_launch", ctypes.c_int32),
                ("column_blocks", ctypes.c_int32), ("block_columns", ctypes.c_int32)]


def _check(operation, status):
    if status != _abi.LF_OK:
        raise DeviceError(operation, status)


def _invalid(what: str):
    return DeviceError(what, _abi.LF_INVALID_ARGUMENT)


def low_rank_descriptor(adapters: int, rank: int, hidden: int, widths, max_tokens: int) -> LowRankDescriptor:
    """widths: the output widths of the projections side by side (one, or Q, K, V)."""
    widths = [int(w) if isinstance(w, float) and w.is_integer() else w for w in widths]
    try:  # (ctypes would cut them to their fields)
        adapters, rank, hidden, max_tokens, *widths = map(operator.index, (adapters, rank, hidden, max_tokens, *widths))
    except TypeError:
        raise _invalid("low-rank shape") from None
    for value in (adapters, rank, max_tokens, hidden, *widths):
        if not 0 < value < 2 ** 31:
            raise _invalid("low-rank shape")
    d = LowRankDescriptor()
    _check("low_rank_descriptor", _abi.lib().lunaflux_fp8_low_rank_descriptor(
        adapters, rank, hidden, (ctypes.c_int64 * max(1, len(widths)))(*widths), len(widths), max_tokens, ctypes.byref(d)))
    return d


def workspace_bytes(desc: LowRankDescriptor) -> int:
    n = _abi.lib().lunaflux_fp8_low_rank_workspace_bytes(ctypes.byref(desc))
    if n < 0:
        raise _invalid("low_rank_workspace_bytes")
    return n


def launch_geometry(entry: int, desc: LowRankDescriptor):
    """(dims, symbol), or None for an entry that the profile does not launch."""
    dims = (ctypes.c_int32 * 7)()
    symbol = ctypes.create_string_buffer(128)
    status = _abi.lib().lunaflux_fp8_low_rank_launch_geometry(entry, ctypes.byref(desc), dims, symbol)
    if status == _abi.LF_UNSUPPORTED:
        return None
    _check("low_rank_launch_geometry", status)
    return (KernelLaunchDimensions.new(tuple(dims[0:3]), tuple(dims[3:6]), dims[6]),
            symbol.value.decode("ascii"))


class LowRankAdapters:
    """The adapters of one projection on the device: regions a bf16 [adapters,
    slices * rank, hidden], b bf16 [adapters, columns, rank], scaling fp32
    [adapters]. Adapters may be rewritten in place between steps (an adapter
    loaded into the place of another)."""

    def __init__(self, rt: ProjectionRuntime, *, hidden: int, widths, rank: int, adapters: int, a: KernelArgument,
                 b: KernelArgument, scaling: KernelArgument):
        d = low_rank_descriptor(adapters, rank, hidden, widths, 1)
        ends = [0, *d.ends[:d.slices]]
        self.hidden, self.rank, self.adapters = d.hidden, d.rank, d.adapters
        self.widths = tuple(end - begin for begin, end in zip(ends, ends[1:]))
        _holds("a", a, 2 * d.adapters * d.slices * d.rank * d.hidden, 16)
        _holds("b", b, 2 * d.adapters * d.columns * d.rank, 16)
        _holds("scaling", scaling, 4 * d.adapters, 4)
        self.a, self.b, self.scaling = a, b, scaling

    @staticmethod
    def upload(rt: ProjectionRuntime, a: np.ndarray, b: np.ndarray, scaling: np.ndarray, widths) -> "LowRankAdapters":
        """From host arrays: a bf16 bits [adapters, slices, rank, hidden], b bf16
        bits [adapters, columns, rank]. A rank that is no multiple of 16 is
        filled up with zeros."""
        a, b = np.ascontiguousarray(a, np.uint16), np.ascontiguousarray(b, np.uint16)
        scaling = np.ascontiguousarray(scaling, np.float32)
        widths = list(widths)
        if a.ndim != 4 or b.ndim != 3 or a.shape[0] != b.shape[0] or a.shape[1] != len(widths) or \
                b.shape[1:] != (sum(widths), a.shape[2]) or scaling.shape != (a.shape[0],):
            raise _invalid("low-rank arrays")
        rank = -(-a.shape[2] // 16) * 16
        if rank != a.shape[2]:
            a = np.concatenate([a, np.zeros((*a.shape[:2], rank - a.shape[2], a.shape[3]), np.uint16)], axis=2)
            b = np.concatenate([b, np.zeros((*b.shape[:2], rank - b.shape[2]), np.uint16)], axis=2)
        regions = [_region(rt.context.upload(v), alignment=256) for v in (a, b, scaling)]
        return LowRankAdapters(rt, hidden=a.shape[3], widths=widths, rank=rank, adapters=a.shape[0], a=regions[0],
                               b=regions[1], scaling=regions[2])


@dataclass
class BoundLowRank(BoundOperation):
    """check(): DeviceError(INVALID_ARGUMENT) if a launch met an adapter id past
    the adapters (its row was left without one); the error word is cleared.
    After asynchronous launches the caller synchronizes the stream first."""

    def check(self):
        if self.workspace.read(np.int32, (1,))[0] != 0:
            self.workspace.copy_from_host(np.zeros(1, np.int32))
            raise DeviceError("a row names an adapter that does not exist", _abi.LF_INVALID_ARGUMENT)


def _holds(what: str, region: KernelArgument, byte_count: int, alignment: int):
    if region.byte_count < byte_count or region.alignment < alignment:
        raise _invalid(f"{what}: {byte_count} bytes aligned to {alignment} are wanted")


def _overlap(p: KernelArgument, p_bytes: int, q: KernelArgument, q_bytes: int) -> bool:
    return p.allocation is q.allocation and p.offset < q.offset + q_bytes and q.offset < p.offset + p_bytes


def bind_low_rank(rt: ProjectionRuntime, counts: Allocation, ids: KernelArgument, x: KernelArgument,
                  adapters: LowRankAdapters, y: KernelArgument, out: KernelArgument, max_tokens: int) -> BoundLowRank:
    """out = y + the adapters' part of the live rows. x [max_tokens, hidden] is
    the projection's input, y [max_tokens, columns] its output; out may be y (in
    place) and otherwise overlaps nothing that is read."""
    desc = low_rank_descriptor(adapters.adapters, adapters.rank, adapters.hidden, adapters.widths, max_tokens)
    columns = 2 * max_tokens * desc.columns
    _holds("ids", ids, 4 * max_tokens, 4)
    _holds("x", x, 2 * max_tokens * desc.hidden, 16)
    _holds("y", y, columns, 16)
    _holds("out", out, columns, 16)
    c, a, b, scaling = _region(counts, COUNTS_BYTES, alignment=4), adapters.a, adapters.b, adapters.scaling
    n, r = desc.adapters, desc.rank
    read = [(c, COUNTS_BYTES), (ids, 4 * max_tokens), (x, 2 * max_tokens * desc.hidden), (scaling, 4 * n),
            (a, 2 * n * desc.slices * r * desc.hidden), (b, 2 * n * desc.columns * r)]
    if (_overlap(out, columns, y, columns) and out.offset != y.offset) or \
            any(_overlap(out, columns, region, size) for region, size in read):
        raise _invalid("out overlaps what is read")
    nbytes = workspace_bytes(desc)
    ws = rt.context.allocate(nbytes)
    ws.copy_from_host(np.zeros(nbytes, np.uint8))
    desc_alloc = rt.context.upload(np.frombuffer(bytes(desc), np.uint8).copy())
    dr, wsr = _region(desc_alloc, alignment=4), _region(ws, alignment=256)

    def step(entry, args):
        geometry = launch_geometry(entry, desc)
        return None if geometry is None else LaunchStep(rt.function(geometry[1]), geometry[0], KernelArguments(args),
                                                        geometry[1])

    steps = [step(_abi.LOW_RANK_ONE_LAUNCH, [c, ids, dr, scaling, x, a, b, y, out, wsr]),
             step(_abi.LOW_RANK_SHRINK, [c, ids, dr, x, a, wsr]),
             step(_abi.LOW_RANK_EXPAND, [c, ids, dr, scaling, b, y, out, wsr])]
    return BoundLowRank([s for s in steps if s is not None], workspace=ws, keep=[adapters])


def low_rank(rt: ProjectionRuntime, x: np.ndarray, y: np.ndarray, ids, adapters: LowRankAdapters,
             max_tokens: int | None = None) -> np.ndarray:
    """x bf16 bits [M, hidden], y bf16 bits [M, columns] -> out bf16 bits, in place on the device."""
    x, y = np.ascontiguousarray(x, np.uint16), np.ascontiguousarray(y, np.uint16)
    ids = np.asarray(ids)
    if ids.size and (ids.dtype.kind not in "iu" or ids.min() < -2 ** 31 or ids.max() >= 2 ** 31):
        raise _invalid("adapter ids are whole numbers of 32 bits")
    ids = np.ascontiguousarray(ids, np.int32)
    m = x.shape[0]
    max_tokens = max(m, 1) if max_tokens is None else max_tokens
    if m > max_tokens or y.shape != (m, sum(adapters.widths)) or ids.shape != (m,) or x.shape[1] != adapters.hidden:
        raise _invalid("low-rank rows")
    regions = []
    for values, row in ((x, 2 * x.shape[1]), (y, 2 * y.shape[1]), (ids, 4)):
        alloc = rt.context.allocate(max_tokens * row)
        alloc.copy_from_host(values)
        regions.append(_region(alloc, alignment=256))
    op = bind_low_rank(rt, rt.step_counts(m), regions[2], regions[0], adapters, regions[1], regions[1], max_tokens)
    op.launch(rt.stream, synchronous=True)
    return regions[1].allocation.read(np.uint16, y.shape) if m else y
