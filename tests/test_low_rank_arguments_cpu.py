"""Arguments of the low-rank adapters' host side: regions of one allocation, and
integers that 32- or 64-bit fields do not hold as they are."""
import numpy as np
import pytest

from lunaflux_amd import _abi, low_rank
from lunaflux_amd.device import DeviceError, KernelArgument
from test_attention_cpu import FakeAllocation, FakeRuntime, region

M, HIDDEN, WIDTHS, RANK, N = 8, 512, [128, 64], 16, 3
COLUMNS = sum(WIDTHS)
X, Y, IDS = 2 * M * HIDDEN, 2 * M * COLUMNS, 4 * M
A, B, S = 2 * N * len(WIDTHS) * RANK * HIDDEN, 2 * N * COLUMNS * RANK, 4 * N


def within(alloc, offset, n):
    return KernelArgument.device_region(alloc, offset, n, 16)


def bind(rt, counts, ids, x, y, out, a, b, scaling):
    adapters = low_rank.LowRankAdapters(rt, hidden=HIDDEN, widths=WIDTHS, rank=RANK, adapters=N, a=a, b=b, scaling=scaling)
    return low_rank.bind_low_rank(rt, counts, ids, x, adapters, y, out, M)


def test_regions_side_by_side_in_any_order():
    """An arena's regions, whichever is the longer and whichever comes first."""
    rt, counts = FakeRuntime(), FakeAllocation(20)
    sizes = {"ids": IDS, "x": X, "y": Y, "out": Y, "a": A, "b": B, "scaling": 16}
    for order in (["out", "x", "y", "ids", "a", "b", "scaling"], ["y", "out", "x", "b", "a", "scaling", "ids"],
                  ["x", "out", "a", "scaling", "b", "ids", "y"], ["ids", "out", "b", "y", "scaling", "x", "a"]):
        arena, at, regions = FakeAllocation(sum(sizes.values())), 0, {}
        for name in order:
            regions[name] = within(arena, at, sizes[name])
            at += sizes[name]
        bind(rt, counts, **regions)
        bind(rt, counts, **{**regions, "out": regions["y"]})   # in place


@pytest.mark.parametrize("read,size", [("ids", IDS), ("x", X), ("y", Y), ("a", A), ("b", B), ("scaling", S)])
def test_out_overlaps_nothing_that_is_read(read, size):
    rt, counts = FakeRuntime(), FakeAllocation(20)
    arena = FakeAllocation(Y + size + Y)
    good = {"ids": region(IDS, 4), "x": region(X), "y": region(Y), "a": region(A), "b": region(B), "scaling": region(S, 4),
            "out": within(arena, 0, Y), read: within(arena, Y, size)}
    bind(rt, counts, **good)
    for offset in (16, Y + (size - 1) // 16 * 16):   # over its first and its last bytes
        with pytest.raises(DeviceError) as e:
            bind(rt, counts, **{**good, "out": within(arena, offset, Y)})
        assert e.value.status == _abi.LF_INVALID_ARGUMENT


def test_out_does_not_overlap_the_counts():
    rt, arena = FakeRuntime(), FakeAllocation(Y + 64)
    regions = {"ids": region(IDS, 4), "x": region(X), "y": region(Y), "a": region(A), "b": region(B), "scaling": region(S, 4)}
    bind(rt, arena, out=within(arena, 32, Y), **regions)
    with pytest.raises(DeviceError):
        bind(rt, arena, out=within(arena, 16, Y), **regions)
