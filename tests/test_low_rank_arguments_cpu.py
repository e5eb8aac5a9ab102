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


@pytest.mark.parametrize("args", [
    (2, 16, 512, [(1 << 64) + 64], 8), (2, 16, 512, [64.5], 8), (2, 16, (1 << 64) + 512, [64], 8), (2, 16, 512.5, [64], 8),
    (2, 16.0, 512, [64], 8), (2.5, 16, 512, [64], 8), (2, 16, 512, [64], 8.5), (2, 16, 512, ["64"], 8), (2, 16, 512, [None], 8),
])
def test_integers_of_a_descriptor(args):
    with pytest.raises(DeviceError) as e:
        low_rank.low_rank_descriptor(*args)
    assert e.value.status == _abi.LF_INVALID_ARGUMENT


def test_integers_of_any_type():
    d = low_rank.low_rank_descriptor(np.int64(2), np.uint8(16), np.int32(512), np.array([64, 128]), np.int16(8))
    assert (d.adapters, d.rank, d.hidden, d.columns, d.max_tokens) == (2, 16, 512, 192, 8)
    held = low_rank.LowRankAdapters(FakeRuntime(), hidden=np.int16(512), widths=[64.0, np.uint8(128)], rank=np.uint8(16),
                                    adapters=np.uint8(20), a=region(2 * 20 * 32 * 512), b=region(2 * 20 * 192 * 16),
                                    scaling=region(80, 4))
    assert held.widths == (64, 128) and held.rank == 16


@pytest.mark.parametrize("ids", [np.full(M, 1 << 32), np.full(M, 0.5), np.full(M, -(1 << 32) + 1), np.full(M, (1 << 64) - 1, np.uint64),
                                 np.ones(M, bool), [1 << 70] * M])
def test_ids_of_rows(ids):
    """Ids that a cast would turn into another adapter's."""
    rt = FakeRuntime()
    adapters = low_rank.LowRankAdapters(rt, hidden=HIDDEN, widths=WIDTHS, rank=RANK, adapters=N, a=region(A), b=region(B),
                                        scaling=region(S, 4))
    with pytest.raises(DeviceError) as e:
        low_rank.low_rank(rt, np.zeros((M, HIDDEN), np.uint16), np.zeros((M, COLUMNS), np.uint16), ids, adapters)
    assert e.value.status == _abi.LF_INVALID_ARGUMENT


@pytest.mark.parametrize("rows,widths,block", [
    (2368, [4096, 1024, 1024], 512), (2369, [4096, 1024, 1024], 1024), (3600, [4096, 1024, 1024], 1024),
    (14272, [64], 512), (14273, [64], 1024),
])
def test_columns_of_a_block(rows, widths, block):
    """1024 columns from 224 blocks of 64 rows on."""
    assert low_rank.low_rank_descriptor(4, 64, 4096, widths, rows).block_columns == block
