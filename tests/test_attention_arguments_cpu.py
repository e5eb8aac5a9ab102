"""Arguments of the attention's host side that no 32- or 64-bit field holds as
they are, page tables among them: refused, not cut."""
from types import SimpleNamespace

import numpy as np
import pytest

from lunaflux_amd import _abi, attention
from lunaflux_amd.device import DeviceError, KernelArgument
from test_attention_cpu import FakeAllocation, bound, make, region


@pytest.mark.parametrize("strides", [
    ((1 << 64) + 2 * 16 * 128, 16 * 128, 128), (2 * 16 * 128, 16 * 128 - (1 << 64), 128),
    (2 * 16 * 128, 16 * 128, 128, 1), (2 * 16 * 128, 16 * 128), (4096.0, 2048, 128), 128,
])
def test_strides(strides):
    make(strides=(2 * 16 * 128, 16 * 128, 128))
    with pytest.raises(DeviceError) as e:
        make(strides=strides)
    assert e.value.status == _abi.LF_INVALID_ARGUMENT


@pytest.mark.parametrize("axes", [(1 << 32) + 1, -(1 << 32) + 1, 1.5])
def test_axes(axes):
    with pytest.raises(DeviceError):
        make(rotary=attention.Rotary(np.ones(8), np.zeros(8), axes=axes))


@pytest.mark.parametrize("axis", [np.full(8, 0.5), np.full(8, 1 << 32, np.int64), np.full(8, np.nan), [1 << 40] * 8])
def test_axis_of_a_pair(axis):
    with pytest.raises(DeviceError):
        attention.Rotary(np.ones(8), axis)


@pytest.mark.parametrize("table", [
    [0.5], np.array([1.0]), np.array([(1 << 32) + 3]), np.array([-(1 << 32)]), np.array([1 << 63], np.uint64), [1 << 31],
    [1 << 80], ["1"], np.array([True]), [None],
])
def test_page_tables_of_a_step(table):
    """Page indices are whole numbers of 32 bits: others would name pages that nobody meant."""
    _, _, step = bound()
    before = [a.data.copy() for a in (step.counts, step.lengths, step.page_offsets, step.page_indices)]
    with pytest.raises(DeviceError) as e:
        step.stage([0, 1], [1], [table])
    assert e.value.status == _abi.LF_INVALID_ARGUMENT
    for a, b in zip((step.counts, step.lengths, step.page_offsets, step.page_indices), before):
        np.testing.assert_array_equal(a.data, b)


@pytest.mark.parametrize("dim", [65, 1, -64, -1, 64.0, 64.5])
def test_dimensions_of_a_rotation(dim):
    """Pairs of values: an odd number of them has none of its own frequencies."""
    assert attention.Rotary.of_theta(1e4, 64).turns.size == 32
    with pytest.raises(DeviceError):
        attention.Rotary.of_theta(1e4, dim)


def rotary_append(rotary):
    rt, layer, step = bound(rotary=rotary)
    qkv, q, cache = region(2 * 32 * 12 * 128), region(2 * 32 * 8 * 128), layer.cache_bytes
    op = attention.bind_qk_norm_rope(rt, layer, step, qkv, None, None, q, region(cache), region(cache))
    launched = []
    op.steps = [SimpleNamespace(launch=lambda stream, synchronous: launched.append(stream))]
    return step, op, launched


def test_rows_without_positions_are_not_rotated():
    """A step that was staged without positions does not turn by those of the one before."""
    step, op, launched = rotary_append(attention.Rotary.of_theta(1e4, 64))
    launch = lambda: op.launch("a stream", synchronous=False)  # noqa: E731
    launch()                                        # no rows
    step.stage([0, 1], [4], [[0]])
    with pytest.raises(DeviceError) as e:
        launch()
    assert e.value.status == _abi.LF_INVALID_ARGUMENT and len(launched) == 1
    step.stage([0, 1], [4], [[0]], [3])
    launch()
    step.stage([0, 2], [6], [[0]], prefill_rows=1)
    with pytest.raises(DeviceError):
        launch()
    step.stage([0, 2], [6], [[0]], attention.AS_THEY_ARE, prefill_rows=1)   # written by the caller
    launch()
    assert step.positions.data[:4].view(np.int32).tolist() == [3]
    with pytest.raises(DeviceError):                # a step that is refused leaves the one before
        step.stage([0, 2], [1], [[0]], prefill_rows=1)
    launch()
    step.stage([0], [], [])
    launch()
    assert len(launched) == 5


def test_rows_without_positions_without_rotation():
    step, op, launched = rotary_append(None)
    step.stage([0, 1], [4], [[0]])
    op.launch("a stream", synchronous=False)
    assert len(launched) == 1


def test_page_tables_that_are_taken():
    """Any integer type, an empty list, and indices outside the cache, which the device reports."""
    _, _, step = bound()
    step.stage([0, 1, 2, 2], [1, 17, 0], [np.array([[-1]], np.int64), np.array([2 ** 31 - 1, 3], np.uint64), []], prefill_rows=3)
    assert step.page_indices.data[:12].view(np.int32).tolist() == [-1, 2 ** 31 - 1, 3]
    for kind in (np.int32, np.int64, np.uint16):
        step.stage([0, 1, 2], [3, 18], [np.array([4], kind), np.array([2, 0], kind)])
        assert step.page_indices.data[:12].view(np.int32).tolist() == [4, 2, 0]


def within(alloc, offset, n):
    return KernelArgument.device_region(alloc, offset, n, 16)


def test_what_the_append_writes_overlaps_nothing_it_reads():
    rt, layer, step = bound(norm=1e-6)
    qkv, q, cache = 2 * 32 * 12 * 128, 2 * 32 * 8 * 128, layer.cache_bytes
    arena = FakeAllocation(qkv + q + 2 * cache + 512)
    at = [0, qkv, qkv + 256, qkv + 512, qkv + q + 512, qkv + q + cache + 512]
    size = [qkv, 256, 256, q, cache, cache]
    good = [within(arena, a, n) for a, n in zip(at, size)]
    bind = lambda args: attention.bind_qk_norm_rope(rt, layer, step, *args)  # noqa: E731
    bind(good)                                     # side by side
    bind([good[0], good[1], good[1], *good[3:]])   # weights are only read
    for read in (0, 1, 2):
        for written in (3, 4, 5):
            args = list(good)
            args[read] = within(arena, at[written] + size[written] - 256, size[read]) if read else good[0]
            if read == 0:
                args[written] = within(arena, qkv - 256, size[written])
            with pytest.raises(DeviceError):
                bind(args)
    # a step's own regions
    for alloc in (step.counts, step.positions, step.lengths, step.row_offsets, step.page_offsets, step.page_indices):
        alloc.byte_count = 1 << 20
        with pytest.raises(DeviceError):
            bind([*good[:3], within(alloc, 0, q), *good[4:]])


def test_what_decode_writes_overlaps_nothing_it_reads():
    rt, layer, step = bound()
    q, cache = 2 * 32 * 8 * 128, layer.cache_bytes
    arena = FakeAllocation(2 * q + 2 * cache)
    good = [within(arena, 0, q), within(arena, q, q), within(arena, 2 * q, cache), within(arena, 2 * q + cache, cache)]
    attention.bind_paged_decode(rt, layer, step, *good)
    for alloc in (step.counts, step.lengths, step.row_offsets, step.page_offsets, step.page_indices, layer.allocation):
        alloc.byte_count = 1 << 20
        with pytest.raises(DeviceError):
            attention.bind_paged_decode(rt, layer, step, good[0], within(alloc, 0, q), *good[2:])
