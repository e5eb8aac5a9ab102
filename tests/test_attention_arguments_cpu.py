"""Arguments of the attention's host side that no 32- or 64-bit field holds as
they are, page tables among them: refused, not cut."""
import numpy as np
import pytest

from lunaflux_amd import _abi, attention
from lunaflux_amd.device import DeviceError
from test_attention_cpu import bound, make


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


def test_page_tables_that_are_taken():
    """Any integer type, an empty list, and indices outside the cache, which the device reports."""
    _, _, step = bound()
    step.stage([0, 1, 2, 2], [1, 17, 0], [np.array([[-1]], np.int64), np.array([2 ** 31 - 1, 3], np.uint64), []], prefill_rows=3)
    assert step.page_indices.data[:12].view(np.int32).tolist() == [-1, 2 ** 31 - 1, 3]
    for kind in (np.int32, np.int64, np.uint16):
        step.stage([0, 1, 2], [3, 18], [np.array([4], kind), np.array([2, 0], kind)])
        assert step.page_indices.data[:12].view(np.int32).tolist() == [4, 2, 0]
