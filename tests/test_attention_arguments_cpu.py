"""Arguments of the attention's host side that no 32- or 64-bit field holds as
they are, page tables among them: refused, not cut."""
import numpy as np
import pytest

from lunaflux_amd import _abi, attention
from lunaflux_amd.device import DeviceError
from test_attention_cpu import make


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
