"""Attention descriptors that were changed after they were made."""
import ctypes

import numpy as np
import pytest

from lunaflux_amd import _abi, attention
from lunaflux_amd.device import DeviceError
from test_attention_cpu import make

F32P, F64P, I32P, U8P = (ctypes.POINTER(t) for t in (ctypes.c_float, ctypes.c_double, ctypes.c_int32, ctypes.c_uint8))


@pytest.mark.parametrize("field,value,pairs,scales", [
    ("rotary_dim", 128, 64, 0),            # turns and axes behind the end of the region
    ("kv_heads", 8, 0, 16),
    ("turns_offset", 1 << 20, 0, 0), ("axis_offset", 256, 0, 0), ("scale_offset", 0, 0, 0), ("region_bytes", 256, 0, 0),
])
def test_a_changed_descriptor_is_refused(field, value, pairs, scales):
    d = make(max_sequences=1, kv_heads=1, query_heads=8)
    setattr(d, field, value)
    lib, ref = _abi.lib(), ctypes.byref(d)
    assert lib.lunaflux_fp8_attn_workspace_bytes(_abi.ATTN_DECODE, ref) == -1
    assert lib.lunaflux_fp8_attn_cache_bytes(ref) == -1
    with pytest.raises(DeviceError):
        attention.launch_geometry(_abi.ATTN_DECODE, d)
    # a region with room behind it, which has to stay as it was
    room = np.full(1 << 21, 0x5A, np.uint8)
    turns, axis, ones = np.ones(pairs), np.zeros(pairs, np.int32), np.ones(scales, np.float32)
    status = lib.lunaflux_fp8_attn_region(ref, ones.ctypes.data_as(F32P) if scales else None, scales,
                                          turns.ctypes.data_as(F64P), axis.ctypes.data_as(I32P), pairs,
                                          room.ctypes.data_as(U8P), d.region_bytes)
    assert status == _abi.LF_INVALID_ARGUMENT and (room == 0x5A).all()
