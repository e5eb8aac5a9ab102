"""lunaflux_fp8_attn_descriptor reads what stands before its own results alone: what a caller leaves in the rest of the
structure, which earlier forms of it had as padding, does not count."""
import ctypes

import numpy as np
import pytest

from lunaflux_amd import _abi, attention
from test_attention_cpu import FIELDS

RESULTS = ("scale_offset", "turns_offset", "axis_offset", "region_bytes", "sinks", "block_tokens", "block_scales", "padding")


def filled(byte, **changes):
    """The fields that a caller sets, over a structure of `byte`."""
    d = attention.AttentionDescriptor.from_buffer_copy(bytes([byte]) * ctypes.sizeof(attention.AttentionDescriptor))
    want = attention.attention_descriptor(**{**FIELDS, **changes})
    for name, _ in d._fields_:
        if name not in (*RESULTS, "magic", "reserved"):
            setattr(d, name, getattr(want, name))
    return d, want


@pytest.mark.parametrize("cache", list(attention.CACHES))
@pytest.mark.parametrize("byte", [0x00, 0x01, 0x5A, 0x80, 0xFF])
def test_what_a_caller_leaves_unset_does_not_count(byte, cache):
    d, want = filled(byte, cache=cache, window=9)
    assert _abi.lib().lunaflux_fp8_attn_descriptor(ctypes.byref(d)) == _abi.LF_OK
    assert bytes(d) == bytes(want) and d.sinks == 0


@pytest.mark.parametrize("byte", [0x00, 0xFF])
def test_sinks_are_an_argument(byte):
    d, want = filled(byte, window=9, sinks=4)
    lib = _abi.lib()
    assert lib.lunaflux_fp8_attn_descriptor_sinks(ctypes.byref(d), 4) == _abi.LF_OK
    assert bytes(d) == bytes(want) and d.sinks == 4
    before = bytes(d)
    assert lib.lunaflux_fp8_attn_descriptor_sinks(ctypes.byref(d), -1) == _abi.LF_INVALID_ARGUMENT and bytes(d) == before
    assert lib.lunaflux_fp8_attn_descriptor_sinks(None, 4) == _abi.LF_INVALID_ARGUMENT
    assert lib.lunaflux_fp8_attn_descriptor(ctypes.byref(d)) == _abi.LF_OK and d.sinks == 0


def test_a_region_keeps_the_sinks():
    d = attention.attention_descriptor(**FIELDS, window=9, sinks=4)
    held = attention.AttentionDescriptor.from_buffer_copy(np.asarray(attention.descriptor_region(d))[:256].tobytes())
    assert held.sinks == 4
