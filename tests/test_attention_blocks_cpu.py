"""Prompts, sinks and caches with scales by blocks without a GPU: descriptors and
their regions, sizes and geometry, what bindings and steps refuse, and the
oracle's steps."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

from lunaflux_amd import _abi, attention
from lunaflux_amd.device import DeviceError, KernelArgument
from test_attention_cpu import FIELDS, FakeAllocation, FakeRuntime, bound, make, region


def test_descriptor_of_a_cache_with_scales_by_blocks():
    d = make(cache="e4m3_blocks")
    assert (d.block_tokens, d.block_scales) == (16, 9 * 2 * 16 * 128)
    assert _abi.lib().lunaflux_fp8_attn_cache_bytes(ctypes.byref(d)) == d.block_scales + 9 * 1 * 2 * 4
    small = make(cache="e4m3_blocks", page_size=8)
    assert small.block_tokens == 8
    large = make(cache="e4m3_blocks", page_size=64, strides=(2 * 64 * 144 + 16, 64 * 144, 144))
    assert large.block_tokens == 16 and large.block_scales % 256 == 0
    assert large.block_scales >= 8 * large.page_stride + large.head_stride + 63 * 144 + 128
    assert _abi.lib().lunaflux_fp8_attn_cache_bytes(ctypes.byref(large)) == large.block_scales + 9 * 4 * 2 * 4
    for other in ("bf16", "e4m3"):
        assert (make(cache=other).block_tokens, make(cache=other).block_scales) == (0, 0)
    layer = attention.attention_layer(FakeRuntime(), **{**FIELDS, "page_size": 64}, cache="e4m3_blocks")
    assert layer.block_scales_shape == (9, 4, 2) and layer.block_scales_offset == layer.desc.block_scales
    with pytest.raises(DeviceError):
        attention.attention_layer(FakeRuntime(), **FIELDS).block_scales_shape


def test_scales_of_a_cache_with_scales_by_blocks_are_its_own():
    d = make(cache="e4m3_blocks")
    region = attention.descriptor_region(d)
    np.testing.assert_array_equal(region[d.scale_offset:d.scale_offset + 16].view(np.float32), 1.0)
    with pytest.raises(DeviceError):
        attention.descriptor_region(d, [1.0, 1.0], [1.0, 1.0])


@pytest.mark.parametrize("changes", [
    dict(sinks=-1), dict(sinks=1 << 32), dict(sinks=1.5), dict(window=1 << 31), dict(cache="e4m3_blocks", max_tokens=(1 << 24) - 1),
])
def test_descriptor_refusals(changes):
    make(sinks=4, window=9)
    with pytest.raises(DeviceError) as e:
        make(**changes)
    assert e.value.status == _abi.LF_INVALID_ARGUMENT


@pytest.mark.parametrize("field,value", [("block_tokens", 8), ("block_tokens", 0), ("block_scales", 0), ("cache", 2), ("cache", 4), ("sinks", -1)])
def test_a_changed_descriptor_is_refused(field, value):
    d = make(cache="e4m3_blocks")
    setattr(d, field, value)
    for entry in (_abi.ATTN_QK_NORM_ROPE, _abi.ATTN_DECODE, _abi.ATTN_PREFILL, _abi.ATTN_PREFILL_JOIN):
        assert _abi.lib().lunaflux_fp8_attn_workspace_bytes(entry, ctypes.byref(d)) == -1
        with pytest.raises(DeviceError):
            attention.launch_geometry(entry, d)
    with pytest.raises(DeviceError):
        attention.descriptor_region(d)


def test_geometry():
    code = _abi.code_object_bytes()
    for head_dim in (64, 128, 256):
        for cache in ("bf16", "e4m3", "e4m3_blocks"):
            d = make(head_dim=head_dim, cache=cache, table_entries=4000)
            names = {e: attention.launch_geometry(e, d)[1] for e in range(1, 5)}
            blocks = cache == "e4m3_blocks"
            assert names == {1: f"lf_attn_qk_norm_rope_{cache}" + (f"_d{head_dim}" if blocks else ""), 2: f"lf_attn_decode_d{head_dim}_{cache}",
                             3: f"lf_attn_prefill_d{head_dim}_{cache}", 4: f"lf_attn_prefill_join_d{head_dim}_{cache}"}
            sinks = make(head_dim=head_dim, cache=cache, window=5, sinks=2)
            names[5] = attention.launch_geometry(_abi.ATTN_DECODE, sinks)[1]
            assert names[5] == f"lf_attn_decode_d{head_dim}_{cache}" + ("" if blocks else "_sinks")
            # sinks without a window, or a window without sinks: nothing more to read
            assert attention.launch_geometry(_abi.ATTN_DECODE, make(head_dim=head_dim, cache=cache, sinks=2))[1] == names[2]
            assert attention.launch_geometry(_abi.ATTN_DECODE, make(head_dim=head_dim, cache=cache, window=2))[1] == names[2]
            for name in names.values():
                assert name.encode() + b"\0" in code
            for e in range(1, 5):
                assert attention.launch_geometry(e, d)[0].shared_memory_bytes <= 98304
    # the largest grid of an append keeps its threads in 32 bits
    d = make(cache="e4m3_blocks", max_tokens=(1 << 24) - (1 << 14) - 1, max_sequences=2048, query_heads=1024, kv_heads=1024, head_dim=64)
    assert attention.launch_geometry(_abi.ATTN_QK_NORM_ROPE, d)[0].grid[0] * 256 < 1 << 32


def test_prompts_too_short_to_be_cut_need_no_join():
    """16 key tiles or more of 64 keys (32 for heads of 256) can be cut."""
    for head_dim, most in ((64, 960), (128, 960), (256, 480)):
        d = make(head_dim=head_dim, page_size=16, table_entries=most // 16)
        assert attention.launch_geometry(_abi.ATTN_PREFILL_JOIN, d) is None
        assert attention.workspace_bytes(_abi.ATTN_PREFILL, d) == 256
        d = make(head_dim=head_dim, page_size=16, table_entries=most // 16 + 1)
        assert attention.launch_geometry(_abi.ATTN_PREFILL_JOIN, d) is not None
        assert attention.workspace_bytes(_abi.ATTN_PREFILL, d) == 256 + 2 * 256 * 256 * (head_dim + 2) * 4
    # a window bounds a tile's keys
    assert attention.launch_geometry(_abi.ATTN_PREFILL_JOIN, make(window=600, sinks=100, table_entries=4000)) is None
    assert attention.launch_geometry(_abi.ATTN_PREFILL_JOIN, make(window=900, sinks=100, table_entries=4000)) is not None


def test_bindings_of_prompts():
    rt, layer, step = bound()
    q, cache = 2 * 32 * 8 * 128, layer.cache_bytes
    bind = attention.bind_paged_prefill
    ok = [region(q), region(q), region(cache), region(cache)]
    assert [s.name for s in bind(rt, layer, step, *ok).steps] == ["lf_attn_prefill_d128_bf16"]
    long = attention.attention_layer(rt, **{**FIELDS, "table_entries": 400})
    assert [s.name for s in bind(rt, long, attention.PagedStep(rt, long), *ok).steps] == \
        ["lf_attn_prefill_d128_bf16", "lf_attn_prefill_join_d128_bf16"]
    for at, bad in [(0, region(q - 2)), (1, region(q - 2)), (2, region(cache - 1)), (3, region(cache, 2)), (0, region(q, 8))]:
        with pytest.raises(DeviceError):
            bind(rt, layer, step, *ok[:at], bad, *ok[at + 1:])
    for at in (0, 2, 3):                  # out is one of the others
        with pytest.raises(DeviceError):
            bind(rt, layer, step, *(ok[1] if i == at else r for i, r in enumerate(ok)))
    other = attention.PagedStep(rt, attention.attention_layer(rt, **{**FIELDS, "max_sequences": 5}))
    with pytest.raises(DeviceError):      # a step of another descriptor
        bind(rt, layer, other, *ok)
    for alloc in (step.counts, step.lengths, step.row_offsets, step.page_offsets, step.page_indices, layer.allocation):
        alloc.byte_count = 1 << 20
        with pytest.raises(DeviceError):
            bind(rt, layer, step, ok[0], KernelArgument.device_region(alloc, 0, q, 16), *ok[2:])


def test_a_cache_region_without_room_for_the_scales():
    rt = FakeRuntime()
    layer = attention.attention_layer(rt, **FIELDS, cache="e4m3_blocks")
    step = attention.PagedStep(rt, layer)
    q, qkv, cache = 2 * 32 * 8 * 128, 2 * 32 * 12 * 128, layer.cache_bytes
    for bind, ok in ((attention.bind_paged_prefill, [region(q), region(q), region(cache), region(cache)]),
                     (attention.bind_paged_decode, [region(q), region(q), region(cache), region(cache)]),
                     (attention.bind_qk_norm_rope, [region(qkv), None, None, region(q), region(cache), region(cache)])):
        bind(rt, layer, step, *ok)
        for at in (-1, -2):
            with pytest.raises(DeviceError):
                bind(rt, layer, step, *(region(layer.block_scales_offset) if i == len(ok) + at else r for i, r in enumerate(ok)))


@pytest.mark.parametrize("rows,lengths,tables,apart", [
    ([3, 2], [3, 2], [[0], [1]], True), ([3, 2], [3, 2], [[4], [4]], False), ([20], [20], [[4, 4]], False),
    ([2, 2], [18, 2], [[4, 5], [4]], True),         # what is only read may be another's page
    ([4, 2], [18, 2], [[4, 5], [4]], False),        # two rows before the page's end
    ([1, 1, 1], [17, 33, 1], [[0, 1], [0, 2, 3], [4]], True), ([0, 1], [16, 1], [[4], [4]], True), ([], [], [], True),
])
def test_pages_that_a_step_writes(rows, lengths, tables, apart):
    rt = FakeRuntime()
    layer = attention.attention_layer(rt, **FIELDS, cache="e4m3_blocks")
    step = attention.PagedStep(rt, layer)
    assert step.pages_apart
    q, qkv, cache = 2 * 32 * 8 * 128, 2 * 32 * 12 * 128, layer.cache_bytes
    op = attention.bind_qk_norm_rope(rt, layer, step, region(qkv), None, None, region(q), region(cache), region(cache))
    launched = []
    op.steps = [SimpleNamespace(launch=lambda stream, synchronous: launched.append(stream))]
    step.stage(np.concatenate([[0], np.cumsum(rows)]).astype(np.int64), lengths, tables, prefill_rows=len(rows))
    for _ in range(2):
        assert step.pages_apart == apart
        if apart:
            op.launch("a stream", synchronous=False)
        else:
            with pytest.raises(DeviceError) as e:
                op.launch("a stream", synchronous=False)
            assert e.value.status == _abi.LF_INVALID_ARGUMENT
    assert len(launched) == (2 if apart else 0)
    # attention, which only reads, does not mind
    assert attention.bind_paged_decode(rt, layer, step, region(q), region(q), region(cache), region(cache)).scales is None
