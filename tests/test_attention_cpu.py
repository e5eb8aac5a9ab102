"""Attention without a GPU: the descriptor and its region, sizes and geometry,
what the bindings and a step's staging refuse, and the oracle itself."""
import ctypes
import math

import numpy as np
import pytest

import attention_oracle as ao
from lunaflux_amd import _abi, attention
from lunaflux_amd.device import DeviceError, KernelArgument

FIELDS = dict(query_heads=8, kv_heads=2, head_dim=128, page_size=16, pages=9, max_tokens=32, max_sequences=6,
              table_entries=40)


def make(**changes):
    return attention.attention_descriptor(**{**FIELDS, **changes})


def test_descriptor_defaults_and_layout():
    assert ctypes.sizeof(attention.AttentionDescriptor) == 256
    rotary = attention.Rotary.of_theta(10000.0, 64)
    d = make(rotary=rotary, norm_epsilon=1e-6)
    assert (d.page_stride, d.head_stride, d.token_stride) == (2 * 16 * 128, 16 * 128, 128)
    assert d.softmax_scale == np.float32(1 / math.sqrt(128)) and d.rotary_dim == 64 and d.axes == 1 and d.norm == 1
    assert _abi.lib().lunaflux_fp8_attn_cache_bytes(ctypes.byref(d)) == 9 * 2 * 16 * 128 * 2
    region = attention.descriptor_region(d, rotary=rotary)
    assert region.size == d.region_bytes and bytes(region[:4]) == b"LATN"
    np.testing.assert_array_equal(region[d.scale_offset:d.scale_offset + 16].view(np.float32), 1.0)
    np.testing.assert_array_equal(region[d.turns_offset:d.turns_offset + 256].view(np.float64), rotary.turns)
    np.testing.assert_array_equal(region[d.axis_offset:d.axis_offset + 128].view(np.int32), 0)
    assert rotary.turns[0] == 1 / (2 * math.pi)
    e = make(cache="e4m3")
    assert _abi.lib().lunaflux_fp8_attn_cache_bytes(ctypes.byref(e)) == 9 * 2 * 16 * 128
    scales = attention.descriptor_region(e, [0.5, 0.25], [2.0, 4.0])[e.scale_offset:][:16].view(np.float32)
    np.testing.assert_array_equal(scales, [0.5, 0.25, 2.0, 4.0])


@pytest.mark.parametrize("changes", [
    dict(query_heads=7), dict(query_heads=0), dict(kv_heads=0), dict(query_heads=2048, kv_heads=2048),
    dict(head_dim=96), dict(head_dim=32), dict(head_dim=512), dict(page_size=4), dict(page_size=24),
    dict(page_size=2048), dict(pages=0), dict(max_tokens=0), dict(max_tokens=1 << 25), dict(max_tokens=1 << 24), dict(max_sequences=0),
    dict(max_sequences=2049), dict(table_entries=0), dict(table_entries=1 << 27), dict(table_entries=1 << 40),
    dict(window=-1), dict(norm_epsilon=-1.0), dict(norm_epsilon=math.nan), dict(norm_epsilon=math.inf),
    dict(softmax_scale=math.inf), dict(softmax_scale=math.nan), dict(pages=1 << 33), dict(pages=1.5),
    dict(strides=(2 * 16 * 128 - 8, 16 * 128, 128)),          # pages overlap
    dict(strides=(16 * 128 * 2, 16 * 128, 64)),               # tokens overlap
    dict(strides=(2 * 16 * 128, 16 * 128 + 4, 128 + 4)),      # not multiples of 16 bytes
    dict(strides=(2 * 16 * 128, 16 * 128, 0)), dict(strides=(-4096, 2048, 128)),
    dict(strides=(1 << 30, 16 * 128, 128)),                   # 2^31 bytes
    # more (tile, head) items than 31 bits
    dict(query_heads=1024, kv_heads=1024, table_entries=1 << 20, page_size=1024),
])
def test_descriptor_refusals(changes):
    with pytest.raises(DeviceError) as e:
        make(**changes)
    assert e.value.status == _abi.LF_INVALID_ARGUMENT


def test_other_orders_of_a_cache_are_taken():
    make(strides=(2 * 16 * 128, 128, 2 * 128))                # [page][slot][head]
    make(strides=(128, 9 * 16 * 128, 9 * 128))                # [head][slot][page]
    make(query_heads=1, kv_heads=1)                           # pages and heads step alike
    make(pages=1, strides=(128, 16 * 128, 128))
    d = make(cache="e4m3", strides=(2 * 16 * 144, 16 * 144, 144))   # padded rows
    assert _abi.lib().lunaflux_fp8_attn_cache_bytes(ctypes.byref(d)) == 8 * 4608 + 2304 + 15 * 144 + 128


def test_unknown_cache_type():
    with pytest.raises(ValueError):
        make(cache="fp16")


def test_rotary_refusals():
    R = attention.Rotary
    for bad in (lambda: R(np.ones((2, 2)), np.zeros((2, 2))), lambda: R(np.ones(8), np.zeros(7)),
                lambda: R(np.ones(8), np.zeros(8), "pairs"), lambda: R.of_theta(1e4, 64, (16, 15)),
                lambda: R.of_theta(1e4, 64, (40, -8))):
        with pytest.raises(DeviceError):
            bad()
    for rotary in (R(np.ones(4), np.zeros(4)),                       # 8 values: not a multiple of 16
                   R(np.ones(72), np.zeros(72)),                     # more than the head
                   R(np.ones(8), np.zeros(8), axes=5)):
        with pytest.raises(DeviceError):
            make(rotary=rotary)
    sections = R.of_theta(1e4, 128, (16, 24, 24))
    assert sections.axes == 3 and list(np.bincount(sections.axis)) == [16, 24, 24]


def test_region_refusals():
    rotary = attention.Rotary.of_theta(1e4, 64)
    d, e = make(rotary=rotary), make(cache="e4m3")
    ok = dict(k_scales=[1.0, 1.0], v_scales=[1.0, 1.0])
    attention.descriptor_region(e, **ok)
    attention.descriptor_region(d, rotary=rotary, **ok)
    for desc, kw in [(d, {}), (d, dict(rotary=attention.Rotary.of_theta(1e4, 32))),
                     (d, dict(rotary=attention.Rotary(np.full(32, np.inf), np.zeros(32)))),
                     (d, dict(rotary=attention.Rotary(np.ones(32), np.full(32, 1)))),
                     (d, dict(rotary=attention.Rotary(np.ones(32), np.full(32, -1), axes=1))),
                     (d, dict(rotary=rotary, k_scales=[2.0, 1.0], v_scales=[1.0, 1.0])),
                     (e, {}), (e, dict(k_scales=[1.0, 1.0])), (e, dict(k_scales=[1.0], v_scales=[1.0])),
                     (e, dict(k_scales=[1.0, 1.0, 1.0], v_scales=[1.0])),
                     (e, dict(k_scales=[0.0, 1.0], v_scales=[1.0, 1.0])),
                     (e, dict(k_scales=[1.0, -1.0], v_scales=[1.0, 1.0])),
                     (e, dict(k_scales=[1.0, 1.0], v_scales=[math.nan, 1.0])),
                     (e, dict(k_scales=[1.0, 1.0], v_scales=[math.inf, 1.0])),
                     (e, dict(k_scales=[1e-39, 1.0], v_scales=[1.0, 1.0]))]:    # 1 / scale is infinite
        with pytest.raises(DeviceError):
            attention.descriptor_region(desc, **kw)


def test_geometry_and_workspace():
    for head_dim in (64, 128, 256):
        for cache in ("bf16", "e4m3"):
            d = make(head_dim=head_dim, cache=cache)
            names = [attention.launch_geometry(e, d)[1] for e in (_abi.ATTN_QK_NORM_ROPE, _abi.ATTN_DECODE)]
            assert names == [f"lf_attn_qk_norm_rope_{cache}", f"lf_attn_decode_d{head_dim}_{cache}"]
            for name in names:
                assert name.encode() + b"\0" in _abi.code_object_bytes()
    # the largest head tile and prefix fit the launch's LDS limit
    d = make(query_heads=64, head_dim=256, max_sequences=2048)
    dims, _ = attention.launch_geometry(_abi.ATTN_DECODE, d)
    assert dims.shared_memory_bytes <= 98304
    assert attention.workspace_bytes(_abi.ATTN_DECODE, d) > 0
    with pytest.raises(DeviceError):
        attention.launch_geometry(9, d)
    with pytest.raises(DeviceError):
        attention.workspace_bytes(9, d)
    with pytest.raises(DeviceError):
        attention.launch_geometry(_abi.ATTN_DECODE, attention.AttentionDescriptor())


# -- staging and binding against a stand-in context ---------------------------------
class FakeAllocation:
    def __init__(self, byte_count):
        self.byte_count, self.ptr, self.data = byte_count, 1, np.zeros(byte_count, np.uint8)

    def copy_from_host(self, data, offset=0):
        raw = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        assert offset + raw.size <= self.byte_count
        self.data[offset:offset + raw.size] = raw


class FakeRuntime:
    def __init__(self):
        self.context = self

    def allocate(self, n):
        return FakeAllocation(n)

    def upload(self, data):
        a = FakeAllocation(np.ascontiguousarray(data).nbytes)
        a.copy_from_host(data)
        return a

    def function(self, symbol):
        return symbol


def region(n, alignment=16):
    return KernelArgument.device_region(FakeAllocation(n), 0, n, alignment)


def bound(norm=None, rotary=None):
    rt = FakeRuntime()
    layer = attention.attention_layer(rt, rotary=rotary, norm_epsilon=norm, **FIELDS)
    return rt, layer, attention.PagedStep(rt, layer)


def test_stage_writes_the_runtime_inputs():
    rt, layer, step = bound()
    step.stage([0, 3, 4, 5], [20, 17, 1], [[4, 2], [8, 1, 0], [3]], np.array([17, 18, 19, 16, 0]), prefill_rows=1)
    read = lambda a, n: a.data[:4 * n].view(np.int32).tolist()  # noqa: E731
    assert read(step.counts, 5) == [1, 2, 3, 5, 6]
    assert read(step.row_offsets, 4) == [0, 3, 4, 5] and read(step.lengths, 3) == [20, 17, 1]
    assert read(step.page_offsets, 4) == [0, 2, 5, 6] and read(step.page_indices, 6) == [4, 2, 8, 1, 0, 3]
    assert read(step.positions, 5) == [17, 18, 19, 16, 0]
    step.stage([0], [], [])
    assert read(step.counts, 5) == [0, 0, 0, 0, 0]


@pytest.mark.parametrize("args,kw", [
    (([0, 1], [1, 1], [[0], [1]]), {}), (([0, 1], [1], []), {}), (([1, 2], [1], [[0]]), {}),
    (([0, 2], [5], [[0]]), {}),                                  # a decoded sequence of two rows
    (([0, 0], [5], [[0]]), {}), (([0, 2], [1], [[0]]), dict(prefill_rows=1)),   # fewer tokens than rows
    (([0, 1], [17], [[0]]), {}),                                 # pages too few
    (([0, 1], [1], [[0] * 41]), {}),                             # table too long
    (([0, 33], [40], [[0] * 3]), dict(prefill_rows=1)),          # rows past max_tokens
    ((list(range(8)), [1] * 7, [[0]] * 7), {}),                  # sequences past max_sequences
    (([0, 2, 1], [3, 3], [[0], [0]]), dict(prefill_rows=2)), (([0, 1], [1], [[0]]), dict(prefill_rows=2)),
    (([0, 1], [1], [[0]]), dict(prefill_rows=-1)), (([0, 1], [1], [[0]], [1, 2]), {}),
    (([0, 1], [1], [[0]], [[1, 2]]), {}), (([0, 1], [1], [[0]], [1.5]), {}), (([0, 1], [1], [[0]], [1 << 31]), {}),
    (([0.0, 1.0], [1], [[0]]), {}), (([0, 1], [1.0], [[0]]), {}),
])
def test_stage_refusals(args, kw):
    _, _, step = bound()
    before = [a.data.copy() for a in (step.counts, step.row_offsets, step.lengths, step.page_offsets)]
    with pytest.raises(DeviceError):
        step.stage(*args, **kw)
    for a, b in zip((step.counts, step.row_offsets, step.lengths, step.page_offsets), before):
        np.testing.assert_array_equal(a.data, b)


def test_binding_refusals():
    rt, layer, step = bound(norm=1e-6)
    qkv, q = 2 * 32 * 12 * 128, 2 * 32 * 8 * 128
    cache, g = layer.cache_bytes, region(256)
    bind = attention.bind_qk_norm_rope
    ok = [region(qkv), g, g, region(q), region(cache), region(cache)]
    assert bind(rt, layer, step, *ok).steps[0].name == "lf_attn_qk_norm_rope_bf16"
    for at, bad in [(0, region(qkv - 2)), (0, region(qkv, 8)), (1, None), (2, None), (1, region(254)),
                    (3, region(q - 2)), (4, region(cache - 1)), (5, region(cache - 1)), (5, region(cache, 4))]:
        with pytest.raises(DeviceError):
            bind(rt, layer, step, *ok[:at], bad, *ok[at + 1:])
    one = FakeAllocation(2 * qkv)
    whole = KernelArgument.device_region(one, 0, qkv, 16)
    for at, bad in [(3, KernelArgument.device_region(one, qkv - 16, q, 16)), (4, KernelArgument.device_region(one, 256, cache, 16)),
                    (3, KernelArgument.device_region(one, 0, q, 16))]:
        args = [whole, *ok[1:]]
        args[at] = bad
        with pytest.raises(DeviceError):  # overlap
            bind(rt, layer, step, *args)
    with pytest.raises(DeviceError):
        bind(rt, layer, step, *ok[:4], ok[4], ok[4])
    rt2, plain, step2 = bound()
    with pytest.raises(DeviceError):      # norm weights for a layer without a norm
        bind(rt2, plain, step2, *ok)
    decode = attention.bind_paged_decode
    ok = [region(q), region(q), region(cache), region(cache)]
    assert [s.name for s in decode(rt, layer, step, *ok).steps] == ["lf_attn_decode_d128_bf16"]
    for at, bad in [(0, region(q - 2)), (1, region(q - 2)), (2, region(cache - 1)), (3, region(cache, 2))]:
        with pytest.raises(DeviceError):
            decode(rt, layer, step, *ok[:at], bad, *ok[at + 1:])
    for at in (0, 2, 3):                  # out is one of the others
        with pytest.raises(DeviceError):
            decode(rt, layer, step, *(ok[1] if i == at else r for i, r in enumerate(ok)))
    decode(rt, layer, step, *ok[:3], ok[2])   # keys that are their own values are only read
    other = attention.PagedStep(rt, attention.attention_layer(rt, **{**FIELDS, "max_sequences": 5}))
    with pytest.raises(DeviceError):      # a step of another descriptor
        decode(rt, layer, other, *ok)
    with pytest.raises(DeviceError):
        bind(rt, layer, other, region(qkv), g, g, region(q), region(cache), region(cache))


# -- the oracle ------------------------------------------------------------------
def test_oracle_decode_is_a_softmax_average():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((3, 64)), rng.standard_normal((20, 64)), rng.standard_normal((20, 64))
    out, tol = ao.decode(q, k, v, 0.125)
    want = np.zeros_like(out)
    for r in range(3):
        z = [sum(q[r, i] * k[j, i] for i in range(64)) * 0.125 for j in range(20)]
        w = [math.exp(x) for x in z]
        for j in range(20):
            want[r] += w[j] / sum(w) * v[j]
    np.testing.assert_allclose(out, want, rtol=1e-12, atol=1e-14)
    assert (tol > 0).all() and (tol < 0.05).all()


def test_oracle_rotation_keeps_relative_positions():
    """Rotated q . k depends on the difference of their positions alone."""
    rng = np.random.default_rng(1)
    for pairing in ("half", "neighbour"):
        rotary = attention.Rotary.of_theta(10000.0, 32, pairing=pairing)
        q, k = rng.standard_normal((1, 1, 64)), rng.standard_normal((1, 1, 64))
        at = lambda u, p: ao.turned(u, np.array([[p]]), rotary)[0, 0]  # noqa: E731
        assert abs(at(q, 905) @ at(k, 900) - at(q, 5) @ at(k, 0)) < 1e-9
        np.testing.assert_array_equal(at(q, 7)[32:], q[0, 0, 32:])
        np.testing.assert_allclose(at(q, 0), q[0, 0])
