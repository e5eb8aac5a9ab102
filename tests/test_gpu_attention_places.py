"""Decode attention and the append over caches whose token stride is long, and
steps whose page ranges overlap."""
import math

import numpy as np
import pytest

import attention_oracle as ao
from lunaflux_amd import attention, fp8, synth
from lunaflux_amd.device import DeviceError
from test_gpu_attention import region

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_tokens_a_gigabyte_apart(rt, cache):
    """Order [slot][page][head] with 2^30 bytes from slot to slot: rows 4 to 7 of a
    group of eight lie past 2^32 bytes from its first."""
    rng = np.random.default_rng(21)
    hq, hkv, dim, page, table, length = 4, 2, 64, 8, [5, 0, 4], 23
    size, dtype = (2, np.uint16) if cache == "bf16" else (1, np.uint8)
    strides = (hkv * dim, dim, (1 << 30) // size)
    scales = [np.ones(hkv, np.float32)] * 2 if cache == "bf16" else [np.array(x, np.float32) for x in ([0.03, 0.02], [0.01, 0.05])]
    layer = attention.attention_layer(rt, query_heads=hq, kv_heads=hkv, head_dim=dim, page_size=page, pages=6,
                                      max_tokens=1, max_sequences=1, table_entries=3, strides=strides, cache=cache,
                                      k_scales=scales[0], v_scales=scales[1])
    step = attention.PagedStep(rt, layer)
    step.stage([0, 1], [length], [table])
    q = synth.bf16_bits((1.5 * rng.standard_normal((1, hq, dim))).astype(np.float32))
    qa, oa = rt.context.upload(q), rt.context.allocate(2 * hq * dim)
    at = [size * (strides[0] * table[j // page] + strides[2] * (j % page)) for j in range(length)]
    caches, host = [rt.context.allocate(layer.cache_bytes) for _ in range(2)], []
    for a in caches:
        values = rng.standard_normal((length, hkv, dim)).astype(np.float32)
        codes = synth.bf16_bits(values) if cache == "bf16" else synth.e4m3_encode(values * 30)
        for j in range(length):
            a.copy_from_host(codes[j], offset=at[j])
        host.append(ao.cache_values(codes, cache))

    def check():
        out = synth.bf16_values(oa.read(np.uint16, (hq, dim))).astype(np.float64)
        for h in range(hkv):
            k, v = (x[:, h] * np.float64(s[h]) for x, s in zip(host, scales))
            want, tol = ao.decode(synth.bf16_values(q[0, 2 * h:2 * h + 2]).astype(np.float64), k, v, 1 / math.sqrt(dim))
            assert (np.abs(out[2 * h:2 * h + 2] - want) <= tol).all(), h

    decode = attention.bind_paged_decode(rt, layer, step, region(qa), region(oa), *map(region, caches))
    decode.launch(rt.stream)
    check()

    # the append puts its row (slot 6 of the last page) where decode reads it
    qkv = synth.bf16_bits(rng.standard_normal((1, hq + 2 * hkv, dim)).astype(np.float32))
    a, oq = rt.context.upload(qkv), rt.context.allocate(2 * hq * dim)
    attention.bind_qk_norm_rope(rt, layer, step, region(a), None, None, region(oq), *map(region, caches)).launch(rt.stream)
    for x, c, s, first in zip(host, caches, scales, (hq, hq + hkv)):
        x[length - 1] = ao.cache_values(c.read(dtype, (hkv, dim), offset=at[length - 1]), cache)
        rows = synth.bf16_values(qkv[0, first:first + hkv]).astype(np.float64)
        steps = rows / s[:, None].astype(np.float64)
        limit = 0.0 if cache == "bf16" else ao.rounded_e4m3(np.abs(steps) * 2 * ao.U32, steps)
        assert (np.abs(x[length - 1] - np.clip(steps, -448, 448)) <= limit).all()
    decode.launch(rt.stream)
    check()


@pytest.mark.parametrize("sequences", [63, 64, 300])
def test_overlapping_page_ranges_past_the_items_are_reported(rt, sequences):
    """Every other sequence claims the whole of a table of 2^31 keys, 2^26 tiles each:
    nothing is written, and the launch says so."""
    entries, dim = (1 << 21) - 2, 64
    layer = attention.attention_layer(rt, query_heads=1, kv_heads=1, head_dim=dim, page_size=1024, pages=2,
                                      max_tokens=sequences, max_sequences=sequences, table_entries=entries)
    step = attention.PagedStep(rt, layer)
    step.page_indices.copy_from_host(np.zeros(entries, np.int32))
    step.stage(np.arange(sequences + 1), [1] * sequences, [[0]] * sequences)
    caches = [rt.context.upload(np.zeros(layer.cache_bytes, np.uint8)) for _ in range(2)]
    q = rt.context.upload(np.zeros(sequences * dim, np.uint16))
    out = rt.context.upload(np.full(sequences * dim, 0x7FA5, np.uint16))
    op = attention.bind_paged_decode(rt, layer, step, region(q), region(out), *map(region, caches))
    step.lengths.copy_from_host(np.full(sequences, entries * 1024, np.int32))
    ends = np.zeros(sequences + 1, np.int32)
    ends[1::2] = entries
    step.page_offsets.copy_from_host(ends)
    with pytest.raises(DeviceError):
        op.launch(rt.stream)
    op.check()
    assert (out.read(np.uint16, (sequences * dim,)) == 0x7FA5).all()
