"""Attention of prompts over the paged cache on the GPU against the 64-bit oracle,
every value within the bound that attention_oracle.decode derives (its weights
are bf16 values, as there); steps as attention_steps.py makes them."""
import numpy as np
import pytest

import attention_steps as st
from lunaflux_amd import fp8, synth
from lunaflux_amd.device import DeviceError

pytestmark = pytest.mark.gpu
CACHES = ["bf16", "e4m3", "e4m3_blocks"]


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def run(rt, rng, s, amplitude=1.5, again=1):
    q = st.queries(rng, s, amplitude)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    first = st.read(s, out)
    st.check(s, first, q, range(len(s.rows)))
    for _ in range(again):
        op.launch(rt.stream, synchronous=True)
        np.testing.assert_array_equal(st.read(s, out), first)


# rows and tokens before around tiles (32, 64, 128, 256) and pages; one to many heads a key head
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("rows,before,hq,hkv,dim,page", [
    ([1], [0], 1, 1, 64, 8),
    ([1, 2, 7, 0, 33], [0, 5, 0, 9, 31], 4, 2, 64, 8),
    ([64, 65, 63], [0, 1, 70], 4, 4, 128, 16),
    ([257], [0], 1, 1, 64, 16),
    ([40, 3], [17, 300], 7, 1, 128, 32),            # 36 tokens a tile
    ([5, 9], [60, 0], 40, 1, 128, 128),             # six tokens a tile
    ([3, 1], [30, 64], 300, 1, 64, 16),             # a token's heads in two tiles
    ([33, 6], [95, 0], 16, 2, 256, 16),
    ([2, 3], [10, 0], 130, 1, 256, 1024),           # heads of 256, a token's heads in two tiles
    ([130], [129], 6, 3, 256, 64),
])
def test_prompts(rt, rows, before, hq, hkv, dim, page, cache):
    rng = np.random.default_rng(sum(rows) + hq + dim)
    run(rt, rng, st.make_step(rt, rng, rows=rows, before=before, query_heads=hq, kv_heads=hkv, head_dim=dim, page=page,
                              cache=cache, spare_entries=1, max_tokens=sum(rows) + 3))


# long enough to be cut between blocks, and joined
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("rows,before,hq,hkv,dim", [
    ([3], [5000], 4, 1, 128), ([1, 20], [4000, 1100], 2, 1, 64), ([300], [900], 4, 2, 128), ([9, 2], [3001, 1], 8, 2, 256),
    ([600, 1, 31], [0, 1500, 2], 2, 2, 64),
])
def test_prompts_cut_between_blocks(rt, rows, before, hq, hkv, dim, cache):
    rng = np.random.default_rng(sum(rows) + sum(before))
    run(rt, rng, st.make_step(rt, rng, rows=rows, before=before, query_heads=hq, kv_heads=hkv, head_dim=dim, page=16, cache=cache),
        again=3)


@pytest.mark.parametrize("cache", ["bf16", "e4m3_blocks"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (63, 64), (64, 1), (100, 37), (128, 130), (300, 2000), (5000, 9), (0, 5)])
def test_windows_and_sinks(rt, window, sinks, cache):
    rng = np.random.default_rng(window + sinks)
    run(rt, rng, st.make_step(rt, rng, rows=[150, 1, 40], before=[300, 700, 0], query_heads=4, kv_heads=1, page=16, cache=cache,
                              window=window, sinks=sinks))


def test_a_long_window_with_sinks_is_cut(rt):
    rng = np.random.default_rng(5)
    run(rt, rng, st.make_step(rt, rng, rows=[40], before=[4000], query_heads=2, kv_heads=1, page=8, window=2500, sinks=700))


@pytest.mark.parametrize("strides", [
    lambda pages: (2 * 16 * 64, 64, 2 * 64),                      # [page][slot][head]
    lambda pages: (64, pages * 16 * 64, pages * 64),              # [head][slot][page]
    lambda pages: (2 * 16 * 80 + 16, 16 * 80, 80),                # padded rows and pages
])
@pytest.mark.parametrize("cache", CACHES)
def test_strides(rt, strides, cache):
    rng = np.random.default_rng(6)
    run(rt, rng, st.make_step(rt, rng, rows=[70, 3], before=[40, 200], page=16, cache=cache, strides=strides))


@pytest.mark.parametrize("amplitude,scale", [(0.0, None), (30.0, None), (1.5, -0.2), (1.5, 0.0)])
def test_flat_peaked_and_negative_scores(rt, amplitude, scale):
    rng = np.random.default_rng(7)
    run(rt, rng, st.make_step(rt, rng, rows=[150], before=[65], page=16, head_dim=128, softmax_scale=scale), amplitude)


@pytest.mark.parametrize("cache", ["bf16", "e4m3_blocks"])
@pytest.mark.parametrize("growing", [True, False])
def test_scores_that_change_along_the_keys(rt, growing, cache):
    """Scores that pass the first tile's maximum by far, and ones that fall short of it: later keys are multiples."""
    rng = np.random.default_rng(15)
    s = st.make_step(rt, rng, rows=[70, 5], before=[400, 1200], page=16, cache=cache)
    codes, table = s.codes(s.host["k"])
    for i in range(2):
        for j in range(s.before[i] + s.rows[i]):
            page, slot = s.place(i, j)
            step = 2.0 ** ((j // 64 if growing else 8 - j // 64) % 9)
            if table is not None:
                table[page, slot // 16] = step * 2.0 ** -6
                continue
            for h in range(2):
                at = s.element(page, h, slot)
                codes[at:at + 64] = synth.bf16_bits(synth.bf16_values(codes[at:at + 64]) * np.float32(step))
    s.device["k"].copy_from_host(s.host["k"])
    run(rt, rng, s)


def test_many_sequences(rt):
    """More sequences than threads, few rows each."""
    rng = np.random.default_rng(8)
    rows, before = (list(map(int, rng.integers(0, hi, 600))) for hi in (4, 30))
    run(rt, rng, st.make_step(rt, rng, rows=rows, before=before, query_heads=2, kv_heads=1, max_sequences=700))


def test_only_the_prompts_of_a_mixed_step(rt):
    rng = np.random.default_rng(9)
    s = st.make_step(rt, rng, rows=[7, 9, 1, 1], before=[13, 0, 32, 63], prefill=2, max_tokens=24)
    q = st.queries(rng, s)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    first = st.read(s, out)
    st.check(s, first, q, [0, 1])
    decode, same = st.bind(rt, s, q, prompts=False)
    decode.launch(rt.stream, synchronous=True)
    st.check(s, st.read(s, same), q, [2, 3])


@pytest.mark.parametrize("cache", ["bf16", "e4m3_blocks"])
def test_sequences_that_share_pages(rt, cache):
    """A common beginning that is cached once, read by two prompts and a decoded sequence; one of its pages stands
    in a table twice."""
    rng = np.random.default_rng(16)
    s = st.make_step(rt, rng, rows=[9, 70, 1], before=[80, 64, 90], prefill=2, page=16, cache=cache)
    for i in (1, 2):
        s.tables[i][:4] = s.tables[0][:4]
    s.tables[2][2] = s.tables[2][1]
    s.step.stage(s.row_offsets, [89, 134, 91], s.tables, prefill_rows=2)
    q = st.queries(rng, s)
    for prompts, sequences in ((True, [0, 1]), (False, [2])):
        op, out = st.bind(rt, s, q, prompts)
        op.launch(rt.stream, synchronous=True)
        st.check(s, st.read(s, out), q, sequences)


def test_two_bindings_on_two_streams(rt):
    """Calls of two layers at once, each with a workspace of its own, many times over; cut prompts in both."""
    rng = np.random.default_rng(17)
    steps = [st.make_step(rt, rng, rows=[33, 2], before=[2500, 1800], query_heads=4, kv_heads=2, page=16, cache=cache)
             for cache in ("bf16", "e4m3_blocks")]
    queries = [st.queries(rng, s) for s in steps]
    bound = [st.bind(rt, s, q) for s, q in zip(steps, queries)]
    streams = [rt.stream, rt.context.create_stream()]
    for _ in range(8):
        for (op, _), stream in zip(bound, streams):
            op.launch(stream, synchronous=False)
    for stream in streams:
        stream.synchronize()
    for s, q, (op, out) in zip(steps, queries, bound):
        op.check()
        st.check(s, st.read(s, out), q, [0, 1])


def test_a_step_without_prompts_writes_nothing(rt):
    rng = np.random.default_rng(10)
    s = st.make_step(rt, rng, rows=[1, 1], before=[3, 40], prefill=0)
    q = st.queries(rng, s)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    assert (st.read(s, out) == st.SENTINEL).all()
    s.step.stage([0], [], [])
    op.launch(rt.stream, synchronous=True)
    assert (st.read(s, out) == st.SENTINEL).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinities_and_nan_reach_the_rows_that_count_them(rt, dim):
    """A NaN key or odd value at token 50 reaches the rows from 50 on alone."""
    rng = np.random.default_rng(11)
    s = st.make_step(rt, rng, rows=[90] * 5, before=[0] * 5, query_heads=2, kv_heads=1, head_dim=dim, page=16)
    nan, inf = 0x7FC0, 0x7F80
    for side, i, token, column, bits in (("k", 0, 50, 3, nan), ("v", 1, 50, 3, nan), ("v", 2, 50, 3, inf),
                                         ("v", 3, 50, 3, inf), ("v", 3, 70, 3, inf | 0x8000)):
        page, slot = s.place(i, token)
        s.codes(s.host[side])[0][s.element(page, 0, slot) + column] = bits
        s.device[side].copy_from_host(s.host[side])
    q = st.queries(rng, s)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    got = synth.bf16_values(st.read(s, out)).reshape(5, 90, 2, dim)
    for i in range(5):
        assert np.isfinite(got[i, :50]).all(), i
        assert np.isfinite(np.delete(got[i], 3, axis=2)).all() or i == 0, i
    assert np.isnan(got[0, 50:]).all() and np.isnan(got[1, 50:, :, 3]).all()
    assert (got[2, 50:, :, 3] == np.inf).all() and (got[3, 50:70, :, 3] == np.inf).all() and np.isnan(got[3, 70:, :, 3]).all()
    assert np.isfinite(got[4]).all()


def test_a_page_outside_the_cache_is_left_out(rt):
    rng = np.random.default_rng(12)
    s = st.make_step(rt, rng, rows=[60, 30], before=[40, 0], page=16)
    q = st.queries(rng, s)
    table = np.concatenate(s.tables).astype(np.int32)
    for bad in (s.desc.pages, -1, 2 ** 31 - 1):
        table[2] = bad                     # tokens 32 .. 47 of sequence 0
        s.step.page_indices.copy_from_host(table)
        op, out = st.bind(rt, s, q)
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
        st.check(s, st.read(s, out), q, [0, 1], hidden=lambda i, j: i == 0 and 32 <= j < 48)
        op.check()                         # reported once


def test_sequences_that_contradict_the_step_are_left_out(rt):
    rng = np.random.default_rng(13)
    s = st.make_step(rt, rng, rows=[20, 24], before=[20, 0], page=8)
    q = st.queries(rng, s)

    def launched(left):
        op, out = st.bind(rt, s, q)
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
        st.check(s, st.read(s, out), q, left)

    for lengths in ([19, 24], [41, 24], [2 ** 31 - 1, 24], [-5, 24]):   # fewer tokens than rows, more than the pages hold
        s.step.lengths.copy_from_host(np.array(lengths, np.int32))
        launched([1])
    s.step.lengths.copy_from_host(np.array([40, 24], np.int32))
    s.step.page_offsets.copy_from_host(np.array([0, 5, 2 ** 30], np.int32))
    launched([0])
    s.step.page_offsets.copy_from_host(np.array([0, 5, 8], np.int32))
    for offsets in ([0, 20, 45], [0, 20, -1], [0, 20, 2 ** 31 - 1]):
        s.step.row_offsets.copy_from_host(np.array(offsets, np.int32))
        launched([0])


def test_past_32_bit_offsets(rt):
    """Pages of half a gigabyte apart: offsets past 2^31 elements and 2^32 bytes."""
    from lunaflux_amd import attention
    rng = np.random.default_rng(14)
    stride, page, dim = 1 << 29, 16, 64
    layer = attention.attention_layer(rt, query_heads=4, kv_heads=2, head_dim=dim, page_size=page, pages=6, max_tokens=9,
                                      max_sequences=1, table_entries=3, strides=(stride, page * dim, dim))
    caches = {side: rt.context.allocate(layer.cache_bytes) for side in ("k", "v")}
    step = attention.PagedStep(rt, layer)
    table = [5, 0, 4]
    step.stage([0, 9], [41], [table], prefill_rows=1)
    small = st.make_step(rt, rng, rows=[9], before=[32], page=page)   # the same contents in a cache of three pages and two
    s = st.Step(layer, step, "bf16", [9], [32], np.array([0, 9]), [np.array(table)], host=small.host, device=caches)
    for side in ("k", "v"):
        for e, p in enumerate(table):
            codes = small.codes(small.host[side])[0]
            at = small.element(small.tables[0][e], 0, 0)
            caches[side].copy_from_host(codes[at:at + 2 * page * dim], offset=2 * p * stride)
    q = st.queries(rng, s)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    st.check(small, st.read(s, out), q, [0])
