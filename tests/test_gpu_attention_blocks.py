"""Caches with scales by blocks of tokens and windows with sinks, on the GPU: the
append against the oracle and its rule for scales, decode attention over both."""
import numpy as np
import pytest

import attention_oracle as ao
import attention_steps as st
from lunaflux_amd import attention, fp8, synth
from lunaflux_amd.device import DeviceError

pytestmark = pytest.mark.gpu
EPSILON = 1e-6


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def scale_of(amax):
    """The smallest power of two of 2^-100 .. 2^119 by which amax is at most 448 (fp64, exact)."""
    e = -100
    while e < 119 and amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(rt, s, qkv, rotary=None, norm=None):
    d = s.desc
    x = rt.context.upload(qkv)
    out = rt.context.upload(np.full(d.max_tokens * d.query_heads * d.head_dim, st.SENTINEL, np.uint16))
    g = [None, None] if norm is None else [st.region(rt.context.upload(n)) for n in norm]
    op = attention.bind_qk_norm_rope(rt, s.layer, s.step, st.region(x), g[0], g[1], st.region(out), st.region(s.device["k"]),
                                     st.region(s.device["v"]))
    return op, out, [x, g]


def check_append(s, before, after, values, tolerance, side):
    """values, tolerance [rows, heads, D] of the step's rows; before, after: the cache's bytes."""
    d, block = s.desc, s.desc.block_tokens
    was, was_table = s.codes(before[side].copy())
    got, table = s.codes(after[side].copy())
    want_codes, want_table, free = was.copy(), was_table.copy(), np.zeros(was.size, bool)
    for i in range(len(s.rows)):
        first, end = s.before[i], s.before[i] + s.rows[i]
        for start in range(first // block * block, end, block):
            if s.rows[i] == 0:
                continue
            lo, hi = max(first, start), min(end, start + block)
            r0 = int(s.row_offsets[i]) + lo - first
            page, slot = s.place(i, start)
            for h in range(d.kv_heads):
                v, t = values[r0:r0 + hi - lo, h], tolerance[r0:r0 + hi - lo, h]
                fine = np.where(np.isfinite(v), np.abs(v), 0.0)
                allowed = {scale_of(fine.max()), scale_of((fine + t).max()), scale_of(np.maximum(fine - t, 0).max())}
                old = np.float64(was_table[page, slot // block, h])
                if lo > start:
                    allowed = {max(a, old) for a in allowed}
                scale = np.float64(table[page, slot // block, h])
                assert scale in allowed, (i, start, h, scale, allowed)
                want_table[page, slot // block, h] = scale
                for j in range(start, hi):
                    at = s.element(page, h, slot + j - start)
                    if j < lo:  # raised
                        raised = synth.e4m3_decode(was[at:at + d.head_dim]).astype(np.float64) * (old / scale)
                        want_codes[at:at + d.head_dim] = synth.e4m3_encode(raised.astype(np.float32))
                        continue
                    code = synth.e4m3_decode(got[at:at + d.head_dim]).astype(np.float64)
                    want = v[j - lo] / scale
                    free[at:at + d.head_dim] = True
                    assert (np.isnan(code) == np.isnan(want)).all()
                    want = np.clip(np.where(np.isnan(want), 0, want), -448, 448)
                    limit = ao.rounded_e4m3(t[j - lo] / scale, want)
                    assert (np.abs(np.where(np.isnan(code), 0, code) - want) <= limit).all(), (i, j, h)
    np.testing.assert_array_equal(table, want_table)
    same = lambda a: np.where(a == 0x80, 0, a)  # noqa: E731  a zero has two codes
    np.testing.assert_array_equal(same(got[~free]), same(want_codes[~free]))


def rows_of(rng, s, amplitude=1.0):
    d = s.desc
    x = amplitude * rng.standard_normal((d.max_tokens, d.query_heads + 2 * d.kv_heads, d.head_dim)).astype(np.float32)
    return synth.bf16_bits(x)


def oracle(s, qkv, positions, rotary, norm):
    d, m = s.desc, int(s.row_offsets[-1])
    x = synth.bf16_values(qkv[:m]).astype(np.float64)
    hq, hk = d.query_heads, d.kv_heads
    g = [None, None] if norm is None else [synth.bf16_values(n).astype(np.float64) for n in norm]
    at = None if positions is None else np.asarray(positions).reshape(m, -1)
    q, qt = ao.heads(x[:, :hq], g[0], EPSILON if norm else None, at, rotary)
    k, kt = ao.heads(x[:, hq:hq + hk], g[1], EPSILON if norm else None, at, rotary)
    v = x[:, hq + hk:]
    return (q, qt), (k, kt), (v, np.zeros_like(v))


@pytest.mark.parametrize("rows,before,hq,hkv,dim,page,rotary_dim,pairing,normed", [
    ([1], [0], 1, 1, 64, 8, 0, "half", False),
    ([1, 1, 1, 1], [5, 8, 15, 16], 4, 2, 64, 8, 64, "half", True),
    ([1, 1, 1], [31, 32, 7], 10, 5, 128, 16, 128, "neighbour", True),
    ([40, 0, 17, 3], [0, 9, 30, 14], 6, 3, 128, 32, 64, "half", False),
    ([16, 33], [0, 15], 2, 1, 256, 16, 256, "half", True),
    ([100, 9], [3, 0], 3, 3, 64, 1024, 32, "neighbour", False),
    ([23, 8], [4, 8], 4, 4, 256, 8, 256, "neighbour", True),
])
def test_append(rt, rows, before, hq, hkv, dim, page, rotary_dim, pairing, normed):
    """Into an empty cache, then a next step whose rows follow, larger ones: their blocks' scales rise."""
    rng = np.random.default_rng(sum(rows) + dim)
    rotary = attention.Rotary.of_theta(1e4, rotary_dim, pairing=pairing) if rotary_dim else None
    norm = [synth.bf16_bits((1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)) for _ in range(2)] if normed else None
    m = sum(rows)
    s = st.make_step(rt, rng, rows=rows, before=before, query_heads=hq, kv_heads=hkv, head_dim=dim, page=page,
                     cache="e4m3_blocks", rotary=rotary, norm_epsilon=EPSILON if normed else None, max_tokens=m + 2,
                     spare_entries=2, positions=np.arange(m) * 7)
    for amplitude in (1.0, 300.0, 0.01):
        qkv = rows_of(rng, s, amplitude)
        op, out, keep = append(rt, s, qkv, rotary, norm)
        was = {side: a.read(np.uint8, (a.byte_count,)) for side, a in s.device.items()}
        op.launch(rt.stream, synchronous=True)
        now = {side: a.read(np.uint8, (a.byte_count,)) for side, a in s.device.items()}
        (q, qt), (k, kt), (v, vt) = oracle(s, qkv, np.arange(m) * 7, rotary, norm)
        got = st.read(s, out)
        assert (got[m:] == st.SENTINEL).all()
        limit = ao.rounded_bf16(qt, q)
        assert (np.abs(synth.bf16_values(got[:m]).astype(np.float64) - q) <= limit).all()
        check_append(s, was, now, k, kt, "k")
        check_append(s, was, now, v, vt, "v")
        # the next step's rows follow these
        s.before = [b + r for b, r in zip(s.before, s.rows)]
        if max(b + r for b, r in zip(s.before, s.rows)) > min(len(t) for t in s.tables) * page:
            break
        s.step.stage(s.row_offsets, [b + r for b, r in zip(s.before, s.rows)], s.tables, np.arange(m) * 7, prefill_rows=len(rows))


def test_append_of_the_largest_smallest_and_odd_values(rt):
    """Magnitudes at the scales' ends and at borders between two, zeros, infinities, NaN."""
    rng = np.random.default_rng(3)
    rows = [16] * 8
    s = st.make_step(rt, rng, rows=rows, before=[0] * 8, query_heads=1, kv_heads=1, head_dim=64, page=16, cache="e4m3_blocks", fill=False)
    x = np.zeros((128, 3, 64), np.float32)
    x[0:16] = 0.0
    x[16:32] = 3.3895314e38                                      # the largest bf16: cut to 448 2^119
    x[32:48] = 1e-38
    x[48:64, :, :32], x[48:64, :, 32:] = 448.0 * 2.0 ** 20, 1.0  # the border itself
    x[64:80, :, :32], x[64:80, :, 32:] = 452.0, 0.001            # just past one
    x[80:96], x[80, :, 5], x[81, :, 6], x[82, :, 7] = 0.5, np.inf, -np.inf, np.nan
    x[96:112] = rng.standard_normal((16, 3, 64)) * 2.0 ** rng.integers(-12, 1, (16, 3, 64))
    x[112:128, :, 0], x[112:128, :, 1:] = np.nan, 0.0
    qkv = synth.bf16_bits(x)
    op, out, keep = append(rt, s, qkv)
    was = {side: a.read(np.uint8, (a.byte_count,)) for side, a in s.device.items()}
    op.launch(rt.stream, synchronous=True)
    now = {side: a.read(np.uint8, (a.byte_count,)) for side, a in s.device.items()}
    values = synth.bf16_values(qkv).astype(np.float64)
    for side, head in (("k", 1), ("v", 2)):
        check_append(s, was, now, values[:, head:head + 1], np.zeros((128, 1, 64)), side)


def test_append_drops_rows_of_a_page_outside_and_of_contradicting_sequences(rt):
    rng = np.random.default_rng(4)
    s = st.make_step(rt, rng, rows=[20, 5], before=[10, 40], query_heads=2, kv_heads=2, page=8, cache="e4m3_blocks")
    qkv = rows_of(rng, s)
    _, (k, kt), (v, vt) = oracle(s, qkv, None, None, None)
    table = np.concatenate(s.tables).astype(np.int32)

    def launched():
        op, out, keep = append(rt, s, qkv)
        was = {side: a.read(np.uint8, (a.byte_count,)) for side, a in s.device.items()}
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
        return was, {side: a.read(np.uint8, (a.byte_count,)) for side, a in s.device.items()}

    for bad in (s.desc.pages, -1):
        broken = table.copy()
        broken[2] = bad                                 # tokens 16 .. 23 of sequence 0
        s.step.page_indices.copy_from_host(broken)
        was, now = launched()
        for side in ("k", "v"):
            a, ta = s.codes(was[side])
            b, tb = s.codes(now[side])
            p = s.tables[0][2]
            np.testing.assert_array_equal(ta[p], tb[p])
            for h in range(2):
                at = s.element(p, h, 0)
                np.testing.assert_array_equal(a[at:at + 8 * 64], b[at:at + 8 * 64])
            assert (ta != tb).any() or (a != b).any()
    s.step.page_indices.copy_from_host(table)
    s.step.row_offsets.copy_from_host(np.array([0, 20, 26], np.int32))      # past the batch
    s.rows[1] = 0
    was, now = launched()
    check_append(s, was, now, k, kt, "k")
    check_append(s, was, now, v, vt, "v")


def test_a_page_written_by_two_ways_refuses_to_launch(rt):
    rng = np.random.default_rng(5)
    s = st.make_step(rt, rng, rows=[4, 4], before=[0, 0], query_heads=2, kv_heads=2, page=8, cache="e4m3_blocks", spare_entries=1)
    op, out, keep = append(rt, s, rows_of(rng, s))
    for lengths, tables in (([4, 4], [[1], [1]]), ([10, 4], [[1, 1], [0]])):
        s.step.stage([0, 4, 8], lengths, tables, prefill_rows=2)
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
    s.step.stage([0, 4, 8], [12, 4], [[1, 2], [0]], prefill_rows=2)
    op.launch(rt.stream, synchronous=True)


# -- decode ------------------------------------------------------------------
def decode(rt, rng, s, again=2, amplitude=1.5):
    q = st.queries(rng, s, amplitude)
    op, out = st.bind(rt, s, q, prompts=False)
    op.launch(rt.stream, synchronous=True)
    first = st.read(s, out)
    st.check(s, first, q, range(len(s.rows)))
    for _ in range(again):
        op.launch(rt.stream, synchronous=True)
        np.testing.assert_array_equal(st.read(s, out), first)


@pytest.mark.parametrize("lengths,hq,hkv,dim,page", [
    ([1], 1, 1, 64, 8),
    ([1, 2, 7, 8, 9], 4, 2, 64, 8),
    ([31, 32, 33, 127, 128, 129], 8, 2, 128, 16),
    ([255, 1, 300], 7, 1, 128, 32),
    ([400], 17, 1, 64, 64),
    ([513, 5], 16, 1, 256, 16),
    ([260, 100, 31], 6, 3, 256, 1024),
    ([3000, 3], 4, 2, 128, 8),
])
def test_decode_over_blocks(rt, lengths, hq, hkv, dim, page):
    rng = np.random.default_rng(sum(lengths) + hq)
    n = len(lengths)
    decode(rt, rng, st.make_step(rt, rng, rows=[1] * n, before=[x - 1 for x in lengths], prefill=0, query_heads=hq, kv_heads=hkv,
                                 head_dim=dim, page=page, cache="e4m3_blocks", spare_entries=1, max_tokens=n + 2))


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "e4m3_blocks"])
@pytest.mark.parametrize("window,sinks", [(1, 1), (31, 4), (32, 32), (64, 33), (200, 130), (40, 5000), (5000, 3), (0, 4)])
def test_decode_with_sinks(rt, window, sinks, cache):
    rng = np.random.default_rng(window + sinks)
    lengths = [1, 40, 129, 390, 1700]
    decode(rt, rng, st.make_step(rt, rng, rows=[1] * 5, before=[x - 1 for x in lengths], prefill=0, page=16, query_heads=4,
                                 kv_heads=1, cache=cache, window=window, sinks=sinks))


def test_decode_with_sinks_of_many_sequences(rt):
    """More sequences than a block keeps, blocks of several pairs, and one long sequence."""
    rng = np.random.default_rng(6)
    lengths = [int(x) for x in rng.integers(1, 90, 400)]
    lengths[200] = 1500
    decode(rt, rng, st.make_step(rt, rng, rows=[1] * 400, before=[x - 1 for x in lengths], prefill=0, query_heads=2, kv_heads=2,
                                 window=1200, sinks=17, max_sequences=512), again=0)


@pytest.mark.parametrize("exponents", [(-100, -99), (100, 119), (-30, 30)])
def test_decode_over_scales_of_any_size(rt, exponents):
    rng = np.random.default_rng(7)
    s = st.make_step(rt, rng, rows=[1, 1], before=[200, 33], prefill=0, query_heads=4, kv_heads=2, cache="e4m3_blocks", page=32)
    codes, table = s.codes(s.host["v"])
    live = ~np.isnan(table)
    table[live] = 2.0 ** rng.integers(*exponents, live.sum())
    s.device["v"].copy_from_host(s.host["v"])
    decode(rt, rng, s)


def test_a_conversation(rt):
    """As a serving engine runs it: prompts in parts, then single tokens, appended and attended in turn over
    one cache of blocks; the attention of every step against the oracle over what the cache holds."""
    rng = np.random.default_rng(8)
    lengths, cuts = [37, 70], ([20, 33], [17, 37])
    s = st.make_step(rt, rng, rows=cuts[0], before=[0, 0], query_heads=4, kv_heads=2, head_dim=128, page=16, cache="e4m3_blocks",
                     fill=False, max_tokens=64, spare_entries=6, window=40, sinks=5, positions=np.zeros(53, np.int32),
                     rotary=attention.Rotary.of_theta(1e4, 128), norm_epsilon=EPSILON)
    norm = [synth.bf16_bits((1 + 0.1 * rng.standard_normal(128)).astype(np.float32)) for _ in range(2)]
    qkv = rows_of(rng, s)
    x, qa = rt.context.upload(qkv), rt.context.allocate(2 * 64 * 4 * 128)
    out = rt.context.upload(np.full(64 * 4 * 128, st.SENTINEL, np.uint16))
    k, v = (st.region(s.device[side]) for side in ("k", "v"))
    g = [st.region(rt.context.upload(n)) for n in norm]
    write = attention.bind_qk_norm_rope(rt, s.layer, s.step, st.region(x), *g, st.region(qa), k, v)
    prompt = attention.bind_paged_prefill(rt, s.layer, s.step, st.region(qa), st.region(out), k, v)
    single = attention.bind_paged_decode(rt, s.layer, s.step, st.region(qa), st.region(out), k, v)
    done = [0, 0]
    for rows, prompts in (*((c, 2) for c in cuts), *(([1, 1], 0) for _ in range(3)), ([4, 1], 1)):
        s.rows, s.before = list(rows), list(done)
        s.row_offsets = np.concatenate([[0], np.cumsum(rows)])
        done = [a + b for a, b in zip(done, rows)]
        at = np.concatenate([np.arange(b, b + r) for b, r in zip(s.before, rows)])
        s.step.stage(s.row_offsets, done, s.tables, at, prefill_rows=prompts)
        x.copy_from_host(rows_of(rng, s))
        out.copy_from_host(np.full(64 * 4 * 128, st.SENTINEL, np.uint16))
        for op in (write, prompt, single):
            op.launch(rt.stream, synchronous=False)
        rt.stream.synchronize()
        for op in (write, prompt, single):
            op.check()
        s.host = {side: a.read(np.uint8, (a.byte_count,)) for side, a in s.device.items()}
        q = qa.read(np.uint16, (64, 4, 128))
        st.check(s, st.read(s, out), q, [0, 1])
