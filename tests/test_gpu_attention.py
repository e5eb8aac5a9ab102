"""Attention between the projections on the GPU against the 64-bit oracle
(attention_oracle.py): every value within the bound derived there. Cache places
that no live key occupies hold NaN, page-table entries that no live key needs
hold -1, and outputs start as a sentinel, so a read or write beside the live
ones shows."""
import math
from dataclasses import dataclass, field

import numpy as np
import pytest

import attention_oracle as ao
from lunaflux_amd import _abi, attention, fp8, synth
from lunaflux_amd.device import DeviceError

pytestmark = pytest.mark.gpu

SENTINEL = 0x7FA5  # a bf16 NaN


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def region(a):
    return a.region(0, a.byte_count, 256)


@dataclass
class Setup:
    """A layer with a filled cache and a staged step."""
    layer: attention.AttentionLayer
    step: attention.PagedStep
    kind: str
    scales: tuple
    k: object = None
    v: object = None
    k_host: np.ndarray = None     # the caches as uploaded: codes, flat
    v_host: np.ndarray = None
    at: np.ndarray = None         # element offset of [page, head, slot]
    tables: list = field(default_factory=list)


def build(rt, rng, *, lengths, row_offsets=None, query_heads=4, kv_heads=2, head_dim=64, page=8, cache="bf16",
          strides=None, live=None, prefill=0, max_tokens=None, max_sequences=None, positions=None, spare_entries=0,
          amplitude=1.0, scales=None, **constants):
    """lengths: tokens per sequence with the step's rows; live: cached tokens
    that get values (default: all), the rest of every page stays NaN."""
    n = len(lengths)
    row_offsets = np.arange(n + 1) if row_offsets is None else np.asarray(row_offsets)
    counts = [-(-int(x) // page) + spare_entries for x in lengths]
    pool = sum(counts) + 2
    order = rng.permutation(pool)[:sum(counts)]
    tables = [order[sum(counts[:i]):sum(counts[:i + 1])].astype(np.int32) for i in range(n)]
    if scales is None and cache == "e4m3":
        scales = (rng.uniform(0.01, 0.05, kv_heads).astype(np.float32), rng.uniform(0.01, 0.05, kv_heads).astype(np.float32))
    layer = attention.attention_layer(
        rt, query_heads=query_heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page, pages=pool, cache=cache,
        max_tokens=max_tokens or max(1, int(row_offsets[-1])), max_sequences=max_sequences or max(1, n),
        table_entries=max(1, sum(counts)), strides=strides(pool) if callable(strides) else strides,
        k_scales=None if scales is None else scales[0], v_scales=None if scales is None else scales[1], **constants)
    step = attention.PagedStep(rt, layer)
    s = Setup(layer, step, cache, scales or (np.ones(kv_heads, np.float32),) * 2)
    d = layer.desc
    dtype, nan = (np.uint16, SENTINEL) if cache == "bf16" else (np.uint8, 0x7F)
    elements = layer.cache_bytes // np.dtype(dtype).itemsize
    p, h, t = np.meshgrid(np.arange(pool), np.arange(kv_heads), np.arange(page), indexing="ij")
    s.at = p * d.page_stride + h * d.head_stride + t * d.token_stride
    window = constants.get("window", 0)
    for name in ("k", "v"):
        host = np.full(elements, nan, dtype)
        for i, length in enumerate(lengths if live is None else live):
            first = max(0, lengths[i] - window) if window else 0
            for j in range(first, int(length)):
                values = amplitude * rng.standard_normal((kv_heads, head_dim)).astype(np.float32)
                codes = synth.bf16_bits(values) if cache == "bf16" else synth.e4m3_encode(values * 30)
                for head in range(kv_heads):
                    at = s.at[tables[i][j // page], head, j % page]
                    host[at:at + head_dim] = codes[head]
        setattr(s, name + "_host", host)
        setattr(s, name, rt.context.upload(host))
    s.tables = [x.copy() for x in tables]
    for i, x in enumerate(tables):  # entries no live key needs
        x[-(-int(lengths[i]) // page):] = -1
        if window:
            x[:max(0, int(lengths[i]) - window) // page] = -1
    step.stage(row_offsets, lengths, tables, positions, prefill_rows=prefill)
    return s


def cached(s, host, sequence, head, keys):
    d, page = s.layer.desc, s.layer.desc.page_size
    rows = [host[a:a + d.head_dim] for a in (s.at[s.tables[sequence][j // page], head, j % page] for j in keys)]
    return ao.cache_values(np.stack(rows), s.kind) if rows else np.zeros((0, d.head_dim))


def run_decode(rt, s, q_bits, expect=True):
    d = s.layer.desc
    qa = rt.context.allocate(d.max_tokens * d.query_heads * d.head_dim * 2)
    qa.copy_from_host(q_bits)
    oa = rt.context.upload(np.full(d.max_tokens * d.query_heads * d.head_dim, SENTINEL, np.uint16))
    op = attention.bind_paged_decode(rt, s.layer, s.step, region(qa), region(oa), region(s.k), region(s.v))
    if expect:
        op.launch(rt.stream, synchronous=True)
    return op, oa


def read_out(s, oa):
    d = s.layer.desc
    return oa.read(np.uint16, (d.max_tokens, d.query_heads, d.head_dim))


def check_decode(s, out_bits, q_bits, lengths, sequences=None, row_of=None, keys_of=None):
    d = s.layer.desc
    group, written = d.query_heads // d.kv_heads, np.zeros(d.max_tokens, bool)
    worst = 0.0
    for i in range(len(lengths)) if sequences is None else sequences:
        row = i if row_of is None else row_of[i]
        first = max(0, lengths[i] - d.window) if d.window else 0
        keys = range(first, lengths[i]) if keys_of is None else keys_of(i)
        written[row] = True
        for h in range(d.kv_heads):
            k = cached(s, s.k_host, i, h, keys) * np.float64(s.scales[0][h])
            v = cached(s, s.v_host, i, h, keys) * np.float64(s.scales[1][h])
            heads = slice(h * group, (h + 1) * group)
            want, tol = ao.decode(synth.bf16_values(q_bits[row, heads]).astype(np.float64), k, v, float(d.softmax_scale))
            got = synth.bf16_values(out_bits[row, heads]).astype(np.float64)
            assert np.isfinite(got).all(), (i, h)
            over = np.abs(got - want) - tol
            assert (over <= 0).all(), (i, h, over.max(), np.abs(got - want).max())
            worst = max(worst, float((np.abs(got - want) / tol).max()) if len(want) and tol.any() else 0.0)
    assert (out_bits[~written] == SENTINEL).all()
    return worst


def queries(rng, s, amplitude=1.5):
    d = s.layer.desc
    return synth.bf16_bits((amplitude * rng.standard_normal((d.max_tokens, d.query_heads, d.head_dim))).astype(np.float32))


# lengths around tile (32, 128) and page edges; one to many heads a key head
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,hq,hkv,dim,page", [
    ([1], 1, 1, 64, 8),
    ([1, 2, 7, 8, 9], 4, 2, 64, 8),
    ([31, 32, 33, 127, 128, 129], 8, 2, 128, 16),
    ([255, 1, 300], 7, 1, 128, 32),
    ([400], 17, 1, 64, 64),            # a second head tile of one row
    ([130, 77], 40, 1, 128, 128),      # three head tiles
    ([513, 5], 16, 1, 256, 16),
    ([260, 100, 31], 6, 3, 256, 1024),
    ([1500, 3], 4, 4, 128, 8),
])
def test_decode(rt, lengths, hq, hkv, dim, page, cache):
    rng = np.random.default_rng(len(lengths) * 1000 + hq + dim)
    s = build(rt, rng, lengths=lengths, query_heads=hq, kv_heads=hkv, head_dim=dim, page=page, cache=cache,
              spare_entries=1, max_tokens=len(lengths) + 2)
    q = queries(rng, s)
    op, oa = run_decode(rt, s, q)
    first = read_out(s, oa)
    check_decode(s, first, q, lengths)
    for _ in range(3):  # the workspace is at rest after a launch: the same bits again
        op.launch(rt.stream, synchronous=True)
        np.testing.assert_array_equal(read_out(s, oa), first)


@pytest.mark.parametrize("window", [1, 31, 32, 33, 128, 200, 5000])
def test_decode_window(rt, window):
    rng = np.random.default_rng(window)
    lengths = [1, 40, 129, 390]
    s = build(rt, rng, lengths=lengths, page=16, window=window, query_heads=4, kv_heads=1)
    q = queries(rng, s)
    check_decode(s, read_out(s, run_decode(rt, s, q)[1]), q, lengths)


@pytest.mark.parametrize("strides", [
    lambda pages: (2 * 16 * 64, 64, 2 * 64),                      # [page][slot][head]
    lambda pages: (64, pages * 16 * 64, pages * 64),              # [head][slot][page]
    lambda pages: (2 * 16 * 80 + 16, 16 * 80, 80),                # padded rows and pages
])
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_decode_strides(rt, strides, cache):
    rng = np.random.default_rng(5)
    lengths = [70, 200]
    s = build(rt, rng, lengths=lengths, page=16, cache=cache, strides=strides)
    q = queries(rng, s)
    check_decode(s, read_out(s, run_decode(rt, s, q)[1]), q, lengths)


@pytest.mark.parametrize("longest", [20, 512, 513, 1024, 1025])
@pytest.mark.parametrize("sequences,hq,hkv", [(3, 4, 2), (20, 2, 2), (150, 16, 4)])
def test_decode_by_pairs_or_by_tiles(rt, longest, sequences, hq, hkv):
    """One sequence of `longest` keys among short ones, on both sides of the
    lengths up to which blocks take whole (sequence, head) pairs."""
    rng = np.random.default_rng(longest + sequences)
    lengths = [int(x) for x in rng.integers(1, 40, sequences)]
    lengths[sequences // 2] = longest
    s = build(rt, rng, lengths=lengths, query_heads=hq, kv_heads=hkv, page=16)
    q = queries(rng, s)
    op, oa = run_decode(rt, s, q)
    check_decode(s, read_out(s, oa), q, lengths)
    op.check()


def test_decode_of_many_sequences(rt):
    """More pairs than blocks: blocks hold whole pairs and ends of others."""
    rng = np.random.default_rng(9)
    lengths = [int(x) for x in rng.integers(1, 60, 700)]
    s = build(rt, rng, lengths=lengths, query_heads=4, kv_heads=2, max_sequences=2048, max_tokens=900)
    q = queries(rng, s)
    check_decode(s, read_out(s, run_decode(rt, s, q)[1]), q, lengths)


def test_decode_after_prefill_rows(rt):
    """A mixed step: only the decoded sequences' rows are written."""
    rng = np.random.default_rng(10)
    lengths, row_offsets = [20, 9, 33, 64], [0, 7, 16, 17, 18]
    s = build(rt, rng, lengths=lengths, row_offsets=row_offsets, prefill=2, max_tokens=24)
    q = queries(rng, s)
    check_decode(s, read_out(s, run_decode(rt, s, q)[1]), q, lengths, sequences=[2, 3], row_of=row_offsets)


def test_decode_without_sequences_writes_nothing(rt):
    rng = np.random.default_rng(11)
    s = build(rt, rng, lengths=[3])
    s.step.stage([0], [], [])
    q = queries(rng, s)
    assert (read_out(s, run_decode(rt, s, q)[1]) == SENTINEL).all()


def test_decode_row_without_keys_is_zero(rt):
    rng = np.random.default_rng(12)
    s = build(rt, rng, lengths=[40, 50, 60])
    s.step.lengths.copy_from_host(np.array([40, 0, 60], np.int32))
    q = queries(rng, s)
    out = read_out(s, run_decode(rt, s, q)[1])
    assert (out[1] == 0).all()
    check_decode(s, out, q, [40, 0, 60])


@pytest.mark.parametrize("amplitude", [0.0, 30.0])
def test_decode_flat_and_peaked_scores(rt, amplitude):
    """All scores equal, and scores in the hundreds (one key takes nearly all)."""
    rng = np.random.default_rng(13)
    lengths = [700, 65]
    s = build(rt, rng, lengths=lengths, page=16, head_dim=128)
    q = queries(rng, s, amplitude)
    check_decode(s, read_out(s, run_decode(rt, s, q)[1]), q, lengths)


def test_decode_of_infinities_and_nan(rt):
    """A NaN key or value of a live key reaches the rows that read it, and only those."""
    rng = np.random.default_rng(14)
    lengths = [40, 40, 40, 40]
    s = build(rt, rng, lengths=lengths, query_heads=2, kv_heads=1)
    nan, inf = 0x7FC0, 0x7F80
    for host, device, i, bits in ((s.k_host, s.k, 0, nan), (s.v_host, s.v, 1, nan), (s.v_host, s.v, 2, inf)):
        host[s.at[s.tables[i][20 // 8], 0, 20 % 8] + 3] = bits
        device.copy_from_host(host)
    q = queries(rng, s)
    out = synth.bf16_values(read_out(s, run_decode(rt, s, q)[1]))
    assert np.isnan(out[0]).all()
    assert np.isnan(out[1, :, 3]).all() and np.isfinite(np.delete(out[1], 3, axis=1)).all()
    assert (out[2, :, 3] == np.inf).all() and np.isfinite(np.delete(out[2], 3, axis=1)).all()
    assert np.isfinite(out[3]).all()


def test_decode_leaves_out_a_page_outside_the_cache(rt):
    rng = np.random.default_rng(15)
    lengths = [100, 30]
    s = build(rt, rng, lengths=lengths, page=16)
    pool = s.layer.desc.pages
    table = np.concatenate(s.tables).astype(np.int32)
    for bad in (pool, -1, 2 ** 31 - 1):
        table[2] = bad                     # keys 32 .. 47 of sequence 0
        s.step.page_indices.copy_from_host(table)
        q = queries(rng, s)
        op, oa = run_decode(rt, s, q, expect=False)
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
        check_decode(s, read_out(s, oa), q, lengths,
                     keys_of=lambda i: [j for j in range(lengths[i]) if i or not 32 <= j < 48])
        op.check()                         # reported once


def test_decode_cuts_steps_that_contradict_the_descriptor(rt):
    """Lengths past the pages, offsets past the table, rows past the batch: cut, and reported."""
    rng = np.random.default_rng(16)
    lengths = [40, 24]
    s = build(rt, rng, lengths=lengths, page=8)
    q = queries(rng, s)

    def launched():
        op, oa = run_decode(rt, s, q, expect=False)
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
        return read_out(s, oa)

    s.step.lengths.copy_from_host(np.array([2 ** 31 - 1, 24], np.int32))
    check_decode(s, launched(), q, lengths)          # cut to its five pages
    s.step.lengths.copy_from_host(np.array([-3, 24], np.int32))
    check_decode(s, launched(), q, [0, 24])
    s.step.lengths.copy_from_host(np.array(lengths, np.int32))
    s.step.page_offsets.copy_from_host(np.array([0, 5, 2 ** 30], np.int32))
    check_decode(s, launched(), q, [40, 0])
    s.step.page_offsets.copy_from_host(np.array([0, 5, 8], np.int32))
    s.step.row_offsets.copy_from_host(np.array([0, 77, 78], np.int32))
    check_decode(s, launched(), q, lengths, sequences=[0])


def test_decode_past_32_bit_offsets(rt):
    """Pages of half a gigabyte apart: offsets past 2^31 elements and 2^32 bytes."""
    rng = np.random.default_rng(17)
    stride, page, dim = 1 << 29, 16, 64
    layer = attention.attention_layer(rt, query_heads=4, kv_heads=2, head_dim=dim, page_size=page, pages=6, max_tokens=1,
                                      max_sequences=1, table_entries=3, strides=(stride, page * dim, dim))
    k, v = rt.context.allocate(layer.cache_bytes), rt.context.allocate(layer.cache_bytes)
    step = attention.PagedStep(rt, layer)
    table, length = [5, 0, 4], 41
    step.stage([0, 1], [length], [table])
    s = Setup(layer, step, "bf16", (np.ones(2, np.float32),) * 2, k, v)
    host = {}
    for name, a in (("k", k), ("v", v)):
        for p in table:
            bits = synth.bf16_bits(rng.standard_normal((2, page, dim)).astype(np.float32))
            a.copy_from_host(bits, offset=2 * p * stride)
            host[name, p] = synth.bf16_values(bits).astype(np.float64)
    q = queries(rng, s)
    out = synth.bf16_values(read_out(s, run_decode(rt, s, q)[1]))[0].astype(np.float64)
    for h in range(2):
        kk, vv = (np.concatenate([host[name, p][h] for p in table])[:length] for name in ("k", "v"))
        want, tol = ao.decode(synth.bf16_values(q[0, 2 * h:2 * h + 2]).astype(np.float64), kk, vv, 1 / math.sqrt(dim))
        assert (np.abs(out[2 * h:2 * h + 2] - want) <= tol).all()
    # the append's side of the same offsets: position 40 is slot 8 of page 4
    qkv = synth.bf16_bits(rng.standard_normal((1, 8, dim)).astype(np.float32))
    a, oq = rt.context.upload(qkv), rt.context.allocate(1 * 4 * dim * 2)
    attention.bind_qk_norm_rope(rt, layer, step, region(a), None, None, region(oq), region(k), region(v)).launch(rt.stream)
    for cache, first in ((k, 4), (v, 6)):
        for h in range(2):
            got = cache.read(np.uint16, (dim,), offset=2 * (4 * stride + h * page * dim + 8 * dim))
            np.testing.assert_array_equal(got, qkv[0, first + h])


# ---- norm, rotation, append --------------------------------------------------------

def check_write(rt, rng, *, before, rows, hq=4, hkv=2, dim=64, page=8, cache="bf16", norm=None, rotary=None, extra_rows=0,
                positions=None, x=None, **kw):
    row_offsets = np.concatenate([[0], np.cumsum(rows)]).astype(int)
    m = int(row_offsets[-1])
    axes = 1 if rotary is None else rotary.axes
    if positions is None:
        positions = rng.integers(0, 200000, (m, axes))
    lengths = [b + r for b, r in zip(before, rows)]
    s = build(rt, rng, lengths=lengths, row_offsets=row_offsets, query_heads=hq, kv_heads=hkv, head_dim=dim, page=page,
              cache=cache, live=before, prefill=len(rows), positions=positions, max_tokens=max(1, m) + extra_rows,
              norm_epsilon=norm, rotary=rotary, **kw)
    heads = hq + 2 * hkv
    x = rng.standard_normal((m, heads, dim)) * 2 if x is None else x
    bits = np.full((max(1, m) + extra_rows, heads, dim), 0x7FC0, np.uint16)
    bits[:m] = synth.bf16_bits(np.asarray(x, np.float32))
    g = [synth.bf16_bits(rng.uniform(0.5, 1.5, dim).astype(np.float32)) for _ in range(2)]
    ga = [rt.context.upload(b) for b in g]
    qkv = rt.context.upload(bits)
    oq = rt.context.upload(np.full(bits.shape[0] * hq * dim, SENTINEL, np.uint16))
    if extra_rows:  # rows behind the last sequence
        counts = s.step.counts.read(np.int32, (5,))
        counts[3] += extra_rows
        s.step.counts.copy_from_host(counts)
    op = attention.bind_qk_norm_rope(rt, s.layer, s.step, region(qkv), region(ga[0]) if norm is not None else None,
                                     region(ga[1]) if norm is not None else None, region(oq), region(s.k), region(s.v))
    op.launch(rt.stream, synchronous=True)
    x64 = synth.bf16_values(bits[:m]).astype(np.float64)
    gv = [synth.bf16_values(b).astype(np.float64) for b in g]
    qw, qt = ao.heads(x64[:, :hq], gv[0], norm, positions.reshape(m, axes), rotary)
    kw_, kt = ao.heads(x64[:, hq:hq + hkv], gv[1], norm, positions.reshape(m, axes), rotary)
    got = oq.read(np.uint16, (bits.shape[0], hq, dim))
    assert (got[m:] == SENTINEL).all()
    assert (np.abs(synth.bf16_values(got[:m]) - qw) <= ao.rounded_bf16(qt, qw)).all()
    dtype = np.uint16 if cache == "bf16" else np.uint8
    for name, want, tol, heads_at in (("k", kw_, kt, 0), ("v", x64[:, hq + hkv:], 0.0, 1)):
        host = getattr(s, name + "_host").copy()
        now = getattr(s, name).read(dtype, host.shape)
        for i, b in enumerate(before):
            for r in range(rows[i]):
                j, row = b + r, row_offsets[i] + r
                for h in range(hkv):
                    at = s.at[s.tables[i][j // page], h, j % page]
                    value = ao.cache_values(now[at:at + dim], cache)
                    w, t = want[row, h], np.broadcast_to(tol, want.shape)[row, h] if np.ndim(tol) else np.zeros(dim)
                    if cache == "bf16":
                        limit = ao.rounded_bf16(t, w) if np.ndim(tol) else np.zeros(dim)   # values are copied
                    else:
                        scale = np.float64(s.scales[heads_at][h])
                        w, t = np.clip(w / scale, -448, 448), t / scale + np.abs(w / scale) * 2.0 ** -22
                        limit = ao.rounded_e4m3(t, w)
                    assert (np.abs(value - w) <= limit).all(), (name, i, r, h, np.abs(value - w).max())
                    host[at:at + dim] = now[at:at + dim]
        np.testing.assert_array_equal(now, host)    # nothing else was written
    return s, op


R = attention.Rotary


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,dim,page,norm,rotary", [
    (4, 2, 64, 8, 1e-6, R.of_theta(10000.0, 64)),
    (4, 2, 64, 8, None, None),
    (7, 1, 128, 16, 1e-5, R.of_theta(500000.0, 128)),
    (5, 5, 128, 8, None, R.of_theta(10000.0, 128, pairing="neighbour")),
    (3, 1, 256, 64, 1e-6, R.of_theta(10000.0, 128)),                       # half of the head turns
    (4, 4, 64, 16, 1e-6, R.of_theta(10000.0, 16, pairing="neighbour")),
    (6, 2, 128, 32, None, R.of_theta(10000.0, 128, (16, 24, 24))),         # time, height, width
    (2, 1, 64, 8, 0.0, R(np.linspace(0.0, 0.5, 24), np.arange(24) % 4)),   # axes interleaved
])
def test_write(rt, hq, hkv, dim, page, norm, rotary, cache):
    rng = np.random.default_rng(hq * 100 + dim)
    check_write(rt, rng, before=[0, 5, 31, 8], rows=[1, 3, 40, 8], hq=hq, hkv=hkv, dim=dim, page=page, norm=norm,
                rotary=rotary, cache=cache)


@pytest.mark.parametrize("before,rows", [([0], [1]), ([1000], [1]), ([7], [300]), ([3] * 90, [1] * 90),
                                         ([0, 0, 9], [0, 5, 0])])
def test_write_rows(rt, before, rows):
    rng = np.random.default_rng(sum(rows))
    check_write(rt, rng, before=before, rows=rows, norm=1e-6, rotary=R.of_theta(10000.0, 64))


def test_write_leaves_rows_behind_the_last_sequence(rt):
    rng = np.random.default_rng(3)
    check_write(rt, rng, before=[2, 3], rows=[4, 1], norm=1e-6, rotary=R.of_theta(10000.0, 64), extra_rows=9)


@pytest.mark.parametrize("strides", [lambda pages: (2 * 8 * 64, 64, 2 * 64), lambda pages: (64, pages * 8 * 64, pages * 64)])
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_write_strides(rt, strides, cache):
    rng = np.random.default_rng(4)
    check_write(rt, rng, before=[0, 11], rows=[9, 6], strides=strides, cache=cache, norm=1e-6)


def test_write_far_and_negative_positions(rt):
    """Angles of the first pair reach 2^31 radians: exact to fp32 of a turn."""
    rng = np.random.default_rng(5)
    positions = np.array([[0], [1], [-1], [2 ** 31 - 1], [-2 ** 31], [10 ** 6], [123456789]])
    check_write(rt, rng, before=[0], rows=[7], rotary=R.of_theta(10000.0, 64), positions=positions)


def test_write_zero_rows_and_large_values(rt):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((4, 8, 64))
    x[0] = 0.0          # normalized by sqrt(epsilon): zeros
    x[1] *= 1e15        # squares up to 1e30
    x[2] *= 1e-15
    check_write(rt, rng, before=[0], rows=[4], norm=1e-6, rotary=R.of_theta(10000.0, 64), x=x)


def test_write_saturates_e4m3_and_keeps_nan(rt):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 8, 64)) * 1e4
    s, _ = check_write(rt, rng, before=[0], rows=[2], cache="e4m3", x=x,
                       scales=(np.full(2, 0.5, np.float32), np.full(2, 0.25, np.float32)))
    bits = synth.bf16_bits(x.astype(np.float32))
    bits[0, 6, 0], bits[0, 6, 1], bits[0, 6, 2] = 0x7FC0, 0x7F80, 0xFF80   # NaN, inf, -inf in value head 0
    qkv, oq = rt.context.upload(bits), rt.context.allocate(2 * 4 * 64 * 2)
    attention.bind_qk_norm_rope(rt, s.layer, s.step, region(qkv), None, None, region(oq), region(s.k), region(s.v)).launch(rt.stream)
    at = s.at[s.tables[0][0], 0, 0]
    got = s.v.read(np.uint8, s.v_host.shape)[at:at + 3]
    assert got[0] & 0x7F == 0x7F and got[1] == 0x7E and got[2] == 0xFE


def test_write_drops_a_row_whose_page_is_outside_the_cache(rt):
    rng = np.random.default_rng(8)
    s, op = check_write(rt, rng, before=[6, 0], rows=[4, 2])    # row 2 starts page 1 of sequence 0
    k = s.k.read(np.uint16, s.k_host.shape)
    for bad in (s.layer.desc.pages, -1):
        table = np.concatenate(s.tables).astype(np.int32)
        table[1] = bad
        s.step.page_indices.copy_from_host(table)
        s.k.copy_from_host(s.k_host)
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
        now, want = s.k.read(np.uint16, s.k_host.shape), k.copy()
        for slot in range(2):
            for h in range(2):
                at = s.at[s.tables[0][1], h, slot]
                want[at:at + 64] = s.k_host[at:at + 64]
        np.testing.assert_array_equal(now, want)
        op.check()


def test_write_then_decode_on_two_streams(rt):
    """A generation of 40 steps: what the writer appends is what the reader
    reads; two layers of one step run on streams of their own."""
    rng = np.random.default_rng(18)
    hq, hkv, dim, page, n = 4, 2, 64, 8, 3
    rotary = R.of_theta(10000.0, dim)
    streams = [rt.stream, rt.context.create_stream()]
    constants = dict(query_heads=hq, kv_heads=hkv, head_dim=dim, page_size=page, pages=40, max_tokens=n, max_sequences=n,
                     table_entries=30, rotary=rotary, norm_epsilon=1e-6)
    layers = [attention.attention_layer(rt, **constants) for _ in range(2)]
    step = attention.PagedStep(rt, layers[0])
    state = []
    for layer in layers:
        a = {name: rt.context.allocate(nb) for name, nb in (("qkv", n * 8 * dim * 2), ("q", n * hq * dim * 2),
                                                            ("out", n * hq * dim * 2), ("k", layer.cache_bytes), ("v", layer.cache_bytes))}
        a["k"].copy_from_host(np.full(layer.cache_bytes, 0xFF, np.uint8))
        a["v"].copy_from_host(np.full(layer.cache_bytes, 0xFF, np.uint8))
        g = synth.bf16_bits(rng.uniform(0.5, 1.5, dim).astype(np.float32))
        ga = rt.context.upload(g)
        ops = [attention.bind_qk_norm_rope(rt, layer, step, region(a["qkv"]), region(ga), region(ga), region(a["q"]),
                                           region(a["k"]), region(a["v"])),
               attention.bind_paged_decode(rt, layer, step, region(a["q"]), region(a["out"]), region(a["k"]), region(a["v"]))]
        state.append((a, g, ga, ops, [[[] for _ in range(n)] for _ in range(2)]))
    tables = rng.permutation(40)[:30].reshape(n, 10)
    for t in range(40):
        positions = np.array([t, 3 * t, t + 1000])
        step.stage([0, 1, 2, 3], [t + 1] * n, [x[:t // page + 1] for x in tables], positions)
        inputs = []
        for a, g, _, ops, _ in state:
            bits = synth.bf16_bits(rng.standard_normal((n, 8, dim)).astype(np.float32))
            a["qkv"].copy_from_host(bits)
            inputs.append(bits)
        for (a, _, _, ops, _), stream in zip(state, streams):
            for op in ops:
                op.launch(stream, synchronous=False)
        for stream in streams:
            stream.synchronize()
        for (a, g, _, ops, kept), bits in zip(state, inputs):
            for op in ops:
                op.check()
            x, gv = synth.bf16_values(bits).astype(np.float64), synth.bf16_values(g).astype(np.float64)
            q = a["q"].read(np.uint16, (n, hq, dim))
            out = synth.bf16_values(a["out"].read(np.uint16, (n, hq, dim))).astype(np.float64)
            kw, kt = ao.heads(x[:, hq:hq + hkv], gv, 1e-6, positions[:, None], rotary)
            for i in range(n):
                p, slot = tables[i][t // page], t % page
                rows = [c.read(np.uint16, (40, hkv, page, dim))[p, :, slot] for c in (a["k"], a["v"])]
                assert (np.abs(synth.bf16_values(rows[0]) - kw[i]) <= ao.rounded_bf16(kt[i], kw[i])).all()
                np.testing.assert_array_equal(rows[1], bits[i, hq + hkv:])
                for side, r in zip(kept, rows):
                    side[i].append(synth.bf16_values(r).astype(np.float64))
                for h in range(hkv):
                    kk, vv = (np.stack(side[i])[:, h] for side in kept)
                    want, tol = ao.decode(synth.bf16_values(q[i, 2 * h:2 * h + 2]).astype(np.float64), kk, vv, 1 / math.sqrt(dim))
                    assert (np.abs(out[i, 2 * h:2 * h + 2] - want) <= tol).all(), (t, i, h)
