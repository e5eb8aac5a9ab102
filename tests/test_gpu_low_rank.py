"""Low-rank adapters on the GPU against the definition in 64 bits.

A value of x A^T is a sum of K products of bf16 values, exact in fp32, so fp32
sums in any order err by at most (K + 4) 2^-24 sum|x a| (2^-24: half a step). It
enters the second product as two bf16 terms, which leave 2^-16 of it; that
product sums 2 R terms in fp32 and is scaled and added in fp32, then rounded to
bf16 once (2^-8 of the result)."""
import numpy as np
import pytest

from lunaflux_amd import fp8, low_rank, synth
from lunaflux_amd.device import DeviceError

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def values(bits):
    return synth.bf16_values(bits).astype(np.float64)


def arrays(rng, m, hidden, widths, rank, n):
    bf = lambda *shape, scale=1.0: synth.bf16_bits((scale * rng.standard_normal(shape)).astype(np.float32))  # noqa: E731
    return (bf(m, hidden), bf(m, sum(widths)), bf(n, len(widths), rank, hidden, scale=hidden ** -0.5),
            bf(n, sum(widths), rank, scale=0.2), rng.uniform(0.25, 2.0, n).astype(np.float32))


def expected(x, y, a, b, scaling, ids, widths):
    x, y, a, b = values(x), values(y), values(a), values(b)
    want, tol, column = y.copy(), np.zeros_like(y), 0
    k, r = x.shape[1], a.shape[2]
    for i, width in enumerate(widths):
        cols = slice(column, column + width)
        for row, adapter in enumerate(ids):
            if 0 <= adapter < len(a):
                low, size = a[adapter, i] @ x[row], np.abs(a[adapter, i]) @ np.abs(x[row])
                s, bb = np.float64(scaling[adapter]), b[adapter, cols]
                want[row, cols] += s * (bb @ low)
                tol[row, cols] = s * (np.abs(bb) @ ((k + 4) * U * size + (2.0 ** -16 + (2 * r + 4) * U) * np.abs(low)))
        column += width
    return want, tol


def check(got, y, want, tol, ids, n):
    has = (ids >= 0) & (ids < n)
    g = values(got)
    limit = tol + (np.abs(want) + tol) * 2.0 ** -8 + np.abs(values(y)) * 2 * U
    over = np.abs(g - want) - limit
    assert (over[has] <= 0).all(), over[has].max()
    np.testing.assert_array_equal(got[~has], y[~has])


@pytest.mark.parametrize("m,max_tokens", [(1, 1), (1, 16), (15, 16), (17, 64), (128, 128), (61, 61), (129, 129), (64, 256),
                                          (333, 512), (600, 1000)])
@pytest.mark.parametrize("hidden,widths,rank,n", [(128, [64], 16, 1), (512, [512, 128, 128], 16, 5), (1408, [64, 192], 48, 20),
                                                  (2048, [320], 128, 3), (4096, [64, 64, 64, 128], 64, 40)])
def test_low_rank(rt, m, max_tokens, hidden, widths, rank, n):
    rng = np.random.default_rng(m + hidden)
    x, y, a, b, scaling = arrays(rng, m, hidden, widths, rank, n)
    ids = rng.integers(-1, n, m).astype(np.int32)
    adapters = low_rank.LowRankAdapters.upload(rt, a, b, scaling, widths)
    got = low_rank.low_rank(rt, x, y, ids, adapters, max_tokens)
    check(got, y, *expected(x, y, a, b, scaling, ids, widths), ids, n)


@pytest.mark.parametrize("ids", [lambda m: np.full(m, -1), lambda m: np.full(m, 3), lambda m: np.arange(m) // 100,
                                 lambda m: np.arange(m) % 7, lambda m: np.where(np.arange(m) % 2, -1, 6)])
@pytest.mark.parametrize("m", [40, 300, 700])
def test_low_rank_rows_of_adapters(rt, m, ids):
    rng = np.random.default_rng(m)
    x, y, a, b, scaling = arrays(rng, m, 256, [128, 64], 16, 7)
    which = ids(m).astype(np.int32)
    adapters = low_rank.LowRankAdapters.upload(rt, a, b, scaling, [128, 64])
    got = low_rank.low_rank(rt, x, y, which, adapters)
    check(got, y, *expected(x, y, a, b, scaling, which, [128, 64]), which, 7)


@pytest.mark.parametrize("rank", [16, 48, 112])
def test_low_rank_of_a_large_profile(rt, rank):
    """Blocks of up to 1024 columns, the last one of a slice narrower."""
    rng = np.random.default_rng(rank)
    widths, n, m, most = [1600, 64], 3, 150, 384 * 64
    assert low_rank.low_rank_descriptor(n, rank, 128, widths, most).block_columns == 1024
    x, y, a, b, scaling = arrays(rng, m, 128, widths, rank, n)
    ids = rng.integers(-1, n, m).astype(np.int32)
    adapters = low_rank.LowRankAdapters.upload(rt, a, b, scaling, widths)
    check(low_rank.low_rank(rt, x, y, ids, adapters, most), y, *expected(x, y, a, b, scaling, ids, widths), ids, n)


def test_low_rank_of_ranks_below_a_tile(rt):
    rng = np.random.default_rng(1)
    x, y, a, b, scaling = arrays(rng, 9, 256, [64], 5, 2)
    ids = rng.integers(0, 2, 9).astype(np.int32)
    adapters = low_rank.LowRankAdapters.upload(rt, a, b, scaling, [64])
    check(low_rank.low_rank(rt, x, y, ids, adapters), y, *expected(x, y, a, b, scaling, ids, [64]), ids, 2)


@pytest.mark.parametrize("m", [20, 200, 300, 600])
def test_low_rank_rows_do_not_meet_other_adapters(rt, m):
    """Infinities and NaN in one adapter, or in one row, stay with its rows."""
    rng = np.random.default_rng(2)
    widths = [128]
    x, y, a, b, scaling = arrays(rng, m, 256, widths, 16, 4)
    a[1], b[2], x[3] = 0x7FC0, 0x7F80, 0x7F80
    ids = (np.arange(m) % 4).astype(np.int32)
    ids[3] = 0
    got = values(low_rank.low_rank(rt, x, y, ids, low_rank.LowRankAdapters.upload(rt, a, b, scaling, widths)))
    clean = np.isin(ids, (0, 3)) & (np.arange(m) != 3)
    assert np.isfinite(got[clean]).all()
    assert np.isnan(got[ids == 1]).all() and not np.isfinite(got[ids == 2]).any() and not np.isfinite(got[3]).any()


@pytest.mark.parametrize("m,cap", [(3, 16), (70, 256), (0, 16), (130, 300), (0, 300), (333, 700)])
def test_low_rank_out_of_place_and_rows_behind_the_batch(rt, m, cap):
    rng = np.random.default_rng(3)
    widths, n = [192], 2
    x, y, a, b, scaling = arrays(rng, cap, 256, widths, 16, n)
    ids = rng.integers(-1, n, cap).astype(np.int32)
    adapters = low_rank.LowRankAdapters.upload(rt, a, b, scaling, widths)
    up = lambda v: rt.context.upload(v)  # noqa: E731
    xa, ya, ia, oa = up(x), up(y), up(ids), up(np.full((cap, 192), 0x7FA5, np.uint16))
    r = lambda v: v.region(0, v.byte_count, 256)  # noqa: E731
    op = low_rank.bind_low_rank(rt, rt.step_counts(m), r(ia), r(xa), adapters, r(ya), r(oa), cap)
    first = None
    for _ in range(3):
        op.launch(rt.stream, synchronous=True)
        got = oa.read(np.uint16, (cap, 192))
        first = got if first is None else first
        np.testing.assert_array_equal(got, first)
    assert (got[m:] == 0x7FA5).all()
    np.testing.assert_array_equal(ya.read(np.uint16, (cap, 192)), y)
    if m:
        check(got[:m], y[:m], *expected(x[:m], y[:m], a, b, scaling, ids[:m], widths), ids[:m], n)


def test_low_rank_reports_an_adapter_that_does_not_exist(rt):
    rng = np.random.default_rng(4)
    x, y, a, b, scaling = arrays(rng, 5, 256, [64], 16, 2)
    adapters = low_rank.LowRankAdapters.upload(rt, a, b, scaling, [64])
    for bad in (2, 2 ** 31 - 1):
        ids = np.array([0, bad, 1, -2 ** 31, 0], np.int32)
        xa, ya, ia = rt.context.upload(x), rt.context.upload(y), rt.context.upload(ids)
        r = lambda v: v.region(0, v.byte_count, 256)  # noqa: E731
        op = low_rank.bind_low_rank(rt, rt.step_counts(5), r(ia), r(xa), adapters, r(ya), r(ya), 5)
        with pytest.raises(DeviceError):
            op.launch(rt.stream, synchronous=True)
        check(ya.read(np.uint16, y.shape), y, *expected(x, y, a, b, scaling, ids, [64]), ids, 2)
        op.check()
