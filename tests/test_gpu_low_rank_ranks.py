"""Low-rank adapters of every rank that a profile takes, in each of the forms, with
blocks of both widths, and under profiles far larger than the step."""
import numpy as np
import pytest

from lunaflux_amd import fp8, low_rank
from test_gpu_low_rank import arrays, check, expected

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def run(rt, seed, m, hidden, widths, rank, n, most):
    rng = np.random.default_rng(seed)
    x, y, a, b, scaling = arrays(rng, m, hidden, widths, rank, n)
    ids = rng.integers(-1, n, m).astype(np.int32)
    adapters = low_rank.LowRankAdapters.upload(rt, a, b, scaling, widths)
    got = low_rank.low_rank(rt, x, y, ids, adapters, most)
    check(got, y, *expected(x, y, a, b, scaling, ids, widths), ids, n)


@pytest.mark.parametrize("rank", range(16, 129, 16))
@pytest.mark.parametrize("m,most", [(21, 21), (21, 400), (130, 1000)])
def test_ranks(rt, rank, m, most):
    run(rt, rank, m, 640, [192, 64], rank, 3, most)


@pytest.mark.parametrize("m,most,columns", [(3, 2368, 512), (3, 2369, 1024), (70, 3000, 1024)])
def test_columns_of_a_block(rt, m, most, columns):
    widths = [4096, 1024, 1024]
    assert low_rank.low_rank_descriptor(5, 64, 256, widths, most).block_columns == columns
    run(rt, most, m, 256, widths, 64, 5, most)
