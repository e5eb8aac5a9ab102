"""Infinite values at keys that a prompt's rows count, of weights that fp32 does not hold: the same result wherever the
keys with the large scores are, and wherever the work is cut."""
import numpy as np
import pytest

import attention_oracle as ao
import attention_steps as st
from lunaflux_amd import fp8, synth

pytestmark = pytest.mark.gpu
INF, MINUS_INF, NAN = 0x7F80, 0xFF80, 0x7FC0


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def put(s, side, token, columns, bits):
    page, slot = s.place(0, token)
    s.codes(s.host[side])[0][s.element(page, 0, slot) + np.asarray(columns)] = bits


# before: none cut; cut between blocks. odd: the token with the odd values; large: the one whose score is the largest
@pytest.mark.parametrize("before,odd,large", [(0, 1, 30), (0, 30, 1), (0, 1, 2), (5000, 100, 4900), (5000, 4900, 100), (5000, 2000, 2001)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_an_infinite_value_of_a_weight_that_vanishes(rt, dim, before, odd, large):
    """Weights of at most 2^-369 (4096 / sqrt(256) log2 e) to all keys but one. A counted infinity is that infinity all the same, of both signs NaN; a
    value near the largest of bf16 times such a weight is nothing."""
    rng = np.random.default_rng(before + odd + dim)
    rows = 40
    s = st.make_step(rt, rng, rows=[rows], before=[before], query_heads=2, kv_heads=1, head_dim=dim, page=16)
    for token in range(before + rows):
        put(s, "k", token, range(dim), 0)
    put(s, "k", large, range(dim), synth.bf16_bits(np.float32(8.0)))
    put(s, "v", odd, 3, INF)
    put(s, "v", odd, 5, MINUS_INF)
    put(s, "v", odd, 7, NAN)
    put(s, "v", odd, 9, synth.bf16_bits(np.float32(3e38)))
    put(s, "v", odd, 11, INF)
    put(s, "v", large, 11, MINUS_INF)
    for side in ("k", "v"):
        s.device[side].copy_from_host(s.host[side])
    q = np.full((rows, 2, dim), synth.bf16_bits(np.float32(512 / dim)), np.uint16)  # scores of 2^12 / sqrt(dim)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    got = synth.bf16_values(st.read(s, out))
    hit = slice(max(0, max(odd, large) - before), rows)  # rows that count both
    assert (got[hit, :, 3] == np.inf).all() and (got[hit, :, 5] == -np.inf).all()
    assert np.isnan(got[hit, :, 7]).all() and np.isnan(got[hit, :, 11]).all()
    value = s.values("v", 0, 0, [large])[0]
    rest = [c for c in range(dim) if c not in (3, 5, 7, 11)]
    # the others' weights add up to less than 2^-190, of 3e38 less than 2^-62
    tol = np.abs(value[rest]) * (ao.UBF + 8 * (before + rows) * ao.U32) + 2.0 ** -60
    assert (np.abs(got[hit][:, :, rest] - value[rest]) <= tol).all()
