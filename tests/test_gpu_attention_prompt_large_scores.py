"""Attention of prompts whose scores are large beside what fp32 resolves: a maximum rounded to fp32 is then off by
more than an exponential bears."""
import numpy as np
import pytest

import attention_oracle as ao
import attention_steps as st
from lunaflux_amd import fp8, synth

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def same_keys(s):
    """All keys of the cache the same values: ones, in steps of 2^-6 or of a head's scale over codes."""
    codes, table = s.codes(s.host["k"])
    for i in range(len(s.rows)):
        for j in range(s.before[i] + s.rows[i]):
            page, slot = s.place(i, j)
            if table is not None:
                table[page, slot // s.desc.block_tokens] = 2.0 ** -6
            for h in range(s.desc.kv_heads):
                at = s.element(page, h, slot)
                codes[at:at + s.desc.head_dim] = synth.bf16_bits(np.float32(1.0)) if s.kind == "bf16" else 0x38
    s.device["k"].copy_from_host(s.host["k"])


# rows from a first token on (one key), and ones cut between blocks
@pytest.mark.parametrize("rows,before,dim", [([70], [0], 64), ([70], [0], 128), ([40], [100], 256), ([9], [3000], 64)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("cache", ["bf16", "e4m3", "e4m3_blocks"])
@pytest.mark.parametrize("magnitude", [2.0 ** 20, 2.0 ** 29, 2.0 ** 31, 2.0 ** 36, 2.0 ** 44])
def test_equal_scores_average_the_values(rt, rows, before, dim, sign, magnitude, cache):
    """Keys are alike, so each row's weights are, bit by bit, whatever its score; rows differ in theirs. Bound: sums of
    n fp32 terms, numerator and denominator (their weights are the same bf16 values), the quotient, the rounding to bf16."""
    rng = np.random.default_rng(int(np.log2(magnitude)) + dim)
    s = st.make_step(rt, rng, rows=rows, before=before, query_heads=2, kv_heads=1, head_dim=dim, page=16, cache=cache)
    same_keys(s)
    q = np.full((s.desc.max_tokens, 2, dim), sign * magnitude / dim, np.float32)
    q *= (1 + np.arange(2 * s.desc.max_tokens).reshape(-1, 2, 1) % 97 / 128).astype(np.float32)
    q = synth.bf16_bits(q)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    got = synth.bf16_values(st.read(s, out)).astype(np.float64)
    values = s.values("v", 0, 0, range(before[0] + rows[0]))
    for r in range(rows[0]):
        v = values[:before[0] + r + 1]
        want, size = v.mean(axis=0), np.abs(v).mean(axis=0)
        tol = 2 * (len(v) + 8) * ao.U32 * size
        tol += (np.abs(want) + tol) * ao.UBF
        assert (np.abs(got[r] - want) <= tol).all(), (r, np.abs(got[r] - want).max(), tol.min())
