"""Attention of single tokens whose scores are large beside what fp32 resolves, as test_gpu_attention_prompt_large_scores.py
has them for prompts."""
import numpy as np
import pytest

import attention_oracle as ao
import attention_steps as st
from lunaflux_amd import fp8, synth
from test_gpu_attention_prompt_large_scores import same_keys

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cache", ["bf16", "e4m3", "e4m3_blocks"])
@pytest.mark.parametrize("magnitude", [2.0 ** 20, 2.0 ** 29, 2.0 ** 31, 2.0 ** 36, 2.0 ** 44])
def test_equal_scores_average_the_values(rt, dim, magnitude, window, sinks, cache):
    """Keys are alike, so each row's weights are, bit by bit. Bound as for prompts, of twice as many terms."""
    rng = np.random.default_rng(int(np.log2(magnitude)) + dim)
    before = [0, 1, 31, 32, 70, 900]
    s = st.make_step(rt, rng, rows=[1] * 6, before=before, prefill=0, query_heads=16, kv_heads=1, head_dim=dim, page=16,
                     cache=cache, window=window, sinks=sinks)
    same_keys(s)
    q = np.full((6, 16, dim), magnitude / dim, np.float32) * (1 + np.arange(96).reshape(6, 16, 1) / 128).astype(np.float32)
    op, out = st.bind(rt, s, synth.bf16_bits(q), prompts=False)
    op.launch(rt.stream, synchronous=True)
    got = synth.bf16_values(st.read(s, out)).astype(np.float64)
    for i in range(6):
        v = s.values("v", i, 0, st.visible(before[i], window, sinks))
        want, size = v.mean(axis=0), np.abs(v).mean(axis=0)
        tol = 2 * (2 * len(v) + 8) * ao.U32 * size
        tol += (np.abs(want) + tol) * ao.UBF
        assert (np.abs(got[i] - want) <= tol).all(), (i, np.abs(got[i] - want).max(), tol.min())
