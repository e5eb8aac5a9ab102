"""The softmax weights of decode attention as the second product takes them: two
bf16 terms each. Held to a bound in which a weight is off by 2^-15, which
weights of one bf16 term (2^-8) do not keep."""
import numpy as np
import pytest

import attention_oracle as ao
from lunaflux_amd import fp8, synth
from test_gpu_attention import build, cached, queries, read_out, run_decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def bounded(q, keys, values, scale):
    """(out [G, D] in 64 bits, tolerance) as attention_oracle.decode derives it, with
    another weight: its upper half is cut from the fp32 bits, which leaves less than
    2^-7 of it, exactly, and rounding the rest to bf16 errs by half a step of that,
    2^-8: 2^-15 of the weight, and twice as many terms to add up."""
    z = q @ keys.T * scale
    p = np.exp(z - z.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    out = p @ values
    reach = (np.abs(q) @ np.abs(keys).T).max(axis=1, keepdims=True) * abs(scale)
    spread = np.abs(z - z.max(axis=1, keepdims=True)).max(axis=1, keepdims=True) + np.abs(z).max(axis=1, keepdims=True)
    e = (q.shape[1] + 3) * ao.U32 * reach + (2 + 1.5 * spread) * 2 * ao.U32
    apart = np.stack([(p[r][:, None] * np.abs(values - out[r])).sum(axis=0) for r in range(len(q))])
    tol = 2 * (2.0 ** -15 + 2 * e) * 1.02 * apart + 2 * (2 * len(keys) + 8) * ao.U32 * (p @ np.abs(values))
    return out, tol + (np.abs(out) + tol) * ao.UBF + 1e-38


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,hq,hkv,dim", [
    ([1, 2, 40], 4, 2, 64), ([129, 300], 8, 2, 128), ([90], 17, 1, 256), ([1500, 3], 4, 4, 64),
])
def test_weights_keep_their_second_term(rt, lengths, hq, hkv, dim, cache):
    rng = np.random.default_rng(dim + hq)
    s = build(rt, rng, lengths=lengths, query_heads=hq, kv_heads=hkv, head_dim=dim, page=16, cache=cache)
    q = queries(rng, s)
    out = synth.bf16_values(read_out(s, run_decode(rt, s, q)[1])).astype(np.float64)
    group = hq // hkv
    for i, length in enumerate(lengths):
        for h in range(hkv):
            k = cached(s, s.k_host, i, h, range(length)) * np.float64(s.scales[0][h])
            v = cached(s, s.v_host, i, h, range(length)) * np.float64(s.scales[1][h])
            heads = slice(h * group, (h + 1) * group)
            want, tol = bounded(synth.bf16_values(q[i, heads]).astype(np.float64), k, v, float(s.layer.desc.softmax_scale))
            over = np.abs(out[i, heads] - want) - tol
            assert (over <= 0).all(), (i, h, over.max(), int((over > 0).sum()), over.size)
