"""An attention block as a serving engine runs it, every operator reading what
the one before left on the device: QKV projection, low-rank adapters in place,
per-head norm with rotation and cache append, attention over the paged cache,
output projection, low-rank adapters. Each added operator is held to its own
64-bit bound (attention_oracle.py, test_gpu_low_rank.py) on the inputs that it
read, so the bounds do not add up; the projections, which have tests of their
own, to what their numpy-level calls give."""
import math

import numpy as np
import pytest

import attention_oracle as ao
from lunaflux_amd import attention, fp8, low_rank, synth
from test_gpu_low_rank import arrays, check, expected

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, HIDDEN, PAGE, POOL, N = 8, 2, 64, 512, 16, 24, 5
WIDTHS = [HQ * DIM, HKV * DIM, HKV * DIM]
EPSILON = 1e-6


def region(a):
    return a.region(0, a.byte_count, 256)


def f64(bits):
    return synth.bf16_values(bits).astype(np.float64)


def weight(rt, rng, n):
    return rt.upload_weight(synth.e4m3_encode(rng.standard_normal((n, HIDDEN)).astype(np.float32)),
                            rng.uniform(0.02, 0.06, n).astype(np.float32))


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [0, 9])
def test_prompts_then_decode(cache, window):
    """Prompts of 1 to 40 rows in one step, then three steps of one row each, the
    second of them beside a sequence that is a prompt again; no synchronization
    within a step."""
    rt = fp8.ProjectionRuntime(0)
    rng = np.random.default_rng(77 + window)
    rotary = attention.Rotary.of_theta(10000.0, DIM)
    scales = (rng.uniform(0.02, 0.04, HKV).astype(np.float32),) * 2 if cache == "e4m3" else None
    most = 128
    layer = attention.attention_layer(
        rt, query_heads=HQ, kv_heads=HKV, head_dim=DIM, page_size=PAGE, pages=POOL, cache=cache, max_tokens=most,
        max_sequences=N, table_entries=POOL, rotary=rotary, norm_epsilon=EPSILON, window=window,
        k_scales=scales and scales[0], v_scales=scales and scales[1])
    step = attention.PagedStep(rt, layer)
    wq, wk, wv, wo = (weight(rt, rng, n) for n in (*WIDTHS, HIDDEN))
    _, _, a1, b1, s1 = arrays(rng, 1, HIDDEN, WIDTHS, 32, 4)
    _, _, a2, b2, s2 = arrays(rng, 1, HIDDEN, [HIDDEN], 16, 4)
    first = low_rank.LowRankAdapters.upload(rt, a1, b1, s1, WIDTHS)
    second = low_rank.LowRankAdapters.upload(rt, a2, b2, s2, [HIDDEN])
    g = [synth.bf16_bits(rng.uniform(0.5, 1.5, DIM).astype(np.float32)) for _ in range(2)]
    gq, gk = (rt.context.upload(x) for x in g)
    heads = HQ + 2 * HKV
    size = {"x": HIDDEN, "qkv": heads * DIM, "q": HQ * DIM, "att": HQ * DIM, "o": HIDDEN, "out": HIDDEN}
    at = {name: rt.context.allocate(2 * most * width) for name, width in size.items()}
    ids = rt.context.allocate(4 * most)
    k, v = (rt.context.upload(np.full(layer.cache_bytes, 0xFF, np.uint8)) for _ in range(2))
    r = {name: region(a) for name, a in at.items()}
    ops = [rt.bind_qkv("w8a16", step.counts, r["x"], wq, wk, wv, r["qkv"], most),
           low_rank.bind_low_rank(rt, step.counts, region(ids), r["x"], first, r["qkv"], r["qkv"], most),
           attention.bind_qk_norm_rope(rt, layer, step, r["qkv"], region(gq), region(gk), r["q"], region(k), region(v)),
           attention.bind_paged_decode(rt, layer, step, r["q"], r["att"], region(k), region(v)),
           rt.bind_dense("w8a16", step.counts, r["att"], wo, r["o"], most),
           low_rank.bind_low_rank(rt, step.counts, region(ids), r["att"], second, r["o"], r["out"], most)]

    tables = rng.permutation(POOL)[:4 * N].reshape(N, 4)
    lengths = np.zeros(N, np.int64)
    of_sequence = np.array([2, -1, 0, 2, 3])
    # (new rows of each sequence, how many of the first are prompts)
    for new, prompts in (([1, 40, 16, 3, 17], 5), ([1] * 5, 0), ([7, 1, 1, 1, 1], 1), ([1] * 5, 0)):
        new = np.array(new)
        offsets = np.concatenate([[0], np.cumsum(new)])
        m = int(offsets[-1])
        positions = np.concatenate([np.arange(lengths[i], lengths[i] + new[i]) for i in range(N)])
        before, lengths = lengths, lengths + new
        step.stage(offsets, lengths, [t[:-(-x // PAGE)] for t, x in zip(tables, lengths)], positions, prefill_rows=prompts)
        rows_ids = np.repeat(of_sequence, new).astype(np.int32)
        ids.copy_from_host(rows_ids)
        x = synth.bf16_bits(rng.standard_normal((m, HIDDEN)).astype(np.float32))
        at["x"].copy_from_host(x)
        # rows that attention leaves alone still go through the output projection
        at["att"].copy_from_host(synth.bf16_bits(rng.standard_normal((most, HQ * DIM)).astype(np.float32)))
        for op in ops:
            op.launch(rt.stream, synchronous=False)
        rt.stream.synchronize()
        for op in ops:
            op.check()
        got = {name: a.read(np.uint16, (m, size[name])) for name, a in at.items()}

        y = rt.qkv_projection(x, wq, wk, wv, max_tokens=most)
        check(got["qkv"], y, *expected(x, y, a1, b1, s1, rows_ids, WIDTHS), rows_ids, 4)

        packed = f64(got["qkv"]).reshape(m, heads, DIM)
        want, tol = ao.heads(packed[:, :HQ], f64(g[0]), EPSILON, positions[:, None], rotary)
        assert (np.abs(f64(got["q"]).reshape(m, HQ, DIM) - want) <= ao.rounded_bf16(tol, want)).all()
        shape = (POOL, HKV, PAGE, DIM)
        codes = [c.read(np.uint16 if cache == "bf16" else np.uint8, shape) for c in (k, v)]
        want, tol = ao.heads(packed[:, HQ:HQ + HKV], f64(g[1]), EPSILON, positions[:, None], rotary)
        for side, (w, t) in zip(codes, ((want, tol), (packed[:, HQ + HKV:], 0.0))):
            for i in range(N):
                for j in range(new[i]):
                    slot, row = before[i] + j, offsets[i] + j
                    kept = ao.cache_values(side[tables[i][slot // PAGE], :, slot % PAGE], cache)
                    tt = t if np.isscalar(t) else t[row]
                    if cache == "bf16":
                        assert (np.abs(kept - w[row]) <= ao.rounded_bf16(tt, w[row])).all()
                    else:  # in steps of the scale; 1 / scale and the product round in fp32
                        steps = w[row] / scales[0][:, None].astype(np.float64)
                        ts = tt / scales[0][:, None] + np.abs(steps) * 2 * ao.U32
                        cut = np.clip(steps, -448, 448)
                        assert (np.abs(kept - cut) <= ao.rounded_e4m3(ts, cut)).all()

        attended = f64(got["att"]).reshape(m, HQ, DIM)
        for i in range(prompts, N):
            row, length = offsets[i], lengths[i]
            low = max(0, length - window) if window else 0
            slots = np.arange(low, length)
            for h in range(HKV):
                kk, vv = (ao.cache_values(c[tables[i][slots // PAGE], h, slots % PAGE], cache) *
                          (1.0 if scales is None else np.float64(scales[0][h])) for c in codes)
                group = slice(h * (HQ // HKV), (h + 1) * (HQ // HKV))
                want, tol = ao.decode(f64(got["q"]).reshape(m, HQ, DIM)[row, group], kk, vv, 1 / math.sqrt(DIM))
                assert (np.abs(attended[row, group] - want) <= tol).all(), (i, h)

        o = rt.dense_projection(got["att"], wo, max_tokens=most)
        np.testing.assert_array_equal(got["o"], o)
        check(got["out"], o, *expected(got["att"], o, a2, b2, s2, rows_ids, [HIDDEN]), rows_ids, 4)
