"""Attention of prompts where every cache place holds a finite number, so that the matrix kernel's results are the ones
that are read: its masks under windows with sinks in every kind of tile, and steps of thousands of rows, whose pairs are
cut at every eighth tile and of which a block has several. (A NaN where no key counts, as attention_steps.py fills
those places by default, makes a row of the path for odd values of every row whose tiles hold it.)"""
import numpy as np
import pytest

import attention_oracle as ao
import attention_steps as st
from lunaflux_amd import attention, fp8, synth

pytestmark = pytest.mark.gpu
CACHES = ["bf16", "e4m3", "e4m3_blocks"]


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def fill_hidden(s):
    """Keys of zeros, whose scores are as good as any, and large values where no row of the step counts a key."""
    for side in ("k", "v"):
        codes, table = s.codes(s.host[side])
        if s.kind == "bf16":
            codes[codes == st.SENTINEL] = synth.bf16_bits(np.float32(0.0 if side == "k" else 1000.0))
        else:
            codes[codes == 0x7F] = 0x00 if side == "k" else 0x7E   # 448 steps
        if table is not None:
            table[np.isnan(table)] = 4.0
        s.device[side].copy_from_host(s.host[side])


def run(rt, rng, **fields):
    s = st.make_step(rt, rng, **fields)
    fill_hidden(s)
    q = st.queries(rng, s)
    op, out = st.bind(rt, s, q)
    op.launch(rt.stream, synchronous=True)
    first = st.read(s, out)
    st.check(s, first, q, range(len(s.rows)))
    op.launch(rt.stream, synchronous=True)
    np.testing.assert_array_equal(st.read(s, out), first)


WINDOWS = [(1, 0), (1, 1), (16, 4), (63, 64), (64, 1), (100, 37), (128, 130), (300, 2000), (5000, 9), (0, 5)]


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_windows_and_sinks(rt, window, sinks, cache):
    rng = np.random.default_rng(window + sinks)
    run(rt, rng, rows=[150, 1, 40], before=[300, 700, 0], query_heads=4, kv_heads=1, page=16, cache=cache, window=window, sinks=sinks)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("window,sinks", [(16, 4), (100, 37), (128, 130)])
def test_windows_and_sinks_of_larger_heads(rt, window, sinks, dim, cache):
    rng = np.random.default_rng(window + sinks + dim)
    run(rt, rng, rows=[150, 1, 40], before=[300, 700, 0], query_heads=4, kv_heads=1, head_dim=dim, page=16, cache=cache,
        window=window, sinks=sinks)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_long_window_with_sinks_is_cut(rt, dim, cache):
    rng = np.random.default_rng(5 + dim)
    run(rt, rng, rows=[40], before=[4000], query_heads=2, kv_heads=1, head_dim=dim, page=8, cache=cache, window=2500, sinks=700)


# ---- large steps -----------------------------------------------------------------------

def ranges_of(rows, before, group, kv_heads, tile_keys, window, sinks):
    """(weight of a block's range, most key tiles of a query tile, query tiles of several key tiles) of a step, as
    attention_index.h has them."""
    tokens, total, most, several = 256 // group, 0, 0, 0
    for r, b in zip(rows, before):
        for x in range(-(-r // tokens)):
            weight = b + tokens + 256 + tokens * x
            total += kv_heads * (min(weight, window + sinks + tokens + 256) if window else weight)
            last = b + min(r, tokens * (x + 1)) - 1
            lo = max(0, b + tokens * x + 1 - window) if window else 0
            sink_tiles = min(-(-min(sinks, lo) // tile_keys), lo // tile_keys)
            tiles = sink_tiles + last // tile_keys + 1 - lo // tile_keys
            most = max(most, tiles)
            several += kv_heads * (tiles > 1)
    return -(-total // 256), most, several


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("rows,before,hq,hkv,dim,window,sinks", [
    ([2100, 900, 333], [100, 3000, 0], 32, 8, 64, 0, 0),
    ([700] * 8, [0, 100, 200, 300, 400, 500, 600, 700], 16, 16, 128, 0, 0),
    ([2301, 700], [300, 1000], 28, 4, 128, 1021, 4),
    ([1000, 411], [700, 2000], 16, 4, 256, 0, 0),
    ([1300, 600], [0, 900], 16, 16, 256, 600, 70),
])
def test_large_steps(rt, rows, before, hq, hkv, dim, window, sinks, cache):
    """Blocks' ranges of at least 512 of weight, which cut pairs at every eighth tile, and, of heads of 64 and 128, more
    pairs of several tiles than blocks. The bound is attention_oracle.decode's, with sum p |v - out| <= sum p |v| + |out|."""
    import torch
    rng = np.random.default_rng(sum(rows) + dim)
    n, page, group, m = len(rows), 16, hq // hkv, sum(rows)
    share, most, several = ranges_of(rows, before, group, hkv, 32 if dim == 256 else 64, window, sinks)
    assert share >= 512 and most >= 16 and (dim == 256 or several > 256)
    lengths = np.array(rows) + before
    counts = -(-lengths // page)
    pool = int(counts.sum()) + 3
    starts = np.concatenate([[0], np.cumsum(counts)])
    tables = np.split(rng.permutation(pool)[:starts[-1]].astype(np.int32), starts[1:-1])
    scales = tuple(rng.uniform(0.01, 0.05, hkv).astype(np.float32) for _ in range(2)) if cache == "e4m3" else (None, None)
    layer = attention.attention_layer(rt, query_heads=hq, kv_heads=hkv, head_dim=dim, page_size=page, pages=pool, max_tokens=m,
                                      max_sequences=n, table_entries=int(starts[-1]), cache=cache, k_scales=scales[0],
                                      v_scales=scales[1], window=window, sinks=sinks)
    step = attention.PagedStep(rt, layer)
    offsets = np.concatenate([[0], np.cumsum(rows)])
    step.stage(offsets, lengths, tables, prefill_rows=n)
    values, device = [], []
    for side in range(2):
        x = rng.standard_normal((pool, hkv, page, dim), dtype=np.float32)
        host = np.zeros(layer.cache_bytes, np.uint8)
        if cache == "bf16":
            codes = synth.bf16_bits(x)
            x = synth.bf16_values(codes)
            host[:codes.nbytes] = codes.view(np.uint8).reshape(-1)
        else:
            codes = torch.from_numpy(x * 30).to(torch.float8_e4m3fn)
            host[:x.size] = codes.view(torch.uint8).numpy().reshape(-1)
            x = codes.float().numpy()
            if cache == "e4m3":
                x = x * scales[side][None, :, None, None]
            else:
                table = 2.0 ** rng.integers(-8, -4, (pool, 1, hkv))
                host[layer.block_scales_offset:].view(np.float32)[:] = table.reshape(-1)
                x = x * table.reshape(pool, hkv, 1, 1)
        values.append(x.astype(np.float64))
        device.append(rt.context.upload(host))
    q = synth.bf16_bits(1.5 * rng.standard_normal((m, hq, dim), dtype=np.float32))
    qa, out = rt.context.upload(q), rt.context.upload(np.full(q.size, st.SENTINEL, np.uint16))
    op = attention.bind_paged_prefill(rt, layer, step, st.region(qa), st.region(out), *map(st.region, device))
    op.launch(rt.stream, synchronous=True)
    first = out.read(np.uint16, (m, hq, dim))
    got, scale = torch.from_numpy(synth.bf16_values(first).astype(np.float64)), float(layer.desc.softmax_scale)
    for i in range(n):
        position = torch.arange(before[i], int(lengths[i])).repeat_interleave(group)[:, None]
        j = torch.arange(int(lengths[i]))
        hidden = (j > position) | ((j <= position - window) & (j >= sinks) if window else j < 0)
        for h in range(0, hkv, 3):
            k, v = (torch.from_numpy(x[tables[i], h].reshape(-1, dim)[:int(lengths[i])].copy()) for x in values)
            heads = slice(h * group, (h + 1) * group)
            qh = torch.from_numpy(synth.bf16_values(q[offsets[i]:offsets[i + 1], heads]).astype(np.float64)).reshape(-1, dim)
            z = (qh @ k.t()) * scale
            z[hidden] = -np.inf
            top = z.amax(dim=1, keepdim=True)
            reach = (qh.abs() @ k.abs().t()).amax(dim=1, keepdim=True) * scale
            size = z.masked_fill(hidden, 0.0).abs().amax(dim=1, keepdim=True)
            p = torch.exp(z - top)
            p /= p.sum(dim=1, keepdim=True)
            want, reached = p @ v, p @ v.abs()
            e = (dim + 3) * ao.U32 * reach + (2 + 1.5 * 3 * size) * 2 * ao.U32
            tol = 2 * (ao.UBF + 2 * e) * 1.02 * (reached + want.abs()) + 2 * (len(k) + 8) * ao.U32 * reached
            tol = tol + (want.abs() + tol) * ao.UBF
            over = (got[offsets[i]:offsets[i + 1], heads].reshape(-1, dim) - want).abs() - tol
            assert bool((over <= 0).all()), (i, h, float(over.max()))
    op.launch(rt.stream, synchronous=True)
    np.testing.assert_array_equal(out.read(np.uint16, (m, hq, dim)), first)
