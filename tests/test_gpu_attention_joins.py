"""Decode attention where pairs of sequence and heads are cut over many blocks:
partial results added up in one and in two levels, beside windows, several head
tiles, missing pages, sequences without keys and NaN. A part is at least 8 tiles
of 32 keys, and more than 32 parts take the second level: sequences of one key
head from 8193 keys on."""
import numpy as np
import pytest

from lunaflux_amd import fp8, synth
from lunaflux_amd.device import DeviceError
from test_gpu_attention import build, check_decode, queries, read_out, run_decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return fp8.ProjectionRuntime(0)


def decoded(rt, s, q, lengths, **checks):
    """Launched four times, which has to give the same bits, and checked."""
    op, oa = run_decode(rt, s, q)
    first = read_out(s, oa)
    check_decode(s, first, q, lengths, **checks)
    for _ in range(3):
        op.launch(rt.stream, synchronous=True)
        np.testing.assert_array_equal(read_out(s, oa), first)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,hq,hkv,dim,page", [
    ([8193], 2, 1, 64, 64),              # 33 parts: a second group of one
    ([10001], 3, 1, 128, 128),
    ([40000], 2, 1, 64, 256),            # 157 parts in five groups
    ([9000, 33, 12000], 2, 2, 64, 64),   # groups of neighbouring pairs side by side
    ([700, 3], 17, 1, 64, 16),           # two head tiles, cut
    ([9500], 40, 1, 64, 128),            # three head tiles, two levels
    ([8500, 1200], 16, 1, 256, 32),      # the largest partial result
])
def test_cut_pairs(rt, lengths, hq, hkv, dim, page, cache):
    rng = np.random.default_rng(lengths[0] + hq)
    s = build(rt, rng, lengths=lengths, query_heads=hq, kv_heads=hkv, head_dim=dim, page=page, cache=cache,
              max_tokens=len(lengths) + 1)
    decoded(rt, s, queries(rng, s), lengths)


@pytest.mark.parametrize("window", [600, 1000, 8300, 9001])
def test_cut_windows(rt, window):
    """19 to 282 tiles from the middle of a page on."""
    rng = np.random.default_rng(window)
    lengths = [12345, 40, 700]
    s = build(rt, rng, lengths=lengths, query_heads=2, kv_heads=1, page=64, window=window)
    decoded(rt, s, queries(rng, s), lengths)


def test_one_long_sequence_among_many(rt):
    """700 short sequences and one of more than 1024 keys: dealt out by tiles, blocks
    hold whole pairs and ends of others."""
    rng = np.random.default_rng(31)
    lengths = [int(x) for x in rng.integers(1, 60, 700)]
    lengths[333] = 1500
    s = build(rt, rng, lengths=lengths, query_heads=4, kv_heads=2, max_sequences=2048, max_tokens=900)
    decoded(rt, s, queries(rng, s), lengths)


def test_sequences_without_keys_among_cut_pairs(rt):
    rng = np.random.default_rng(32)
    lengths = [2000, 50, 9000, 50, 1300]
    s = build(rt, rng, lengths=lengths, query_heads=4, kv_heads=2, page=16)
    live = [2000, 0, 9000, 0, 1300]
    s.step.lengths.copy_from_host(np.array(live, np.int32))
    q = queries(rng, s)
    decoded(rt, s, q, live)


@pytest.mark.parametrize("length", [1000, 9100])
def test_missing_page_of_a_cut_pair(rt, length):
    rng = np.random.default_rng(length)
    lengths, at = [length, 700], 40                        # keys 640 .. 655 of sequence 0
    s = build(rt, rng, lengths=lengths, page=16, query_heads=2, kv_heads=1)
    table = np.concatenate(s.tables).astype(np.int32)
    table[at] = s.layer.desc.pages
    s.step.page_indices.copy_from_host(table)
    q = queries(rng, s)
    op, oa = run_decode(rt, s, q, expect=False)
    with pytest.raises(DeviceError):
        op.launch(rt.stream, synchronous=True)
    check_decode(s, read_out(s, oa), q, lengths,
                 keys_of=lambda i: [j for j in range(lengths[i]) if i or j // 16 != at])
    op.check()


@pytest.mark.parametrize("cache,nan", [("bf16", 0x7FC0), ("e4m3", 0x7F)])
@pytest.mark.parametrize("length", [100, 3000, 9000])
def test_nan_of_a_live_key_or_value(rt, length, cache, nan):
    """It reaches every value (a key) or its column (a value) of the rows that read it, and no other row."""
    rng = np.random.default_rng(33)
    lengths = [length] * 3
    s = build(rt, rng, lengths=lengths, query_heads=2, kv_heads=1, page=32, cache=cache)
    for host, device, i in ((s.k_host, s.k, 0), (s.v_host, s.v, 1)):
        j = 2 * length // 3
        host[s.at[s.tables[i][j // 32], 0, j % 32] + 3] = nan
        device.copy_from_host(host)
    out = synth.bf16_values(read_out(s, run_decode(rt, s, queries(rng, s))[1]))
    assert np.isnan(out[0]).all()
    assert np.isnan(out[1, :, 3]).all() and np.isfinite(np.delete(out[1], 3, axis=1)).all()
    assert np.isfinite(out[2]).all()


@pytest.mark.parametrize("amplitude", [1.5, 40.0])
def test_infinite_values_keep_their_sign(rt, amplitude):
    """An infinite value at a key whose weight fp32 holds is that infinity in the
    output, weights that are bf16 values (one key; equal scores) among them."""
    rng = np.random.default_rng(34)
    lengths = [1, 2, 33, 2000]
    s = build(rt, rng, lengths=lengths, query_heads=2, kv_heads=1, page=32)
    for i, length in enumerate(lengths):
        for column, bits in ((3, 0x7F80), (9, 0xFF80)):
            s.v_host[s.at[s.tables[i][0], 0, 0] + column] = bits
        a = s.at[s.tables[i][0], 0, 0]
        if amplitude > 2:
            # key 0 has the largest score of all: its weight is one
            for j in range(1, length):
                b = s.at[s.tables[i][j // 32], 0, j % 32]
                s.k_host[b:b + 64] = 0
            s.k_host[a:a + 64] = synth.bf16_bits(np.ones(64, np.float32))
    s.v.copy_from_host(s.v_host)
    s.k.copy_from_host(s.k_host)
    q = queries(rng, s)
    if amplitude > 2:
        q = synth.bf16_bits(np.full((4, 2, 64), 4.0, np.float32))
    out = synth.bf16_values(read_out(s, run_decode(rt, s, q)[1]))
    assert (out[..., 3] == np.inf).all() and (out[..., 9] == -np.inf).all()
    assert np.isfinite(np.delete(out, (3, 9), axis=2)).all()
