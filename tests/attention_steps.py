"""Steps over a paged cache of any type, with what every place of it holds, for
tests of the attention operators against attention_oracle.py. Cache places that
no row of the step counts hold NaN, page-table entries that none needs -1."""
from dataclasses import dataclass, field

import numpy as np

import attention_oracle as ao
from lunaflux_amd import attention, synth

SENTINEL = 0x7FA5  # a bf16 NaN


def region(a):
    return a.region(0, a.byte_count, 256)


def visible(position, window, sinks):
    """Keys that a row at `position` counts."""
    lo = max(0, position + 1 - window) if window else 0
    return [*range(min(sinks, lo)), *range(lo, position + 1)]


@dataclass
class Step:
    layer: attention.AttentionLayer
    step: attention.PagedStep
    kind: str
    rows: list
    before: list
    row_offsets: np.ndarray
    tables: list = field(default_factory=list)     # with the entries that no row needs
    scales: tuple = ()                             # per head, of an e4m3 cache
    host: dict = field(default_factory=dict)       # cache bytes as uploaded
    device: dict = field(default_factory=dict)

    @property
    def desc(self):
        return self.layer.desc

    def element(self, page, head, slot):
        d = self.desc
        return page * d.page_stride + head * d.head_stride + slot * d.token_stride

    def codes(self, host):
        """A cache's elements, and its table of scales by blocks (views), of its bytes."""
        d = self.desc
        if self.kind == "bf16":
            return host.view(np.uint16), None
        if self.kind == "e4m3":
            return host, None
        table = host[d.block_scales:].view(np.float32).reshape(self.layer.block_scales_shape)
        return host[:d.block_scales], table

    def place(self, sequence, token):
        page = self.desc.page_size
        return self.tables[sequence][token // page], token % page

    def values(self, side, sequence, head, tokens, host=None):
        """fp64 values of cached tokens of a key head."""
        d = self.desc
        codes, table = self.codes(self.host[side] if host is None else host)
        out = np.zeros((len(tokens), d.head_dim))
        for n, j in enumerate(tokens):
            page, slot = self.place(sequence, j)
            at = self.element(page, head, slot)
            row = ao.cache_values(codes[at:at + d.head_dim], "bf16" if self.kind == "bf16" else "e4m3")
            step = 1.0 if self.kind == "bf16" else self.scales[side == "v"][head] if table is None else \
                table[page, slot // d.block_tokens, head]
            out[n] = row * np.float64(step)
        return out


def make_step(rt, rng, *, rows, before, prefill=None, query_heads=4, kv_heads=2, head_dim=64, page=8, cache="bf16",
              strides=None, window=0, sinks=0, max_tokens=None, max_sequences=None, spare_entries=0, amplitude=1.0,
              fill=True, spare_pages=2, positions=None, **constants):
    """rows, before: of each sequence; prefill: sequences that are prompts (default: all). fill False: an
    empty cache of NaN, as before any append."""
    n = len(rows)
    lengths = [r + b for r, b in zip(rows, before)]
    counts = [-(-x // page) + spare_entries for x in lengths]
    pool = sum(counts) + spare_pages
    order = rng.permutation(pool)[:sum(counts)]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    tables = [order[starts[i]:starts[i + 1]].astype(np.int32) for i in range(n)]
    scales = None
    if cache == "e4m3":
        scales = tuple(rng.uniform(0.01, 0.05, kv_heads).astype(np.float32) for _ in range(2))
    offsets = np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)
    layer = attention.attention_layer(
        rt, query_heads=query_heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page, pages=pool, cache=cache,
        max_tokens=max_tokens or max(1, int(offsets[-1])), max_sequences=max_sequences or max(1, n),
        table_entries=max(1, sum(counts)), strides=strides(pool) if callable(strides) else strides, window=window,
        sinks=sinks, k_scales=None if scales is None else scales[0], v_scales=None if scales is None else scales[1],
        **constants)
    s = Step(layer, attention.PagedStep(rt, layer), cache, list(rows), list(before), offsets, tables, scales or ())
    d = layer.desc
    needed = []
    for i in range(n):
        keys = set()
        for r in range(rows[i]):
            keys.update(visible(before[i] + r, window, sinks))
        needed.append(sorted(keys))
    for side in ("k", "v"):
        host = np.full(layer.cache_bytes, 0x7F, np.uint8)
        codes, table = s.codes(host)
        if cache == "bf16":
            codes[:] = SENTINEL
        if table is not None:
            table[:] = np.nan
        for i in range(n if fill else 0):
            for j in needed[i]:
                p, slot = s.place(i, j)
                values = amplitude * rng.standard_normal((kv_heads, head_dim)).astype(np.float32)
                if table is not None and np.isnan(table[p, slot // d.block_tokens]).any():
                    table[p, slot // d.block_tokens] = 2.0 ** rng.integers(-8, -4, kv_heads)
                for h in range(kv_heads):
                    at = s.element(p, h, slot)
                    codes[at:at + head_dim] = synth.bf16_bits(values[h]) if cache == "bf16" else synth.e4m3_encode(values[h] * 30)
        s.host[side] = host
        s.device[side] = rt.context.upload(host)
    staged = [t.copy() for t in tables]
    for i, t in enumerate(staged):
        pages = {j // page for j in needed[i]} | {j // page for j in range(before[i], lengths[i])}
        for e in range(len(t)):
            if e not in pages:
                t[e] = -1
    s.step.stage(offsets, lengths, staged, positions, prefill_rows=n if prefill is None else prefill)
    return s


def queries(rng, s, amplitude=1.5):
    d = s.desc
    return synth.bf16_bits((amplitude * rng.standard_normal((d.max_tokens, d.query_heads, d.head_dim))).astype(np.float32))


def bind(rt, s, q, prompts=True):
    """(operation, allocation of out, filled with a sentinel)."""
    qa = rt.context.upload(q)
    out = rt.context.upload(np.full(q.size, SENTINEL, np.uint16))
    f = attention.bind_paged_prefill if prompts else attention.bind_paged_decode
    return f(rt, s.layer, s.step, region(qa), region(out), region(s.device["k"]), region(s.device["v"])), out


def read(s, out):
    d = s.desc
    return out.read(np.uint16, (d.max_tokens, d.query_heads, d.head_dim))


def check(s, got_bits, q, sequences, hidden=lambda i, j: False):
    """Every row of `sequences` against the oracle; other rows are the sentinel. hidden: keys that do not count."""
    d = s.desc
    group, written = d.query_heads // d.kv_heads, np.zeros(d.max_tokens, bool)
    for i in sequences:
        for h in range(d.kv_heads):
            tokens = sorted({j for r in range(s.rows[i]) for j in visible(s.before[i] + r, d.window, d.sinks)})
            at = {j: n for n, j in enumerate(tokens)}
            k, v = (s.values(side, i, h, tokens) for side in ("k", "v"))
            for r in range(s.rows[i]):
                row = int(s.row_offsets[i]) + r
                written[row] = True
                keys = [at[j] for j in visible(s.before[i] + r, d.window, d.sinks) if not hidden(i, j)]
                heads = slice(h * group, (h + 1) * group)
                want, tol = ao.decode(synth.bf16_values(q[row, heads]).astype(np.float64), k[keys], v[keys], float(d.softmax_scale))
                got = synth.bf16_values(got_bits[row, heads]).astype(np.float64)
                assert np.isfinite(got).all(), (i, h, r)
                over = np.abs(got - want) - tol
                assert (over <= 0).all(), (i, h, r, over.max(), np.abs(got - want).max())
    assert (got_bits[~written] == SENTINEL).all()
