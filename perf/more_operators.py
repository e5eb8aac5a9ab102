"""Attention of prompts, windows with sinks and caches scaled by blocks, as cases to be timed.

  prompt  attention of the rows of whole prompts, or of parts of them, over the
          paged cache (attention.bind_paged_prefill)
  decode  attention of one new token per sequence: a window with the first
          tokens still visible, or a cache of e4m3 codes with a scale for each
          block of 16 tokens and head (attention.bind_paged_decode)
  write   per-head norm, rotary positions and append to a cache with scales by
          blocks, which are found, or raised, as the rows arrive
          (attention.bind_qk_norm_rope)

Heads and widths are Llama-3-8B's (32 query and 8 key / value heads of 128), a
small model's (8 heads of 64) or generic ones. `run` computes them in elementary
torch operations, or, where `own` is true, with the framework's kernels.
"""
import ctypes
import math

import numpy as np
import torch

own = False

EPSILON = 1e-6
THETA = 500000.0
KEY_SCALE, VALUE_SCALE = 0.03, 0.02  # steps of an e4m3 cache with a scale per head (times 1 + head / 16)
BLOCK = 16                           # tokens of a block with its own scale (a whole page, where pages are shorter)
LEAST, MOST = -100, 119              # exponents of the blocks' scales


def listed():
    return [
        # A small model, a few short prompts at once: launch latency.
        _prompt("prompt_small", 3, 37, 0.6, 0, 8, 8, 64, "bf16", 16),
        # An ordinary batch of prompts of a grouped-query model.
        _prompt("prompt_b4", 4, 2039, 0.3, 0, 32, 8, 128, "bf16", 16),
        # One long prompt.
        _prompt("prompt_long", 1, 8192, 0.0, 0, 32, 8, 128, "bf16", 64),
        # The last part of a very long prompt, or drafted tokens checked at its end.
        _prompt("prompt_chunk", 1, 61, 0.0, 131010, 32, 8, 128, "bf16", 64),
        # Long prompts under a window, the first tokens visible, over a cache scaled by blocks.
        _prompt("prompt_window", 3, 2731, 0.7, 300, 28, 4, 128, "e4m3_blocks", 32, 1021, 4),
        # Large heads, parts of prompts behind what an e4m3 cache already holds.
        _prompt("prompt_d256", 5, 509, 0.4, 2500, 16, 8, 256, "e4m3", 16),
        # A few conversations of a small model under a window.
        _decode("decode_sinks_small", 3, 301, 0.6, 8, 8, 64, "bf16", 16, 64, 4),
        # Long conversations under a window: what lies between is not read.
        _decode("decode_sinks_b64", 64, 9973, 0.8, 32, 8, 128, "bf16", 16, 2039, 4),
        # A large ragged batch over a cache scaled by blocks.
        _decode("decode_blocks_b96", 96, 5003, 0.9, 32, 8, 128, "e4m3_blocks", 32),
        # A few users with very long contexts, few key heads.
        _decode("decode_blocks_long", 3, 65521, 0.4, 16, 2, 128, "e4m3_blocks", 64),
        # A decode step's new rows: most fall into blocks that already hold tokens.
        _write("write_blocks_m32", 32, 32, 32, 8, 128, 128, "half", True, 1, 16),
        # Prompts' rows: whole blocks at once.
        _write("write_blocks_m8191", 8191, 5, 32, 8, 128, 128, "half", True, 1, 32),
    ]


def _prompt(name, sequences, rows, spread, before, query_heads, kv_heads, head_dim, cache, page, window=0, sinks=0):
    """rows: of the longest sequence of the step, down to (1 - spread) of them; before: tokens cached before them."""
    return dict(name=name, kind="prompt", sequences=sequences, rows=rows, spread=spread, before=before,
                query_heads=query_heads, kv_heads=kv_heads, head_dim=head_dim, cache=cache, page=page, window=window, sinks=sinks)


def _decode(name, sequences, longest, spread, query_heads, kv_heads, head_dim, cache, page, window=0, sinks=0):
    return dict(name=name, kind="decode", sequences=sequences, longest=longest, spread=spread, query_heads=query_heads,
                kv_heads=kv_heads, head_dim=head_dim, cache=cache, page=page, window=window, sinks=sinks)


def _write(name, rows, sequences, query_heads, kv_heads, head_dim, rotary, pairing, norm, axes, page):
    return dict(name=name, kind="write", rows=rows, sequences=sequences, query_heads=query_heads, kv_heads=kv_heads,
                head_dim=head_dim, rotary=rotary, pairing=pairing, norm=norm, axes=axes, cache="e4m3_blocks", page=page)


HEADS = [(8, 8, 64), (32, 8, 128), (32, 8, 128), (28, 4, 128), (16, 2, 128), (16, 8, 256), (12, 12, 64), (32, 1, 128), (5, 1, 64)]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5))))


def draw(rng):
    taken = [{k: v for k, v in c.items() if k != "name"} for c in listed()]
    while True:
        case = _draw(rng)
        case.pop("name")
        if case not in taken:
            return case


def _draw(rng):
    kind = rng.choice(["prompt", "prompt", "decode", "write"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([8, 16, 32, 64, 128])
    if kind == "prompt":
        sequences = _log_uniform(rng, 1, 12)
        # padded scores of the plain form, and products of the operator, at most those of the longest prompt listed
        rows = _log_uniform(rng, 1, int(8192 * min(1.0, (32 * 128 / (hq * d * sequences)) ** 0.5)))
        most = 32 * 8192 * 4096 * 128 // (hq * d * rows * sequences) - rows
        before = 0 if rng.random() < 0.4 or most < 8 else _log_uniform(rng, 4, min(most, 131072 // sequences))
        window = rng.choice([0, 0, _log_uniform(rng, 1, rows + before)])
        return _prompt("", sequences, rows, round(rng.uniform(0, 0.9), 2), before, hq, hkv, d,
                       rng.choice(["bf16", "bf16", "e4m3", "e4m3_blocks"]), page, window,
                       rng.choice([0, 1, 4, 37]) if window else 0)
    if kind == "decode":
        sequences = _log_uniform(rng, 1, 128)
        blocks = rng.random() < 0.6
        most = 500_000_000 // (sequences * hkv * d * (2 if blocks else 4))
        longest = _log_uniform(rng, 8, max(8, min(131072, most)))
        window = rng.choice([0, 0, _log_uniform(rng, 1, longest)]) if blocks else _log_uniform(rng, 1, longest)
        return _decode("", sequences, longest, round(rng.uniform(0, 0.95), 2), hq, hkv, d,
                       "e4m3_blocks" if blocks else rng.choice(["bf16", "e4m3"]), page, window,
                       rng.choice([1, 4, 37, 130]) if window else 0)
    rows = _log_uniform(rng, 1, 8192 * 6144 // ((hq + 2 * hkv) * d) if d > 64 else 8192)
    return _write("", rows, rng.randint(1, min(rows, 64)), hq, hkv, d, rng.choice([d, d, d // 2]),
                  rng.choice(["half", "half", "neighbour"]), rng.random() < 0.5, rng.choice([1, 1, 3]), page)


# -- inputs, from the seed -----------------------------------------------------

def _spread(n, longest, spread):
    """n lengths, the longest down to (1 - spread) of it."""
    return np.maximum(1, np.round(longest * (1 - spread * ((np.arange(n) * 0.6180339887) % 1.0)))).astype(np.int64)


def _rows_and_before(case):
    """Rows of each sequence of the step, and the tokens cached before them."""
    n = case["sequences"]
    if case["kind"] == "decode":
        return np.ones(n, np.int64), _spread(n, case["longest"], case["spread"]) - 1
    if case["kind"] == "prompt":
        return _spread(n, case["rows"], case["spread"]), case["before"] - (np.arange(n) * 37 % (case["before"] // 4 + 1))
    rows = case["rows"]
    cuts = np.concatenate([[0], np.sort((np.arange(1, n) * rows) // n + (np.arange(1, n) % 3 - 1) * (rows // n > 2)), [rows]])
    return np.diff(cuts), (np.arange(n) * 37 + 5) % 200


class _Draws:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.host = np.random.default_rng(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")


def _block(case):
    return min(BLOCK, case["page"])


def _cache(d, case, pages):
    """One side of a paged cache [pages, kv heads, page, head dim], N(0, 1) values or e4m3 codes, and its steps:
    one per head, or a power of two per block [pages, page / block, kv heads]."""
    hkv, page = case["kv_heads"], case["page"]
    x = torch.empty((pages, hkv, page, case["head_dim"]), dtype=torch.bfloat16, device="cuda").normal_(generator=d.g)
    if case["cache"] == "bf16":
        return x, torch.ones(hkv, device="cuda")
    if case["cache"] == "e4m3":
        return (x * 30.0).to(torch.float8_e4m3fn), 1.0 + torch.arange(hkv, device="cuda") / 16.0
    shape = (pages, page // _block(case), hkv)
    return (x * 60.0).to(torch.float8_e4m3fn), torch.exp2(torch.randint(-8, -4, shape, generator=d.g, device="cuda").float())


def _tables(d, lengths, page):
    """Page table of each sequence (pages of a shuffled pool), its offsets, and the pool's size."""
    counts = -(-lengths // page)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    pool = int(offsets[-1]) + 3
    return d.host.permutation(pool)[:offsets[-1]].astype(np.int32), offsets.astype(np.int32), pool


def _inputs(case, seed):
    d = _Draws(seed)
    hq, hkv, dim = case["query_heads"], case["kv_heads"], case["head_dim"]
    t = {}
    rows, before = _rows_and_before(case)
    order = d.host.permutation(case["sequences"])
    rows, before = rows[order], before[order]
    m, lengths = int(rows.sum()), rows + before
    t["row_offsets"] = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    t["lengths"] = lengths.astype(np.int32)
    t["slot"] = np.concatenate([before[s] + np.arange(rows[s]) for s in range(case["sequences"])])
    if case["kind"] == "write":
        t["qkv"] = d.normal(m, hq + 2 * hkv, dim).to(torch.bfloat16)
        t["gq"], t["gk"] = ((1.0 + 0.1 * d.normal(dim)).to(torch.bfloat16) for _ in range(2))
        at = t["slot"]
        if case["axes"] == 1:
            t["positions"] = at[:, None].astype(np.int32) + d.host.integers(0, 100000)
        else:  # time, height, width of image rows far into a conversation
            t["positions"] = np.stack([at // 256 + 30000, at // 16 % 16 + 30000, at % 16 + 30000], 1).astype(np.int32)
        t["turns"] = THETA ** (-np.arange(0, case["rotary"], 2, dtype=np.float64) / case["rotary"]) / (2 * math.pi)
        t["axis"] = (np.arange(case["rotary"] // 2) * case["axes"] // (case["rotary"] // 2)).astype(np.int32)
    else:
        t["q"] = (1.5 * d.normal(m, hq, dim)).to(torch.bfloat16)
    t["pages"], t["page_offsets"], t["pool"] = _tables(d, lengths, case["page"])
    t["k"], t["k_scale"] = _cache(d, case, t["pool"])
    t["v"], t["v_scale"] = _cache(d, case, t["pool"])
    if case["cache"] == "e4m3":
        t["k_scale"], t["v_scale"] = KEY_SCALE * t["k_scale"], VALUE_SCALE * t["v_scale"]
    return t


# -- the plain form ------------------------------------------------------------

def _device(x):
    return torch.as_tensor(x).to("cuda")


class _Plain:
    """What the plain form keeps: the inputs, with the step's integers on the GPU."""

    def __init__(self, case, t):
        self.case = case
        self.t = {name: _device(v) if isinstance(v, np.ndarray) else v for name, v in t.items()}
        self.longest = int(t["lengths"].max())
        self.rows = int(np.diff(t["row_offsets"]).max())


def _plain_attention(s):
    """Sequences padded to the longest: rows [n, rows], keys [n, longest]."""
    case, t = s.case, s.t
    n, hq, hkv, dim, page = case["sequences"], case["query_heads"], case["kv_heads"], case["head_dim"], case["page"]
    lengths, offsets = t["lengths"].long()[:, None], t["row_offsets"].long()
    j = torch.arange(s.longest, device="cuda")
    entry = torch.minimum(t["page_offsets"][:-1].long()[:, None] + j // page, t["page_offsets"][1:].long()[:, None] - 1)
    at, slot = t["pages"][entry].long(), (j % page)[None].expand(n, -1)

    def gathered(cache, scale):
        if case["cache"] == "bf16":
            return cache[at, :, slot].float().transpose(1, 2).contiguous()
        codes = cache.view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn).float()
        step = scale[at, slot // _block(case)] if case["cache"] == "e4m3_blocks" else scale[None, None]
        return (codes * step[..., None]).transpose(1, 2).contiguous()

    i = torch.arange(s.rows, device="cuda")
    counts = offsets[1:] - offsets[:-1]
    position = (t["lengths"].long() - counts)[:, None] + i
    last = position[:, :, None]
    keep = (j <= last) & (j < lengths[:, :, None])
    if case["window"]:
        keep = keep & ((j > last - case["window"]) | (j < case["sinks"]))
    row = torch.minimum(offsets[:-1, None] + i, offsets[1:, None] - 1)
    q = t["q"][row].float().view(n, s.rows, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, dim)
    scores = torch.matmul(q, gathered(t["k"], t["k_scale"]).transpose(2, 3).contiguous()) / math.sqrt(dim)
    scores = scores.view(n, hkv, hq // hkv, s.rows, s.longest).masked_fill(~keep[:, None, None], -math.inf)
    top = scores.amax(dim=4, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(dim=4, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), gathered(t["v"], t["v_scale"])).view(n, hkv, hq // hkv, s.rows, dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s.rows, hq, dim)
    m = torch.arange(t["q"].shape[0], device="cuda")
    sequence = torch.searchsorted(offsets[1:], m, right=True)
    return o[sequence, m - offsets[sequence]].to(torch.bfloat16)


def _rotated(u, cos, sin, rotary, pairing):
    """u [M, heads, D] with its first `rotary` values turned; cos, sin [M, rotary / 2]."""
    half = rotary // 2
    x, rest = u[..., :rotary], u[..., rotary:]
    a, b = (x[..., :half], x[..., half:]) if pairing == "half" else (x[..., 0::2], x[..., 1::2])
    c, s = cos[:, None], sin[:, None]
    turned = (a * c - b * s, b * c + a * s)
    x = torch.cat(turned, dim=-1) if pairing == "half" else torch.stack(turned, dim=-1).flatten(-2)
    return torch.cat([x, rest], dim=-1)


def _least_step(amax):
    """The smallest power of two with amax <= 448 of it."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa 2^exponent, mantissa in [0.5, 1)
    exponent = exponent - 9 + (mantissa > 0.875).int()
    return torch.exp2(torch.where(amax > 0, exponent, LEAST).clamp(LEAST, MOST).double()).float()


def _codes(values, step):
    return (values / step).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_write(s):
    case, t = s.case, s.t
    hq, hkv, page, block = case["query_heads"], case["kv_heads"], case["page"], _block(case)
    x = t["qkv"].float()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(dim=-1, keepdim=True) + EPSILON) * t["gq"].float()
        k = k * torch.rsqrt(k.square().mean(dim=-1, keepdim=True) + EPSILON) * t["gk"].float()
    angle = 2 * math.pi * torch.frac(t["positions"].double()[:, t["axis"].long()] * t["turns"])
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = (_rotated(u, cos, sin, case["rotary"], case["pairing"]) for u in (q, k))
    rows, offsets, slot = torch.arange(case["rows"], device="cuda"), t["row_offsets"].long(), t["slot"] % page
    sequence = torch.searchsorted(offsets[1:], rows, right=True)
    at = t["pages"][t["page_offsets"][sequence].long() + t["slot"] // page].long()
    index = (at * (page // block) + slot // block)[:, None].expand(-1, hkv)
    # the block that each sequence's first row falls into, and its tokens from before
    first = t["slot"][offsets[:-1]]
    place = t["pages"][t["page_offsets"][:-1].long() + first // page].long()
    inside = first // block * block % page + torch.arange(block, device="cuda")[:, None]
    old = (inside < first % page).t()  # [n, block]
    begun = torch.zeros(t["k_scale"].numel() // hkv, dtype=torch.bool, device="cuda")
    begun[place * (page // block) + first % page // block] = first % block > 0

    def append(cache, table, values):
        codes, steps = cache.view(torch.uint8), table.view(-1, hkv)
        amax = torch.zeros_like(steps).scatter_reduce(0, index, values.abs().amax(dim=2), "amax")
        step = _least_step(amax)
        step = torch.where(begun[:, None], torch.maximum(step, steps), step)
        mine = place * (page // block) + first % page // block
        held = codes[place[:, None], :, inside.t()]  # [n, block, heads, dim]
        raised = _codes(held.view(torch.float8_e4m3fn).float() * steps[mine][:, None, :, None], step[mine][:, None, :, None])
        codes[place[:, None], :, inside.t()] = torch.where(old[:, :, None, None], raised, held)
        written = torch.gather(step, 0, index)
        codes[at, :, slot] = _codes(values, written[:, :, None])
        steps.scatter_(0, index, written)

    append(t["k"], t["k_scale"], k)
    append(t["v"], t["v_scale"], v)
    return [q.to(torch.bfloat16), t["k"], t["v"], t["k_scale"], t["v_scale"]]


# -- the framework's side ------------------------------------------------------

_runtime = None


def _rt():
    """The process's runtime: one context, stream and loaded code object."""
    global _runtime
    if _runtime is None:
        from lunaflux_amd import fp8
        torch.cuda.init()
        _runtime = fp8.ProjectionRuntime(0)
    return _runtime


class _Bytes:
    """A device allocation as an array torch can wrap (it keeps the
    allocation). Device addresses do not cross the framework's boundary, so
    the address is taken from the allocation's handle: {vtable, magic and
    kind, counters, flag, parent, base, size}."""

    def __init__(self, allocation):
        self.allocation = allocation
        words = (ctypes.c_uint64 * 8).from_address(allocation.ptr)
        if words[1] & 0xFFFFFFFF != 0x4C464855 or words[7] != allocation.byte_count:
            raise RuntimeError("unexpected allocation handle")
        self.__cuda_array_interface__ = dict(shape=(allocation.byte_count,), typestr="|u1",
                                             data=(int(words[6]), False), strides=None, version=2)


def _view(allocation, dtype, shape, offset=0):
    count = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
    return torch.as_tensor(_Bytes(allocation), device="cuda")[offset:offset + count].view(dtype).view(shape)


def _held(x):
    """An allocation with x's values."""
    x = _device(x).contiguous()
    a = _rt().context.allocate(x.nbytes)
    _view(a, x.dtype, tuple(x.shape)).copy_(x)
    return a


def _region(a):
    return a.region(0, a.byte_count, 256)


class _Own:
    """A bound operation, its output views and what it reads."""

    def __init__(self, operation, outputs, keep):
        self.operation, self.outputs, self.keep = operation, outputs, keep


def _own(case, t):
    from lunaflux_amd import attention
    rt = _rt()
    hq, hkv, dim, blocks = case["query_heads"], case["kv_heads"], case["head_dim"], case["cache"] == "e4m3_blocks"
    m, kind = int(t["row_offsets"][-1]), case["kind"]
    rotary = attention.Rotary(t["turns"], t["axis"], case["pairing"]) if kind == "write" else None
    layer = attention.attention_layer(
        rt, query_heads=hq, kv_heads=hkv, head_dim=dim, cache=case["cache"], page_size=case["page"], pages=t["pool"],
        max_tokens=m, max_sequences=case["sequences"], table_entries=len(t["pages"]),
        k_scales=None if blocks else t["k_scale"].cpu().numpy(), v_scales=None if blocks else t["v_scale"].cpu().numpy(),
        rotary=rotary, norm_epsilon=EPSILON if case.get("norm") else None, window=case.get("window", 0),
        sinks=case.get("sinks", 0))
    step = attention.PagedStep(rt, layer)
    tables = np.split(t["pages"], t["page_offsets"][1:-1])
    step.stage(t["row_offsets"], t["lengths"], tables, t["positions"] if kind == "write" else None,
               prefill_rows=0 if kind == "decode" else case["sequences"])

    def cache(codes, scale):
        """The cache's allocation: codes, and behind them the blocks' scales; views of both."""
        a = rt.context.allocate(layer.cache_bytes)
        held = [_view(a, codes.dtype, tuple(codes.shape))]
        held[0].view(torch.uint8).copy_(codes.view(torch.uint8))
        if blocks:
            held.append(_view(a, torch.float32, tuple(scale.shape), layer.block_scales_offset))
            held[1].copy_(scale)
        return a, held

    (k, k_views), (v, v_views) = cache(t["k"], t["k_scale"]), cache(t["v"], t["v_scale"])
    out = rt.context.allocate(m * hq * dim * 2)
    out_view = _view(out, torch.bfloat16, (m, hq, dim))
    if kind != "write":
        q = _held(t["q"])
        bind = attention.bind_paged_decode if kind == "decode" else attention.bind_paged_prefill
        op = bind(rt, layer, step, _region(q), _region(out), _region(k), _region(v))
        return _Own(op, out_view, [q, k, v])
    qkv, gq, gk = _held(t["qkv"]), _held(t["gq"]), _held(t["gk"])
    op = attention.bind_qk_norm_rope(rt, layer, step, _region(qkv), _region(gq) if case["norm"] else None,
                                     _region(gk) if case["norm"] else None, _region(out), _region(k), _region(v))
    return _Own(op, [out_view, k_views[0], v_views[0], k_views[1], v_views[1]], [qkv, gq, gk])


def prepare(case, seed):
    t = _inputs(case, seed)
    return _own(case, t) if own else _Plain(case, t)


def run(state):
    if own:
        state.operation.launch(_rt().stream, synchronous=False)
        return state.outputs
    return _plain_write(state) if state.case["kind"] == "write" else _plain_attention(state)


# -- work and the 64-bit result --------------------------------------------------

def work(case):
    hq, hkv, dim, size = case["query_heads"], case["kv_heads"], case["head_dim"], 2 if case["cache"] == "bf16" else 1
    rows, before = _rows_and_before(case)
    m = int(rows.sum())
    if case["kind"] == "write":
        blocks = float(((before + rows + _block(case) - 1) // _block(case) - before // _block(case)).sum())
        return {"bytes": m * (2.0 * (2 * hq + 2 * hkv) * dim + 2 * hkv * dim) + 8.0 * hkv * blocks,
                "flops": 6.0 * m * (hq + hkv) * dim}
    seen, pairs = 0, 0  # tokens that some row sees, (row, token) pairs
    for r, b in zip(rows.tolist(), before.tolist()):
        last = np.arange(b, b + r)
        low = np.maximum(0, last + 1 - case["window"]) if case["window"] else np.zeros(r, np.int64)
        sinks = np.minimum(case["sinks"], low)
        pairs += int((last + 1 - low + sinks).sum())
        seen += int(b + r - low[0] + sinks[0])
    scales = 8.0 * hkv * seen / _block(case) if case["cache"] == "e4m3_blocks" else 0.0
    return {"bytes": 2.0 * seen * hkv * dim * size + scales + 4.0 * m * hq * dim, "flops": 4.0 * pairs * hq * dim}


def exact(case, seed):
    """run()'s result from the definitions in 64 bits. New and raised codes are
    given in steps of their scale, before their rounding."""
    t = _inputs(case, seed)
    return _exact_write(case, t) if case["kind"] == "write" else _exact_attention(case, t)


def _exact_attention(case, t):
    hq, hkv, dim, page = case["query_heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = hq // hkv
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for s, length in enumerate(t["lengths"].tolist()):
        r0, r1 = t["row_offsets"][s:s + 2].tolist()
        token = np.arange(length)
        at, slot = _device(t["pages"][t["page_offsets"][s] + token // page]).long(), _device(token % page)
        for h in range(hkv):
            def side(name):
                x = t[name].view(torch.bfloat16 if case["cache"] == "bf16" else torch.uint8)[at, h, slot].view(t[name].dtype).double()
                scale = t[name + "_scale"].double()
                return x * (scale[at, slot // _block(case), h][:, None] if case["cache"] == "e4m3_blocks" else scale[h])
            k, v = side("k").t().contiguous(), side("v")
            for a in range(r0, r1, 2048):
                b = min(r1, a + 2048)
                z = (t["q"][a:b, h * group:(h + 1) * group].double().reshape(-1, dim) @ k) / dim ** 0.5
                position = torch.arange(length - r1 + a, length - r1 + b, device="cuda").repeat_interleave(group)[:, None]
                hidden = _device(token) > position
                if case["window"]:
                    hidden |= (_device(token) <= position - case["window"]) & (_device(token) >= case["sinks"])
                z[hidden] = -math.inf
                out[a:b, h * group:(h + 1) * group] = (torch.softmax(z, dim=1) @ v).view(b - a, group, dim)
    return out.cpu()


def _exact_write(case, t):
    hq, hkv, page, rotary, half, block = case["query_heads"], case["kv_heads"], case["page"], case["rotary"], case["rotary"] // 2, _block(case)
    x = t["qkv"].double()
    heads = x[:, :hq + hkv].clone()
    if case["norm"]:
        heads /= torch.sqrt((heads ** 2).mean(dim=2, keepdim=True) + EPSILON)
        heads[:, :hq] *= t["gq"].double()
        heads[:, hq:] *= t["gk"].double()
    turn = _device(t["positions"][:, t["axis"]].astype(np.float64) * t["turns"])
    z = torch.polar(torch.ones_like(turn), 2 * math.pi * (turn - torch.floor(turn)))[:, None]
    i = torch.arange(half, device="cuda")
    first, second = (i, i + half) if case["pairing"] == "half" else (2 * i, 2 * i + 1)
    w = torch.complex(heads[..., first], heads[..., second]) * z
    heads[..., first], heads[..., second] = w.real, w.imag
    caches, tables = [], []
    for name, values in (("k", heads[:, hq:]), ("v", x[:, hq + hkv:])):
        values = values.cpu().numpy()
        cache, table = t[name].double().cpu().numpy(), t[name + "_scale"].double().cpu().numpy()
        for s in range(case["sequences"]):
            a, end = t["row_offsets"][s:s + 2].tolist()
            while a < end:
                token = int(t["slot"][a])
                count = min(end - a, block - token % block)
                p, b, lo = int(t["pages"][t["page_offsets"][s] + token // page]), token % page // block, token % page
                begin = lo - token % block
                rows = values[a:a + count]  # [count, heads, dim]
                amax = np.abs(rows).max(axis=(0, 2))
                step = 2.0 ** np.clip(np.ceil(np.log2(np.maximum(amax, 1e-300) / 448.0)), LEAST, MOST)
                if lo > begin:
                    step = np.maximum(step, table[p, b])
                    cache[p, :, begin:lo] *= (table[p, b] / step)[:, None, None]
                cache[p, :, lo:lo + count] = np.clip(rows.transpose(1, 0, 2) / step[:, None, None], -448, 448)
                table[p, b] = step
                a += count
        caches.append(torch.from_numpy(cache))
        tables.append(torch.from_numpy(table))
    return [heads[:, :hq].cpu()] + caches + tables
