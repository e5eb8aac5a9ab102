"""The attention block's operators between the projections, as cases to be timed.

  write   per-head norm, rotary positions and cache append of the packed Q|K|V
          rows (attention.bind_qk_norm_rope)
  decode  attention of one new token per sequence over the paged cache
          (attention.bind_paged_decode)
  adapt   low-rank adapters of many requests beside a shared projection
          (low_rank.bind_low_rank)

Heads and widths are Llama-3-8B's (32 query and 8 key / value heads of 128,
hidden 4096, packed Q|K|V 6144, intermediate 14336), a small model's (hidden
512) or generic ones. `run` computes them in elementary torch operations, or,
where `own` is true, with the framework's kernels.
"""
import ctypes
import math

import numpy as np
import torch

own = False

EPSILON = 1e-6
THETA = 500000.0
KEY_SCALE, VALUE_SCALE = 0.03, 0.02  # steps of an e4m3 cache (times 1 + head / 16)


def listed():
    return [
        # A small model, a few short conversations: launch latency.
        _decode("decode_small", 3, 61, 0.6, 8, 8, 64, "bf16", 16),
        # Ordinary continuous batching of a grouped-query model.
        _decode("decode_b32", 32, 2311, 0.7, 32, 8, 128, "bf16", 16),
        # One user with a very long context: the split over the length.
        _decode("decode_long", 1, 131071, 0.0, 32, 8, 128, "bf16", 64),
        # A large ragged batch over an e4m3 cache.
        _decode("decode_e4m3", 96, 5003, 0.9, 32, 8, 128, "e4m3", 32),
        # The decode step's new rows of that batch.
        _write("write_m32", 32, 32, 32, 8, 128, 128, "half", True, 1, "bf16", 16),
        # A long prompt, or many prompts at once.
        _write("write_m8192", 8192, 5, 32, 8, 128, 128, "half", True, 1, "bf16", 16),
        # Image and text rows with time, height and width positions, e4m3 cache.
        _write("write_axes_m1021", 1021, 3, 28, 4, 128, 128, "half", False, 3, "e4m3", 32),
        # Partial rotation of neighbouring pairs, small heads.
        _write("write_partial_m333", 333, 7, 12, 12, 64, 32, "neighbour", False, 1, "bf16", 8),
        # Adapters on a small model's Q|K|V.
        _adapt("adapt_small", 4, 512, 512, 512, 16, 4, 1),
        # Decode: 61 requests over 16 adapters, Llama Q|K|V.
        _adapt("adapt_decode", 61, 4096, 4096, 1024, 16, 16, 1),
        # Prefill: prompts of a few hundred rows each.
        _adapt("adapt_prefill", 4093, 4096, 4096, 1024, 64, 8, 700),
        # One output (the down projection) from the intermediate width.
        _adapt("adapt_down", 509, 14336, 4096, 0, 32, 5, 100),
    ]


def _decode(name, sequences, longest, spread, query_heads, kv_heads, head_dim, cache, page, window=0):
    return dict(name=name, kind="decode", sequences=sequences, longest=longest, spread=spread,
                query_heads=query_heads, kv_heads=kv_heads, head_dim=head_dim, cache=cache, page=page, window=window)


def _write(name, rows, sequences, query_heads, kv_heads, head_dim, rotary, pairing, norm, axes, cache, page):
    return dict(name=name, kind="write", rows=rows, sequences=sequences, query_heads=query_heads, kv_heads=kv_heads,
                head_dim=head_dim, rotary=rotary, pairing=pairing, norm=norm, axes=axes, cache=cache, page=page)


def _adapt(name, rows, hidden, nq, nkv, rank, adapters, run):
    """run: mean number of consecutive rows of one adapter; nkv 0: one output of nq columns."""
    return dict(name=name, kind="adapt", rows=rows, hidden=hidden, nq=nq, nkv=nkv, rank=rank, adapters=adapters, run=run)


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
    kind = rng.choice(["decode", "write", "adapt"])
    hq, hkv, d = rng.choice(HEADS)
    cache, page = rng.choice(["bf16", "bf16", "e4m3"]), rng.choice([8, 16, 32, 64, 128])
    if kind == "decode":
        sequences = _log_uniform(rng, 1, 256)
        most = 500_000_000 // (sequences * hkv * d * (4 if cache == "bf16" else 2))
        longest = _log_uniform(rng, 8, max(8, min(131072, most)))
        return _decode("", sequences, longest, round(rng.uniform(0, 0.95), 2), hq, hkv, d, cache, page,
                       rng.choice([0, 0, 0, max(1, longest // 3)]))
    if kind == "write":
        rows = _log_uniform(rng, 1, 8192 * 6144 // ((hq + 2 * hkv) * d) if d > 64 else 8192)
        return _write("", rows, rng.randint(1, min(rows, 64)), hq, hkv, d, rng.choice([d, d, d // 2]),
                      rng.choice(["half", "half", "neighbour"]), rng.random() < 0.5, rng.choice([1, 1, 3]), cache, page)
    rows = _log_uniform(rng, 1, 4096)
    hidden, nq, nkv = rng.choice([(4096, 4096, 1024), (4096, 4096, 0), (512, 512, 512), (2048, 2048, 512), (1408, 2048, 0)])
    return _adapt("", rows, hidden, nq, nkv, rng.choice([16, 16, 32, 64]), rng.randint(1, 16),
                  1 if rows <= 128 else _log_uniform(rng, 16, 1000))


# -- inputs, from the seed -----------------------------------------------------

def _lengths(case):
    """Cached tokens of each sequence: the longest down to (1 - spread) of it."""
    s = np.arange(case["sequences"])
    return np.maximum(1, np.round(case["longest"] * (1 - case["spread"] * ((s * 0.6180339887) % 1.0)))).astype(np.int64)


def _rows_of(case):
    """Rows of each sequence of a write case, and the tokens cached before them."""
    n, rows = case["sequences"], case["rows"]
    cuts = np.concatenate([[0], np.sort((np.arange(1, n) * rows) // n + (np.arange(1, n) % 3 - 1) * (rows // n > 2)), [rows]])
    return np.diff(cuts), (np.arange(n) * 37 + 5) % 200


class _Draws:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.host = np.random.default_rng(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")


def _cache(d, case, pages):
    """One side of a paged cache [pages, kv heads, page, head dim]: N(0, 1) values, or codes of their e4m3 steps."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=d.g)
    return x if case["cache"] == "bf16" else (x * 30.0).to(torch.float8_e4m3fn)


def _tables(d, lengths, page):
    """Page table of each sequence (pages of a shuffled pool), its offsets, and the pool's size."""
    counts = -(-lengths // page)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    pool = int(offsets[-1]) + 3
    return d.host.permutation(pool)[:offsets[-1]].astype(np.int32), offsets.astype(np.int32), pool


def _scales(case):
    step = 1.0 + torch.arange(case["kv_heads"], device="cuda") / 16.0
    one = case["cache"] == "bf16"
    return (torch.ones_like(step), torch.ones_like(step)) if one else (KEY_SCALE * step, VALUE_SCALE * step)


def _inputs(case, seed):
    d = _Draws(seed)
    if case["kind"] == "adapt":
        return _adapt_inputs(case, d)
    hq, hkv, dim = case["query_heads"], case["kv_heads"], case["head_dim"]
    t = {}
    if case["kind"] == "decode":
        lengths = d.host.permutation(_lengths(case))
        t["row_offsets"] = np.arange(case["sequences"] + 1, dtype=np.int32)
        t["q"] = (1.5 * d.normal(case["sequences"], hq, dim)).to(torch.bfloat16)
    else:
        new, before = _rows_of(case)
        order = d.host.permutation(case["sequences"])
        new, before = new[order], before[order]
        lengths = new + before
        t["row_offsets"] = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        t["qkv"] = d.normal(case["rows"], hq + 2 * hkv, dim).to(torch.bfloat16)
        t["gq"], t["gk"] = ((1.0 + 0.1 * d.normal(dim)).to(torch.bfloat16) for _ in range(2))
        at = np.concatenate([before[s] + np.arange(new[s]) for s in range(case["sequences"])])
        t["slot"] = at
        if case["axes"] == 1:
            t["positions"] = at[:, None].astype(np.int32) + d.host.integers(0, 100000)
        else:  # time, height, width of image rows far into a conversation
            t["positions"] = np.stack([at // 256 + 30000, at // 16 % 16 + 30000, at % 16 + 30000], 1).astype(np.int32)
        t["turns"] = THETA ** (-np.arange(0, case["rotary"], 2, dtype=np.float64) / case["rotary"]) / (2 * math.pi)
        t["axis"] = (np.arange(case["rotary"] // 2) * case["axes"] // (case["rotary"] // 2)).astype(np.int32)
    t["lengths"] = lengths.astype(np.int32)
    t["pages"], t["page_offsets"], t["pool"] = _tables(d, lengths, case["page"])
    t["k"], t["v"] = _cache(d, case, t["pool"]), _cache(d, case, t["pool"])
    t["k_scale"], t["v_scale"] = _scales(case)
    return t


def _slices(case):
    return [case["nq"]] + ([case["nkv"]] * 2 if case["nkv"] else [])


def _adapt_inputs(case, d):
    m, k, r, n = case["rows"], case["hidden"], case["rank"], case["adapters"]
    widths = _slices(case)
    # runs of rows of one adapter; one in eight has none
    runs = np.repeat(d.host.integers(0, n, m), np.maximum(1, d.host.integers(1, 2 * case["run"], m)) if case["run"] > 1 else 1)[:m]
    t = dict(ids=np.where(d.host.random(m) < 0.125, -1, runs) if case["run"] == 1 else runs)
    t["ids"] = t["ids"].astype(np.int32)
    t["x"] = d.normal(m, k).to(torch.bfloat16)
    t["y"] = d.normal(m, sum(widths)).to(torch.bfloat16)
    t["a"] = (d.normal(n, len(widths) * r, k) / math.sqrt(k)).to(torch.bfloat16)
    t["b"] = (0.1 * d.normal(n, sum(widths), r)).to(torch.bfloat16)
    t["scaling"] = 0.5 + torch.arange(n, device="cuda") / n
    return t


# -- the plain form ------------------------------------------------------------

def _device(x):
    return torch.as_tensor(x).to("cuda")


class _Plain:
    """What the plain form keeps: the inputs, with the step's integers on the GPU."""

    def __init__(self, case, t):
        self.case = case
        self.t = {name: _device(v) if isinstance(v, np.ndarray) else v for name, v in t.items()}
        self.longest = int(t["lengths"].max()) if "lengths" in t else 0


def _plain_decode(s):
    case, t = s.case, s.t
    n, hq, hkv, dim, page = case["sequences"], case["query_heads"], case["kv_heads"], case["head_dim"], case["page"]
    lengths = t["lengths"].long()
    j = torch.arange(s.longest, device="cuda")
    last = t["page_offsets"][1:].long() - 1
    entry = torch.minimum(t["page_offsets"][:-1].long()[:, None] + (j // page)[None], last[:, None])
    at, slot = t["pages"][entry].long(), (j % page)[None].expand(n, -1)

    def gathered(cache, scale):
        if cache.dtype == torch.bfloat16:
            return cache[at, :, slot].float().transpose(1, 2)
        raw = cache.view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn)
        return (raw.float() * scale[:, None]).transpose(1, 2)

    keep = j[None] < lengths[:, None]
    if case["window"]:
        keep = keep & (j[None] >= lengths[:, None] - case["window"])
    q = t["q"].float().view(n, hkv, hq // hkv, dim)
    scores = torch.matmul(q, gathered(t["k"], t["k_scale"]).contiguous().transpose(2, 3).contiguous()) / math.sqrt(dim)
    scores = scores.masked_fill(~keep[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(dim=3, keepdim=True))
    o = torch.matmul(p, gathered(t["v"], t["v_scale"]).contiguous()) / p.sum(dim=3, keepdim=True)
    return o.reshape(n, hq, dim).to(torch.bfloat16)


def _rotated(u, cos, sin, rotary, pairing):
    """u [M, heads, D] with its first `rotary` values turned; cos, sin [M, rotary / 2]."""
    half = rotary // 2
    x, rest = u[..., :rotary], u[..., rotary:]
    a, b = (x[..., :half], x[..., half:]) if pairing == "half" else (x[..., 0::2], x[..., 1::2])
    c, s = cos[:, None], sin[:, None]
    turned = (a * c - b * s, b * c + a * s)
    x = torch.cat(turned, dim=-1) if pairing == "half" else torch.stack(turned, dim=-1).flatten(-2)
    return torch.cat([x, rest], dim=-1)


def _plain_write(s):
    case, t = s.case, s.t
    hq, hkv, page = case["query_heads"], case["kv_heads"], case["page"]
    x = t["qkv"].float()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(dim=-1, keepdim=True) + EPSILON) * t["gq"].float()
        k = k * torch.rsqrt(k.square().mean(dim=-1, keepdim=True) + EPSILON) * t["gk"].float()
    angle = 2 * math.pi * torch.frac(t["positions"].double()[:, t["axis"].long()] * t["turns"])
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = (_rotated(u, cos, sin, case["rotary"], case["pairing"]) for u in (q, k))
    rows = torch.arange(case["rows"], device="cuda")
    sequence = torch.searchsorted(t["row_offsets"][1:].long(), rows, right=True)
    at = t["pages"][t["page_offsets"][sequence].long() + t["slot"] // page].long()

    def append(cache, values, scale):
        if cache.dtype == torch.bfloat16:
            cache[at, :, t["slot"] % page] = values.to(torch.bfloat16)
        else:
            codes = (values / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            cache.view(torch.uint8)[at, :, t["slot"] % page] = codes.view(torch.uint8)

    append(t["k"], k, t["k_scale"])
    append(t["v"], v, t["v_scale"])
    return [q.to(torch.bfloat16), t["k"], t["v"]]


def _plain_adapt(s):
    """Every row against every adapter's A, then its own picked out; the rest of the wide row zero for B."""
    case, t = s.case, s.t
    m, r, n, widths = case["rows"], case["rank"], case["adapters"], _slices(case)
    ids = t["ids"].long()
    mine = torch.arange(n, device="cuda")[None] == ids[:, None]
    low = torch.matmul(t["x"].float(), t["a"].float().flatten(0, 1).t()).view(m, n, len(widths), r)
    low = torch.where(mine[:, :, None, None], low * t["scaling"][None, :, None, None], 0.0)
    b = t["b"].float().split(widths, dim=1)
    added = [torch.matmul(low[:, :, i].reshape(m, n * r), b[i].permute(0, 2, 1).reshape(n * r, -1))
             for i in range(len(widths))]
    return (t["y"].float() + torch.cat(added, dim=1)).to(torch.bfloat16)


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


def _view(allocation, dtype, shape):
    count = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
    return torch.as_tensor(_Bytes(allocation), device="cuda")[:count].view(dtype).view(shape)


def _held(x, rows=None):
    """An allocation of `rows` rows (its own by default) that starts with x's values."""
    x = _device(x).contiguous()
    a = _rt().context.allocate(x.nbytes if rows is None else x.nbytes // max(1, x.shape[0]) * rows)
    _view(a, x.dtype, tuple(x.shape)).copy_(x)
    return a


def _region(a):
    return a.region(0, a.byte_count, 256)


class _Own:
    """A bound operation, its output views and what it reads."""

    def __init__(self, operation, outputs, keep):
        self.operation, self.outputs, self.keep = operation, outputs, keep


def _own_attention(case, t):
    from lunaflux_amd import attention
    rt = _rt()
    hq, hkv, dim = case["query_heads"], case["kv_heads"], case["head_dim"]
    m = int(t["row_offsets"][-1])
    rotary = None
    if case["kind"] == "write":
        rotary = attention.Rotary(t["turns"], t["axis"], case["pairing"])
    layer = attention.attention_layer(
        rt, query_heads=hq, kv_heads=hkv, head_dim=dim, cache=case["cache"], page_size=case["page"], pages=t["pool"],
        max_tokens=m, max_sequences=case["sequences"], table_entries=len(t["pages"]),
        k_scales=t["k_scale"].cpu().numpy(), v_scales=t["v_scale"].cpu().numpy(), rotary=rotary,
        norm_epsilon=EPSILON if case.get("norm") else None, window=case.get("window", 0))
    step = attention.PagedStep(rt, layer)
    tables = np.split(t["pages"], t["page_offsets"][1:-1])
    decode = case["kind"] == "decode"
    step.stage(t["row_offsets"], t["lengths"], tables, None if decode else t["positions"],
               prefill_rows=0 if decode else case["sequences"])
    k, v = _held(t["k"]), _held(t["v"])
    out = rt.context.allocate(m * hq * dim * 2)
    if decode:
        q = _held(t["q"])
        op = attention.bind_paged_decode(rt, layer, step, _region(q), _region(out), _region(k), _region(v))
        return _Own(op, _view(out, torch.bfloat16, (m, hq, dim)), [q, k, v])
    qkv, gq, gk = _held(t["qkv"]), _held(t["gq"]), _held(t["gk"])
    op = attention.bind_qk_norm_rope(rt, layer, step, _region(qkv), _region(gq) if case["norm"] else None,
                                     _region(gk) if case["norm"] else None, _region(out), _region(k), _region(v))
    outputs = [_view(out, torch.bfloat16, (m, hq, dim))] + [_view(a, t["k"].dtype, tuple(t["k"].shape)) for a in (k, v)]
    return _Own(op, outputs, [qkv, gq, gk])


def _own_adapt(case, t):
    from lunaflux_amd import low_rank
    rt = _rt()
    m = case["rows"]
    counts = rt.step_counts(m)
    x, y, a, b, scaling, ids = (_held(t[name]) for name in ("x", "y", "a", "b", "scaling", "ids"))
    out = rt.context.allocate(y.byte_count)
    adapters = low_rank.LowRankAdapters(rt, hidden=case["hidden"], widths=_slices(case), rank=case["rank"],
                                        adapters=case["adapters"], a=_region(a), b=_region(b), scaling=_region(scaling))
    op = low_rank.bind_low_rank(rt, counts, _region(ids), _region(x), adapters, _region(y), _region(out), m)
    return _Own(op, _view(out, torch.bfloat16, tuple(t["y"].shape)), [counts, x, y, a, b, scaling, ids, adapters])


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _own_adapt(case, t) if case["kind"] == "adapt" else _own_attention(case, t)
    return _Plain(case, t)


def run(state):
    if own:
        state.operation.launch(_rt().stream, synchronous=False)
        return state.outputs
    return {"decode": _plain_decode, "write": _plain_write, "adapt": _plain_adapt}[state.case["kind"]](state)


# -- work and the 64-bit result --------------------------------------------------

def work(case):
    if case["kind"] == "adapt":
        m, k, widths, r = case["rows"], case["hidden"], _slices(case), case["rank"]
        used = min(case["adapters"], max(1.0, m / case["run"]))
        n = sum(widths)
        return {"bytes": 2.0 * m * (k + 2 * n) + 2.0 * used * r * (len(widths) * k + n),
                "flops": 2.0 * m * r * (len(widths) * k + n)}
    hq, hkv, dim, size = case["query_heads"], case["kv_heads"], case["head_dim"], 2 if case["cache"] == "bf16" else 1
    if case["kind"] == "write":
        m = case["rows"]
        return {"bytes": float(m * (2 * (2 * hq + 2 * hkv) * dim + 2 * hkv * dim * size)), "flops": 6.0 * m * (hq + hkv) * dim}
    lengths = _lengths(case)
    tokens = int(np.minimum(lengths, case["window"]).sum() if case["window"] else lengths.sum())
    return {"bytes": float(2 * tokens * hkv * dim * size + 4 * case["sequences"] * hq * dim), "flops": 4.0 * tokens * hq * dim}


def exact(case, seed):
    """run()'s result from the definitions in 64 bits. An e4m3 cache's new values
    are given in steps of their scale, before their rounding."""
    t = _inputs(case, seed)
    if case["kind"] == "adapt":
        return _exact_adapt(case, t)
    return _exact_decode(case, t) if case["kind"] == "decode" else _exact_write(case, t)


def _exact_decode(case, t):
    hq, hkv, dim, page = case["query_heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(case["sequences"], hq, dim, dtype=torch.float64, device="cuda")
    for s, length in enumerate(t["lengths"].tolist()):
        first = max(0, length - case["window"]) if case["window"] else 0
        j = np.arange(first, length)
        at = _device(t["pages"][t["page_offsets"][s] + j // page]).long()
        slot = _device(j % page)
        for h in range(hkv):
            k = t["k"].view(torch.uint8 if case["cache"] == "e4m3" else torch.bfloat16)[at, h, slot].view(t["k"].dtype).double()
            v = t["v"].view(torch.uint8 if case["cache"] == "e4m3" else torch.bfloat16)[at, h, slot].view(t["v"].dtype).double()
            group = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            z = (t["q"][s, group].double() @ (k * t["k_scale"][h].double()).t()) / dim ** 0.5
            out[s, group] = torch.softmax(z, dim=1) @ (v * t["v_scale"][h].double())
    return out.cpu()


def _exact_write(case, t):
    hq, hkv, page, rotary, half = case["query_heads"], case["kv_heads"], case["page"], case["rotary"], case["rotary"] // 2
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
    caches = []
    for name, values in (("k", heads[:, hq:]), ("v", x[:, hq + hkv:])):
        cache = t[name].double()
        scale = t[name + "_scale"].double()[:, None]
        sequence = np.searchsorted(t["row_offsets"][1:], np.arange(case["rows"]), side="right")
        at = _device(t["pages"][t["page_offsets"][sequence] + t["slot"] // page]).long()
        values = values if case["cache"] == "bf16" else (values / scale).clamp(-448, 448)
        cache[at, :, _device(t["slot"] % page)] = values
        caches.append(cache.cpu())
    return [heads[:, :hq].cpu()] + caches


def _exact_adapt(case, t):
    out, r = t["y"].double(), case["rank"]
    ids = _device(t["ids"])
    for adapter in range(case["adapters"]):
        rows = (ids == adapter).nonzero()[:, 0]
        low = t["x"][rows].double() @ t["a"][adapter].double().t()
        column = 0
        for i, width in enumerate(_slices(case)):
            b = t["b"][adapter, column:column + width].double()
            out[rows, column:column + width] += t["scaling"][adapter].double() * (low[:, i * r:(i + 1) * r] @ b.t())
            column += width
    return out.cpu()
