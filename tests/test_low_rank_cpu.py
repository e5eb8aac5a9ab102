"""Low-rank adapters without a GPU: descriptor, sizes, geometry and refusals."""
import ctypes

import numpy as np
import pytest

from lunaflux_amd import _abi, low_rank
from lunaflux_amd.device import DeviceError
from test_attention_cpu import FakeAllocation, FakeRuntime, region


def test_descriptor_and_geometry():
    d = low_rank.low_rank_descriptor(16, 16, 4096, [4096, 1024, 1024], 64)
    assert ctypes.sizeof(d) == 64 and bytes(d)[:4] == b"LRNK"
    assert list(d.ends) == [4096, 5120, 6144, 0] and d.columns == 6144 and d.slices == 3 and d.splits >= 1
    entries = (_abi.LOW_RANK_ONE_LAUNCH, _abi.LOW_RANK_SHRINK, _abi.LOW_RANK_EXPAND)
    geometry = [low_rank.launch_geometry(e, d) for e in entries]
    assert geometry[0][1] == "lf_low_rank_n1" and geometry[1:] == [None, None]
    assert geometry[0][0].grid == (4 * 16, 6, 1) and d.slots == 16 and d.one_launch == 1
    assert low_rank.workspace_bytes(d) == 256
    for rank, hidden, rows, first, last in ((32, 4096, 128, "n2", None), (64, 2048, 128, "n4", None),
                                            (128, 1024, 1, "n4", None), (128, 4096, 32, "n4", None), (80, 4096, 128, "shrink_64x64", "expand_64x128"),
                                            (16, 4096, 256, "n1", None), (64, 4096, 128, "shrink_64x64", "expand_16x64"),
                                            (64, 4096, 256, "shrink_64x64", "expand_16x64"),
                                            (16, 4096, 257, "shrink_64x32", "expand_16x32"),
                                            (48, 14336, 1, "shrink_64x64", "expand_16x64"),
                                            (80, 14336, 1, "shrink_64x64", "expand_64x128"),
                                            (16, 128, 513, "shrink_64x32", "expand_64x32"),
                                            (64, 128, 513, "shrink_64x64", "expand_64x64")):
        d = low_rank.low_rank_descriptor(5, rank, hidden, [512, 64], rows)
        names = [g[1][len("lf_low_rank_"):] for g in (low_rank.launch_geometry(e, d) for e in entries) if g is not None]
        assert names == [n for n in (first, last) if n], (rank, hidden, rows)
    for rows, widths, block, blocks in ((128, [1600, 64], 1024, 3), (512, [1600, 64], 512, 5), (4096, [4096, 1024, 1024], 1024, 6),
                                        (2048, [4096, 1024, 1024], 512, 12)):
        d = low_rank.low_rank_descriptor(4, 16, 4096, widths, rows)
        assert (d.block_columns, d.column_blocks) == (block, blocks)
    d = low_rank.low_rank_descriptor(16, 16, 4096, [512], 300)  # 5 tiles of 64 rows, 19 of 16
    assert d.slots == 8 and d.splits == 2
    assert low_rank.launch_geometry(_abi.LOW_RANK_SHRINK, d)[0].grid == (16, 8, 1)
    assert low_rank.launch_geometry(_abi.LOW_RANK_EXPAND, d)[0].grid == (24, 4, 1)
    d = low_rank.low_rank_descriptor(4, 128, 512, [512], 4096)
    geometry = [low_rank.launch_geometry(e, d) for e in entries]
    assert geometry[0] is None and [g[1] for g in geometry[1:]] == ["lf_low_rank_shrink_64x64", "lf_low_rank_expand_64x128"]
    for name in ("n1", "n2", "n4", "shrink_64x32", "shrink_64x64", "expand_16x32", "expand_16x64", "expand_64x32",
                 "expand_64x64", "expand_64x128"):
        assert b"lf_low_rank_" + name.encode() + b"\0" in _abi.code_object_bytes()
    assert low_rank.workspace_bytes(d) >= 256 + 4096 * 128 * 4
    for bad in (low_rank.LowRankDescriptor(),):
        with pytest.raises(DeviceError):
            low_rank.workspace_bytes(bad)
        with pytest.raises(DeviceError):
            low_rank.launch_geometry(_abi.LOW_RANK_SHRINK, bad)
    with pytest.raises(DeviceError):
        low_rank.launch_geometry(4, d)


@pytest.mark.parametrize("args", [
    (0, 16, 512, [512], 8), (65537, 16, 512, [512], 8), (-1, 16, 512, [512], 8), (2, 8, 512, [512], 8),
    (2, 24, 512, [512], 8), (2, 144, 512, [512], 8), (2, 16, 500, [512], 8), (2, 16, 0, [512], 8),
    (2, 16, 1 << 40, [512], 8), (2, 16, 512, [], 8), (2, 16, 512, [64] * 5, 8), (2, 16, 512, [96], 8),
    (2, 16, 512, [512, 0], 8), (2, 16, 512, [-64, 128], 8), (2, 16, 512, [1 << 40], 8), (2, 16, 512, [512], 0),
    (2, 16, 512, [1 << 20], 1 << 24), (2, 16, 512, [512], 1 << 25), (2, 16, 512, [512], 1 << 40), (1 << 40, 16, 512, [512], 8),
])
def test_descriptor_refusals(args):
    with pytest.raises(DeviceError):
        low_rank.low_rank_descriptor(*args)


def adapters(rt, **changes):
    kw = dict(hidden=256, widths=[128, 64], rank=16, adapters=3, a=region(2 * 3 * 32 * 256), b=region(2 * 3 * 192 * 16),
              scaling=region(12, 4))
    return low_rank.LowRankAdapters(rt, **{**kw, **changes})


def test_adapter_refusals():
    rt = FakeRuntime()
    adapters(rt)
    for bad in (dict(a=region(2 * 3 * 32 * 256 - 2)), dict(b=region(2 * 3 * 192 * 16 - 1)), dict(scaling=region(11, 4)),
                dict(a=region(2 * 3 * 32 * 256, 8)), dict(scaling=region(12, 2)), dict(rank=12), dict(widths=[100])):
        with pytest.raises(DeviceError):
            adapters(rt, **bad)
    a, b, s = np.zeros((3, 2, 10, 256), np.uint16), np.zeros((3, 192, 10), np.uint16), np.ones(3, np.float32)
    assert low_rank.LowRankAdapters.upload(rt, a, b, s, [128, 64]).rank == 16
    for bad in ((a[0], b, s), (a[:2], b, s), (a[:, :1], b, s), (a, b[:, :64], s), (a, b[:, :, :9], s), (a, b, s[:2])):
        with pytest.raises(DeviceError):
            low_rank.LowRankAdapters.upload(rt, *bad, [128, 64])


def test_binding_refusals():
    rt = FakeRuntime()
    ad, counts = adapters(rt), FakeAllocation(20)
    x, y = region(2 * 8 * 256), region(2 * 8 * 192)
    bind = lambda ids=region(32, 4), x=x, y=y, out=y, m=8: low_rank.bind_low_rank(rt, counts, ids, x, ad, y, out, m)  # noqa: E731
    assert [s.name for s in bind().steps] == ["lf_low_rank_n1"]
    wide = FakeAllocation(4 * 8 * 192)
    part = lambda offset: wide_region(wide, offset)  # noqa: E731
    bind(y=part(0), out=part(2 * 8 * 192))
    for bad in (dict(ids=region(31, 4)), dict(ids=region(32, 2)), dict(x=region(2 * 8 * 256 - 2)), dict(x=region(2 * 8 * 256, 8)),
                dict(y=region(2 * 8 * 192 - 2), out=y), dict(out=region(2 * 8 * 192 - 2)), dict(m=9), dict(m=0),
                dict(y=part(0), out=part(384)), dict(y=part(384), out=part(0)), dict(out=x)):
        with pytest.raises(DeviceError):
            bind(**bad)


def wide_region(alloc, offset):
    from lunaflux_amd.device import KernelArgument
    return KernelArgument.device_region(alloc, offset, 2 * 8 * 192, 16)
