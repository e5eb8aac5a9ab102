"""What a binding uploads to its workspace: zeros where the kernels count, not where they write before they read."""
import numpy as np
import pytest

from lunaflux_amd import _abi, attention
from test_attention_cpu import FIELDS, FakeAllocation, FakeRuntime, region


class Recording(FakeAllocation):
    def __init__(self, byte_count):
        super().__init__(byte_count)
        self.data[:] = 0x5A
        self.uploaded = 0

    def copy_from_host(self, data, offset=0):
        super().copy_from_host(data, offset)
        self.uploaded += np.asarray(data).nbytes


@pytest.mark.parametrize("bind,entry", [(attention.bind_paged_prefill, _abi.ATTN_PREFILL), (attention.bind_paged_decode, _abi.ATTN_DECODE)])
def test_zeros_of_a_workspace(bind, entry):
    rt = FakeRuntime()
    rt.allocate = Recording
    layer = attention.attention_layer(rt, **{**FIELDS, "table_entries": 400})
    q, cache = 2 * 32 * 8 * 128, layer.cache_bytes
    ws = bind(rt, layer, attention.PagedStep(rt, layer), region(q), region(q), region(cache), region(cache)).workspace
    assert ws.byte_count == attention.workspace_bytes(entry, layer.desc)
    prompts = entry == _abi.ATTN_PREFILL
    assert ws.uploaded == (_abi.LF_FP8_ATTN_STATUS_BYTES if prompts else ws.byte_count)
    assert (ws.data[:ws.uploaded] == 0).all() and (ws.byte_count > 1 << 26) == prompts
