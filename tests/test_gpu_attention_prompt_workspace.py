"""Attention of prompts over a workspace that holds anything behind its first line."""
import numpy as np
import pytest

import attention_steps as st
from lunaflux_amd import _abi, fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("byte", [0xFF, 0x01])
def test_partial_results_are_written_before_they_are_read(byte, dim):
    rt, rng = fp8.ProjectionRuntime(0), np.random.default_rng(dim)
    s = st.make_step(rt, rng, rows=[33, 2, 0, 5], before=[2500, 1800, 9, 0], query_heads=4, kv_heads=2, head_dim=dim, page=16)
    q = st.queries(rng, s)
    op, out = st.bind(rt, s, q)
    behind = op.workspace.byte_count - _abi.LF_FP8_ATTN_STATUS_BYTES
    op.workspace.copy_from_host(np.full(behind, byte, np.uint8), offset=_abi.LF_FP8_ATTN_STATUS_BYTES)
    for rows, lengths in (([0, 33, 35, 35, 40], [2533, 1802, 9, 5]), ([0, 0, 1, 1, 1], [0, 1802, 0, 0]), ([0, 33, 35, 35, 40], [2533, 1802, 9, 5])):
        s.step.stage(rows, lengths, s.tables, prefill_rows=4)
        op.launch(rt.stream, synchronous=True)
        op.check()
    st.check(s, st.read(s, out), q, range(4))
