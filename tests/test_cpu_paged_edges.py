"""Calls at the edges of what the paged operators and the beam selection allow,
as the host takes them: no GPU needed, no pointer is read."""
import pytest

from fishai_engine import _lib as L
from test_cpu_paged import P, call_attn


@pytest.mark.parametrize("chunks", [1 << 31, (1 << 32) - 128, (1 << 32) - 1])
def test_attention_refuses_more_chunks_than_the_kernels_count(chunks):
    assert call_attn(chunks=chunks, seq=P) == L.ERR_INVALID
    assert "chunks" in L.last_error()
