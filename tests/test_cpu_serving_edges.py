"""Calls of the operators on pages that Python has to pass on, or to refuse, before any kernel runs: no GPU needed."""
import inspect

import pytest

torch = pytest.importorskip("torch")

from fishai_engine import paged  # noqa: E402


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


# ------------------------------------------------------------------ arguments by their place
def test_attention_takes_err_and_stream_behind_the_window():
    """arguments that came later stand last, so calls by place mean what they meant"""
    names = list(inspect.signature(paged.attention).parameters)
    assert names[:13] == ["kv", "layer", "q", "q_start", "kv_len", "out", "max_q", "workspace", "seqs", "scale", "window", "err", "stream"]
    kv = paged.PagedKV(torch.zeros(1, 8, 2, 4, 16, 64, dtype=torch.float16), i32(2, 4))
    q = torch.zeros(0, 512, dtype=torch.float16)
    ws = torch.zeros(paged.workspace_bytes(64), dtype=torch.uint8)
    args = (kv, 0, q, i32(3), i32(2), torch.empty_like(q), 3, ws, None, 0.0, 5)
    paged.attention(*args, i32(1), 0)
    paged.attention(*args, None, 0)
    with pytest.raises(ValueError, match="err"):
        paged.attention(*args, i32(2), 0)
