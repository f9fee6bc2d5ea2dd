"""Calls of the operators on pages that Python has to pass on, or to refuse, before any kernel runs: no GPU needed."""
import inspect

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_cpu_serving import call_plan  # noqa: E402

from fishai_engine import _lib as L  # noqa: E402
from fishai_engine import beam, paged, sampling  # noqa: E402


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


# ------------------------------------------------------------------ whole numbers of other libraries
class Whole:
    def __init__(self, v):
        self.v = v

    def __index__(self):
        return self.v


KINDS = [np.int64, np.int32, np.uint32, np.uint8, Whole, torch.tensor]


@pytest.mark.parametrize("kind", KINDS, ids=lambda k: k.__name__)
def test_whole_numbers_of_any_kind(kind):
    """the maximum of an array of lengths is one of numpy's; its value arrives, and calls of no rows end before the device is asked"""
    kv = paged.PagedKV(torch.zeros(1, 8, 2, 4, 16, 64, dtype=torch.float16), i32(2, 4))
    q, k = torch.zeros(0, 512, dtype=torch.float16), torch.zeros(0, 256, dtype=torch.float16)
    ws = torch.zeros(paged.workspace_bytes(64), dtype=torch.uint8)
    for kw in (dict(), dict(window=kind(5)), dict(window=kind(5), sinks=kind(2)), dict(sinks=kind(0))):
        paged.attention(kv, kind(0), q, i32(3), i32(2), torch.empty_like(q), kind(3), ws, **kw)
    with pytest.raises(L.FishaiError, match="layer"):
        paged.attention(kv, kind(1), q, i32(3), i32(2), torch.empty_like(q), kind(3), ws)
    paged.rope_append(kv, kind(0), paged.Rope(64), q, k, k, i32(0), i32(0), torch.empty_like(q))
    paged.rope_append(kv, kind(0), paged.Rope(64, axes=[16, 16]), q, k, k, i32(2, 0), i32(0), torch.empty_like(q), slots=i32(0))
    with pytest.raises(L.FishaiError, match="layer"):
        paged.rope_append(kv, kind(1), paged.Rope(64), q, k, k, i32(0), i32(0), torch.empty_like(q))
    f = torch.zeros(0, 2)
    beam.select(torch.zeros(0, 50), f, None, f.clone(), i32(0, 2), i32(0, 2), None, ws, eos=kind(3), pad=kind(49))
    with pytest.raises(L.FishaiError, match="pad"):
        beam.select(torch.zeros(0, 50), f, None, f.clone(), i32(0, 2), i32(0, 2), None, ws, eos=kind(3), pad=kind(50))


@pytest.mark.parametrize("bad", [3.0, None, b"3", "3"], ids=str)
def test_what_is_no_whole_number_is_refused(bad):
    kv = paged.PagedKV(torch.zeros(1, 8, 2, 4, 16, 64, dtype=torch.float16), i32(2, 4))
    q, k = torch.zeros(0, 512, dtype=torch.float16), torch.zeros(0, 256, dtype=torch.float16)
    ws = torch.zeros(paged.workspace_bytes(64), dtype=torch.uint8)
    good = dict(layer=0, max_q=3, window=5, sinks=2)
    for name in good:
        with pytest.raises(TypeError):
            paged.attention(kv, q=q, q_start=i32(3), kv_len=i32(2), out=torch.empty_like(q), workspace=ws, **{**good, name: bad})
    with pytest.raises(TypeError):
        paged.rope_append(kv, bad, paged.Rope(64), q, k, k, i32(0), i32(0), torch.empty_like(q))
    f = torch.zeros(0, 2)
    for kw in (dict(eos=bad), dict(pad=bad)):
        with pytest.raises(TypeError):
            beam.select(torch.zeros(0, 50), f, None, f.clone(), i32(0, 2), i32(0, 2), None, ws, **kw)


@pytest.mark.parametrize("name", ["layer", "max_q", "window", "sinks"])
@pytest.mark.parametrize("v", [-1, 2 ** 32, 2 ** 70])
def test_numbers_that_32_bits_do_not_hold(name, v):
    kv = paged.PagedKV(torch.zeros(1, 8, 2, 4, 16, 64, dtype=torch.float16), i32(2, 4))
    q, ws = torch.zeros(0, 512, dtype=torch.float16), torch.zeros(paged.workspace_bytes(64), dtype=torch.uint8)
    good = dict(layer=0, max_q=3, window=5, sinks=2)
    for w in (v, np.int64(v)) if v < 2 ** 63 else (v,):
        with pytest.raises(ValueError):
            paged.attention(kv, q=q, q_start=i32(3), kv_len=i32(2), out=torch.empty_like(q), workspace=ws, **{**good, name: w})


# ------------------------------------------------------------------ buffers that are not torch's
class Buffer:
    """what the module asks of a buffer, and nothing else"""

    def __init__(self, t):
        self._t, self.dtype, self.shape = t, t.dtype, tuple(t.shape)

    def data_ptr(self):
        return self._t.data_ptr()

    def stride(self):
        return tuple(self._t.stride())


def test_buffers_with_an_address_type_shape_and_strides():
    """all that is asked of them is looked at before the library sees the call; here it has no rows, or no device to look at"""
    B = Buffer
    kv = paged.PagedKV(torch.zeros(1, 8, 2, 4, 16, 64, dtype=torch.float16), i32(2, 4))
    q, k = torch.zeros(0, 512, dtype=torch.float16), torch.zeros(0, 256, dtype=torch.float16)
    ws = torch.zeros(paged.workspace_bytes(64), dtype=torch.uint8)
    paged.rope_append(kv, 0, paged.Rope(64), B(q), B(k), B(k), B(i32(0)), B(i32(0)), B(q), slots=B(i32(0)), err=B(i32(1)))
    paged.rope_append(kv, 0, paged.Rope(64, axes=[16, 16]), B(q), B(k), B(k), B(i32(2, 0)), B(i32(0)), B(q), slots=B(i32(0)))
    paged.attention(kv, 0, B(q), B(i32(3)), B(i32(2)), B(q), 3, ws, seqs=B(i32(2)), err=B(i32(1)), window=5, sinks=2)
    sampling.sample_logits(B(torch.zeros(3, 50)), B(torch.zeros(0)), B(i32(0)), temperature=B(torch.zeros(0)), top_k=B(i32(0)), rows=B(i32(0)))
    args = dict(add=i32(2), lengths=i32(2), free_pages=i32(8), n_free=i32(1), q_start=i32(3), kv_len=i32(2), positions=i32(5), row_seqs=i32(5))
    with pytest.raises(L.FishaiError, match="fa_step_plan"):
        paged.plan_step(kv, **{n: B(t) for n, t in args.items()})
    for name, bad in (("add", i32(2, 1)), ("add", i32(4)[::2]), ("positions", i32(5, 1)), ("row_seqs", i32(10)[::2]), ("free_pages", i32(2, 4)),
                      ("free_pages", i32(16)[::2]), ("kv_len", torch.zeros(2))):
        with pytest.raises(ValueError, match=name):
            paged.plan_step(kv, **{**{n: B(t) for n, t in args.items()}, name: B(bad)})
    x, f = torch.zeros(3, 50), torch.zeros
    for name, bad in (("u", f(6)[::2]), ("u", f(3, 1)), ("ids", i32(3, 1)), ("ids", i32(6)[::2]), ("temperature", f(6)[::2]), ("top_k", i32(4))):
        with pytest.raises(ValueError, match=name):
            sampling.sample_logits(**{**dict(logits=B(x), u=B(f(3)), ids=B(i32(3))), name: B(bad)})


@pytest.mark.parametrize("name", ["add", "positions", "free_pages"])
def test_plans_of_more_entries_than_32_bits_count(name):
    """2^32 and a few would be taken for those few"""
    kv = paged.PagedKV(torch.zeros(1, 8, 2, 4, 16, 64, dtype=torch.float16), i32(2, 4))
    long = torch.empty(2 ** 32 + 2, dtype=torch.int32, device="meta")
    args = dict(add=i32(2), lengths=i32(2), free_pages=i32(8), n_free=i32(1), q_start=i32(3), kv_len=i32(2), positions=i32(5), row_seqs=i32(5))
    with_it = {"add": ["add", "kv_len"], "positions": ["positions", "row_seqs"], "free_pages": ["free_pages"]}[name]
    args.update({n: long for n in with_it})
    if name == "add":
        args["q_start"] = torch.empty(2 ** 32 + 3, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match=name):
        paged.plan_step(kv, **args)


@pytest.mark.parametrize("cap", [2 ** 31, 2 ** 32 - 8192, 2 ** 32 - 1])
def test_a_stack_beyond_31_bits_is_refused(cap):
    """the kernel steps through the pages that come back 8192 at a time: near 2^32 of them the count would wrap and not end"""
    assert call_plan(free_cap=cap) == L.ERR_INVALID
    assert "2^31" in L.last_error()
    call_plan(free_cap=2 ** 31 - 1)
    assert "2^31" not in L.last_error()
