"""The calls on a model's cache behind a caller's own work on its pages: each
follows the default stream, and other streams where KVCache.wait names them."""
import numpy as np
import pytest

from fishai_engine import _lib as L
from fishai_engine import paged
from fishai_engine.model import ModelWeights
from fishai_engine.sampling import Sampler, SamplerConfig
from test_gpu_beam import dev, fill, path  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def late_row(kv, seq, slot, stream, n_sleep=40_000_000):
    """A row of new K and V for every layer, written on `stream` only after it has slept: what it holds then"""
    pk = paged.PagedKV.of(kv)
    KVH, hd = pk.n_kv_heads, pk.head_dim
    g = torch.Generator(device="cuda").manual_seed(slot)
    k, v = (torch.randn(1, KVH * hd, device="cuda", generator=g).half() for _ in range(2))
    q, out = torch.zeros(1, KVH * hd, device="cuda").half(), torch.empty(1, KVH * hd, device="cuda").half()
    pos, seqs, slots = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, seq, slot))
    rope = paged.Rope(hd)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(n_sleep)
        for layer in range(pk.n_layers):
            paged.rope_append(pk, layer, rope, q, k, v, pos, seqs, out, slots=slots, stream=stream.cuda_stream)
    return k[0], v[0], (pk, q, out, pos, seqs, slots, rope)  # kept until the work is done


def holds(kv, seq, slot, k, v):
    d = kv.kv_dim
    for layer in range(kv.n_layers()):
        a, b = kv.get(layer, seq)
        if not (np.array_equal(a[slot * d: (slot + 1) * d], k.float().cpu().numpy()) and
                np.array_equal(b[slot * d: (slot + 1) * d], v.float().cpu().numpy())):
            return False
    return True


@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("op", ["get", "fork", "reorder", "truncate", "compact", "forward", "prefill", "decode",
                                "decode batch"])
def test_calls_on_a_cache_follow_work_on_its_pages(dev, side, op):  # noqa: F811
    """rows that a caller's stream has still to write are there for the call behind it: work on the default stream by
    itself, on another one through KVCache.wait"""
    kv = dev.new_kv_cache(96, dtype=L.KV_F16, n_seq=3)
    fill(dev, kv, [37, 20, 5])
    if op == "truncate":
        kv.fork(0, 1)  # sequence 0's first pages are shared, so that dropping to 18 copies two rows of one
    stream = torch.cuda.Stream() if side else torch.cuda.default_stream()
    slot = 36 if op != "truncate" else 17
    other = dev.new_kv_cache(96, dtype=L.KV_F16, n_seq=1)
    step = {"forward": lambda c: dev.forward([11], 37, c, seq=0), "prefill": lambda c: dev.prefill([5, 6, 7], 37, c, seq=0)[0],
            "decode": lambda c: np.asarray(dev.decode_greedy(c, 11, 37, 4, seq=0)),
            "decode batch": lambda c: dev.decode_batch(c, [11], [37], Sampler(SamplerConfig.greedy(), dev.config.vocab_size, seeds=[0]), 1,
                                                       want_logits=True)[1]}.get(op)
    if step:  # the same on a cache whose row is there before
        fill(dev, other, [37])
        k, v, keep = late_row(other, 0, slot, torch.cuda.default_stream(), 1)
        torch.cuda.synchronize()
    k, v, keep = late_row(kv, 0, slot, stream)
    if side:
        kv.wait(stream.cuda_stream)
    at = 0, slot
    if op == "get":
        a, b = kv.get(0, 0)
        assert np.array_equal(a[slot * kv.kv_dim: (slot + 1) * kv.kv_dim], k.float().cpu().numpy())
    elif op == "fork":
        kv.fork(0, 1)
        at = 1, slot
    elif op == "reorder":
        kv.reorder([2, 0, 0])
        at = 2, slot
    elif op == "truncate":
        kv.truncate(0, 18)
    elif op == "compact":
        kv.compact(0, [0, 5, 20, 36])
        at = 0, 3
    else:
        got = step(kv)
        assert np.array_equal(got, step(other))
    torch.cuda.synchronize()
    assert holds(kv, *at, k, v)


def test_wait_refuses_a_stream_that_is_captured(dev):  # noqa: F811
    kv = dev.new_kv_cache(32, dtype=L.KV_F16, n_seq=2)
    kv.wait()  # pages that nobody has: nothing to follow
    x = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        x += 1
        with pytest.raises(L.FishaiError) as e:
            kv.wait(torch.cuda.current_stream().cuda_stream)
        assert e.value.code == L.ERR_INVALID
        x += 1
    g.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [2.0] * 4  # the capture went on
    fill(dev, kv, [20])  # and the model's stream is not part of it
    kv.fork(0, 1)
    assert L.lib().fa_kv_wait(None, None) == L.ERR_INVALID


def test_calls_on_a_cache_whose_model_is_freed_are_refused(path):  # noqa: F811
    model = ModelWeights.load_from_gguf(path)
    kv = model.new_kv_cache(64, dtype=L.KV_F16, n_seq=3)
    fill(model, kv, [37, 20])
    kv.fork(0, 2)
    model.close()
    for call in (lambda: kv.get(0, 0), lambda: kv.fork(0, 1), lambda: kv.reorder([1, 0]), lambda: kv.truncate(2, 18), lambda: kv.compact(0, [1, 5]),
                 lambda: kv.wait(), lambda: paged.PagedKV.of(kv)):
        with pytest.raises(L.FishaiError) as e:
            call()
        assert e.value.code == L.ERR_INVALID
    kv.truncate(1, 3)  # nothing shared: no work on the GPU
    assert kv.seq_len_with_dim(0, kv.kv_dim, 1) == 3
