"""Host memory that runs out within a call on a cache whose sequences share
pages: the call reports it and every sequence keeps what it holds.  A child
process runs under an operator new that fails where it is told to."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SHIM = r"""
#include <cstdlib>
#include <new>
static thread_local long left = -1;  // allocations until one fails; -1: none does
extern "C" void fail_after(long n) { left = n; }
extern "C" int failed() { return left == -2; }
void *operator new(std::size_t n) {
  if (left == 0) {
    left = -2;
    throw std::bad_alloc();
  }
  if (left > 0) --left;
  if (void *p = std::malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void *p) noexcept { std::free(p); }
void operator delete(void *p, std::size_t) noexcept { std::free(p); }
"""

CHILD = r"""
import ctypes as C
import sys
sys.path[:0] = sys.argv[1].split(":")
import numpy as np
from fishai_engine import _lib as L
from fishai_engine import synth
from fishai_engine.model import ModelWeights
shim = C.CDLL(sys.argv[2])
dev = ModelWeights.load_from_gguf(synth.write_preset("tiny-q8_0", sys.argv[3]))
L.check(L.lib().fa_debug_set(dev._h, L.DEBUG_FIXED_ORDER_SUMS, 1))  # caches filled alike are alike
N = 4

def contents(kv):
    return [[kv.get(layer, s) for layer in range(kv.n_layers())] for s in range(N)]

def equal(a, b):
    return all(np.array_equal(x, y) for s, t in zip(a, b) for p, q in zip(s, t) for x, y in zip(p, q))

def start():
    kv = dev.new_kv_cache(96, dtype=L.KV_F16, n_seq=N)
    rng = np.random.default_rng(0)
    for s, n in enumerate([37, 50, 0, 21]):
        if n:
            dev.prefill(rng.integers(3, dev.config.vocab_size, n).tolist(), 0, kv, seq=s, want_logits=False)
    kv.fork(1, 3)
    return kv

OPS = dict(fork=lambda kv: kv.fork(0, 3), reorder=lambda kv: kv.reorder([1, 0, 0, 1]), truncate=lambda kv: kv.truncate(3, 20),
           compact=lambda kv: kv.compact(1, list(range(3, 50, 2))), clear=lambda kv: kv.clear(3))
rest = [lambda kv: kv.fork(3, 2), lambda kv: kv.reorder([3, 0, 1, 0]), lambda kv: kv.fork(2, 0), lambda kv: kv.truncate(0, 5)]
for name, op in OPS.items():
    good = start()
    before = contents(good)
    op(good)
    after, ends = contents(good), []
    for r in rest:
        r(good)
        ends.append(contents(good))
    fails = 0
    for n in range(60):
        kv = start()
        shim.fail_after(n)
        try:
            op(kv)
            code = L.OK
        except L.FishaiError as e:
            code = e.code
        fail = shim.failed()
        shim.fail_after(-1)
        assert code == (L.ERR_OOM if fail else L.OK), (name, n, code, fail)
        assert equal(contents(kv), before if fail else after), (name, n, "contents")
        if fail:
            fails += 1
            op(kv)
            assert equal(contents(kv), after), (name, n, "again")
        for r, e in zip(rest, ends):
            r(kv)
            assert equal(contents(kv), e), (name, n, "then")
        if not fail:
            break
    print(name, "failed at", fails, "places")
for n in range(60):
    shim.fail_after(n)
    h = C.c_void_p()
    rc = L.lib().fa_kv_create(dev._h, 4, 96, L.KV_F16, C.byref(h))
    fail = shim.failed()
    shim.fail_after(-1)
    assert rc == (L.ERR_OOM if fail else L.OK), (n, rc)
    if rc == L.OK:
        L.lib().fa_kv_free(h)
        break
print("done")
"""


def test_memory_that_runs_out_leaves_the_cache_whole(tmp_path):
    src, so, py = tmp_path / "shim.cpp", tmp_path / "shim.so", tmp_path / "child.py"
    src.write_text(SHIM)
    py.write_text(CHILD)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    paths = ":".join(os.path.join(root, p) for p in ("fishai-engine_b200", "oracle", "tests"))
    r = subprocess.run([sys.executable, str(py), paths, str(so), str(tmp_path / "tiny.gguf")], env={**os.environ, "LD_PRELOAD": str(so)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout + r.stderr[-3000:]
