"""A bounded wait of the attention on tcgen05 that runs out: each CTA is told to
leave out one of its copies (fa_debug_set), so that what waits for it gives up
after four seconds, all roles leave, the copies in flight land and the call
sets FLAG_TIMEOUT.  Nothing faults or hangs; the next call is right again."""
import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402
from fishai_engine import _lib as L  # noqa: E402
from fishai_engine import paged  # noqa: E402
from test_gpu_paged import attn, randn, same_bits  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,hd,n,kv,copy", [("f16", 128, 30, 16000, 1), ("f16", 128, 200, 16000, 2), ("bf16", 64, 30, 16000, 3), ("bf16", 64, 200, 16000, 4),
                                            ("f16", 128, 200, 16000, 9), ("f16", 64, 30, 300, 2)])
def test_expired_wait_sets_the_flag_and_the_next_call_is_right(t, hd, n, kv, copy):
    pages, table = R.make_cache([kv], 1, 2, hd, R.TYPES[t], 50)
    wide = torch.zeros(1, 2000, dtype=torch.int32, device="cuda")  # a long table: not a call for the kernel of short ones
    wide[:, : table.shape[1]] = table
    q = randn(2, n, 8 * hd, dtype=R.TYPES[t])
    ws = torch.empty(paged.workspace_bytes(hd), dtype=torch.uint8, device="cuda")
    run = lambda err: attn(pages, wide, q, [0, n], [kv], 8, err=err, workspace=ws)  # noqa: E731
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = run(err)
    torch.cuda.synchronize()
    L.check(L.lib().fa_debug_set(None, L.DEBUG_WITHHOLD_KV, copy))
    try:
        run(err)
        torch.cuda.synchronize()
    finally:
        L.check(L.lib().fa_debug_set(None, L.DEBUG_WITHHOLD_KV, 0))
    assert int(err) == paged.FLAG_TIMEOUT
    err.zero_()
    got = run(err)
    assert int(err) == 0 and same_bits(got, want)
