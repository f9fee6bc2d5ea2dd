import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "fishai-engine_b200"), os.path.join(ROOT, "oracle"), os.path.dirname(__file__)):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")
    config.addinivalue_line("markers", "slow: long-running CPU test")


@pytest.fixture(scope="session")
def oracle():
    import oracle as o
    o.lib()
    return o


@pytest.fixture(autouse=True)
def kept_pages(monkeypatch):
    """Some tests pass C.addressof of an fa_pages that nothing holds any more: each lives as long as its test."""
    from fishai_engine import _lib as L
    made, real = [], L.fa_pages

    def keep(*args, **kw):
        made.append(real(*args, **kw))
        return made[-1]

    monkeypatch.setattr(L, "fa_pages", keep)
