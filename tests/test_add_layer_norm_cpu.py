"""Refusals of bpt_add_layer_norm, which takes whole pieces of 8 elements on 16-byte boundaries only.  None needs a GPU."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from bpt_b200 import _lib, build
    build.build()
    return _lib.lib()


def call(lib, **kw):
    p = 4096  # never dereferenced: every call below is refused before a launch
    a = dict(x=p, r=p, gamma=p, beta=p, eps=1e-5, y=p, rows=4, dim=64, dtype=0, stream=None)
    a.update(kw)
    return lib.bpt_add_layer_norm(*a.values())


def test_refusals(lib):
    for dim in (0, -8, 4, 12, 300, 4097, 4104, 8192):
        assert call(lib, dim=dim) == 1 and b"multiple of 8 in [8, 4096]" in lib.bpt_last_error()
    for name in ("x", "r", "gamma", "beta", "y"):
        for address in (4098, 4104):
            assert call(lib, **{name: address}) == 1 and b"16-byte" in lib.bpt_last_error()
    assert call(lib, rows=-1) == 1
    assert call(lib, x=None) == 1 and call(lib, y=None) == 1
    assert call(lib, dtype=1) == 4 and call(lib, dtype=9) == 4
    assert call(lib, rows=0, x=None, y=None) == 0
