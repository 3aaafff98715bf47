"""Refusals of linear_cross_entropy that need no GPU: the C entry points' argument checks, the workspace sizes, the
Python checks."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from bpt_b200 import _lib, build
    build.build()
    build.build_torch_ext(name="_train_ext")
    return _lib.lib()


P = 4096  # an address that is never read: every call below is refused before a launch


def forward(lib, **kw):
    a = dict(x=P, ldx=64, w=P, ldw=64, bias=None, target=P, ignore=-100, smoothing=0.0, reduction=1, loss=P, lse=P, count=P,
             n=10, vocab=100, dim=64, dtype=2, ws=None, nbytes=0)
    a.update(kw)
    return lib.bpt_linear_ce_forward(*a.values(), None)


def backward(lib, **kw):
    a = dict(x=P, ldx=64, w=P, ldw=64, bias=None, target=P, ignore=-100, smoothing=0.0, reduction=1, lse=P, count=P, grad=P,
             dx=P, dw=P, db=P, n=10, vocab=100, dim=64, dtype=2, ws=None, nbytes=0)
    a.update(kw)
    return lib.bpt_linear_ce_backward(*a.values(), None)


def test_c_entries_refuse_bad_arguments(lib):
    for call in (forward, backward):
        for bad in (dict(n=-1), dict(n=1 << 31), dict(vocab=0), dict(vocab=-3), dict(vocab=(1 << 30) + 1), dict(dim=0), dict(ldx=63),
                    dict(ldw=63), dict(smoothing=-0.1), dict(smoothing=1.5), dict(smoothing=float("nan")), dict(reduction=3),
                    dict(reduction=-1), dict(x=None), dict(w=None), dict(target=None), dict(n=1 << 30, vocab=1 << 30)):
            assert call(lib, **bad) == 1, bad
            assert b"linear_ce" in lib.bpt_last_error()
        assert call(lib, dtype=1) == 4 and call(lib, dtype=9) == 4
        assert call(lib) == 3 and b"workspace" in lib.bpt_last_error()
        assert call(lib, ws=P, nbytes=100) == 3
    assert forward(lib, loss=None) == 1
    assert backward(lib, lse=None) == 1 and backward(lib, grad=None) == 1 and backward(lib, count=None) == 1
    assert backward(lib, dx=None, dw=None, db=None) == 0  # nothing is asked for
    assert forward(lib, n=0, reduction=0, loss=None) == 0


def test_workspace_sizes(lib):
    fwd, bwd = lib.bpt_linear_ce_forward_workspace_bytes, lib.bpt_linear_ce_backward_workspace_bytes
    assert fwd(P, 64, P, 64, 0, 100, 64, 2) == 0 and bwd(P, 64, P, 64, 10, 0, 64, 2, 1, 1, 1) == 0
    assert fwd(P, 64, P, 64, 10, 100, 64, 1) == 0
    aligned, moved = fwd(P, 64, P, 64, 1000, 5000, 64, 2), fwd(P + 2, 64, P + 2, 64, 1000, 5000, 64, 2)
    plain = aligned - 1000 * 64 * 2  # aligned features have room for a copy of the ones whose tokens count
    assert moved >= plain + (1000 + 5000) * 64 * 2
    assert fwd(P, 64, P, 64, 1000, 5000, 64, 0) >= plain + (1000 + 5000) * 64 * 6  # three planes
    # the gradient of the logits is kept a piece at a time: far below the 26 GB it would take whole
    big = bwd(P, 512, P, 512, 1 << 18, 50000, 512, 2, 1, 1, 1)
    assert big < (512 << 20) + 6 * 512 * ((1 << 18) + 50000)


def test_python_refusals(lib):
    from bpt_b200.loss import linear_cross_entropy
    x, w, t = torch.randn(3, 8), torch.randn(5, 8), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_cross_entropy(x, w, t)
