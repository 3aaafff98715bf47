"""Refusals of layer_norm that need no GPU: the C entry points' argument checks and the Python checks."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from bpt_b200 import _lib, build
    build.build()
    build.build_torch_ext(name="_train_ext")
    return _lib.lib()


def test_c_entry_refuses_bad_arguments(lib):
    p = 4096  # never dereferenced: every call below is refused before a launch
    fwd, bwd = lib.bpt_layer_norm_forward, lib.bpt_layer_norm_backward
    for dim in (0, -8, 8193):
        assert fwd(p, None, p, p, 1e-5, p, None, None, 4, dim, 0, None) == 1 and b"dim" in lib.bpt_last_error()
        assert bwd(p, p, None, p, p, p, p, p, p, 4, dim, 0, p, 1 << 20, None) == 1
        assert lib.bpt_layer_norm_backward_workspace_bytes(4, dim) == 0
    assert fwd(p, None, p, p, 1e-5, p, None, None, -1, 8, 0, None) == 1
    assert fwd(None, None, p, p, 1e-5, p, None, None, 4, 8, 0, None) == 1
    assert fwd(p, None, p, p, 1e-5, p, p, None, 4, 8, 0, None) == 1 and b"together" in lib.bpt_last_error()
    assert fwd(p, None, p, p, 1e-5, p, None, None, 4, 8, 1, None) == 4  # fp64
    assert bwd(p, p, None, p, p, p, p, p, p, 4, 8, 1, p, 1 << 20, None) == 4
    assert bwd(p, p, None, p, None, p, p, p, p, 4, 8, 0, p, 1 << 20, None) == 1
    need = lib.bpt_layer_norm_backward_workspace_bytes(100, 512)
    assert need >= 2 * 4 * 512
    assert bwd(p, p, None, p, p, p, p, p, p, 100, 512, 0, p, need - 1, None) == 3
    assert bwd(p, p, None, p, p, p, p, p, p, 100, 512, 0, None, 0, None) == 3
    assert bwd(p, p, None, p, p, p, None, None, None, 100, 512, 0, None, 0, None) == 0  # nothing is asked for
    assert fwd(None, None, None, None, 1e-5, None, None, None, 0, 8, 0, None) == 0      # no rows
    # the workspace does not grow with the rows beyond the blocks that run
    assert lib.bpt_layer_norm_backward_workspace_bytes(1 << 30, 512) == lib.bpt_layer_norm_backward_workspace_bytes(1 << 20, 512)


def test_cpu_tensors_are_refused(lib):
    from bpt_b200.norm import layer_norm
    x = torch.randn(3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(x, None, None)
