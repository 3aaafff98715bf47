"""bpt_add_layer_norm by itself, against the formula in 64 bits (tolerances: test_layer_norm_gpu's note; where a lane has up to
64 elements its sums are chains of 8 and of 8 additions, so the note's 25 levels cover them) and against
bpt_layer_norm_forward, with widths and numbers of rows on both sides of the rule that gives a row to one warp or to several."""
import pytest
import torch

from bpt_b200 import _lib
from test_layer_norm_gpu import DTYPES, formula, inputs, near

pytestmark = pytest.mark.gpu

SHAPES = [(rows, dim) for rows in (1, 9, 2049) for dim in (8, 248, 256, 264, 512, 520, 768, 776, 1024, 1032, 1280, 1536, 1544, 2048, 2056, 4096)]
SHAPES += [(8192, 2048), (8193, 2048), (20001, 40), (20001, 520)]


def run(x, r, w, b, eps=1e-5):
    p, code, rows, dim = _lib.ptr, _lib.dtype_code(x.dtype), x.size(0), x.size(1)
    held = torch.full((x.numel() + 64,), 7.0, dtype=x.dtype, device="cuda")
    y = held[:x.numel()].view_as(x)
    _lib.check(_lib.lib().bpt_add_layer_norm(p(x), p(r), p(w), p(b), eps, p(y), rows, dim, code, _lib.stream()))
    assert bool((held[x.numel():] == 7.0).all())
    same, mean_rstd = torch.empty_like(x), torch.empty((2, rows), device="cuda")
    for stats in ((None, None), (mean_rstd[0].data_ptr(), mean_rstd[1].data_ptr())):
        _lib.check(_lib.lib().bpt_layer_norm_forward(p(x), p(r), p(w), p(b), eps, p(same), *stats, rows, dim, code, _lib.stream()))
        assert bool(((y == same) | (y.isnan() & same.isnan())).all())
    return y, mean_rstd


@pytest.mark.parametrize("dtype", DTYPES)
def test_values(dtype):
    for rows, dim in SHAPES:
        x, r, w, b, gy = inputs(rows, dim, dtype, True, seed=rows + dim)
        for given in ((x, r, w, b), (x, None, None, b), (x, r, w, None)):
            y, (mean, rstd) = run(*given)
            want, off = formula(*given, gy, 1e-5)
            near(y, want[0], off[0])
            a = x.double() if given[1] is None else x.double() + r.double()
            exact = 1 / torch.sqrt(a.var(1, unbiased=False) + 1e-5)
            S = a.abs().amax(1) * exact + 1
            assert bool(((mean.double() - a.mean(1)).abs() <= 2.0 ** -19 * a.abs().amax(1)).all())
            assert bool(((rstd.double() / exact - 1).abs() <= 2.0 ** -19 * S).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_finite_stay_to_themselves(dtype):
    for rows, dim in ((50, 256), (50, 520), (50, 4096)):
        x, r, w, b, _ = inputs(rows, dim, dtype, True)
        want, _ = run(x, r, w, b)
        x[7, dim - 1], x[20, 0] = float("nan"), float("inf")
        got, _ = run(x, r, w, b)
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[7] = keep[20] = False
        assert torch.equal(got[keep], want[keep]) and not bool(torch.isfinite(got[7]).any())
        assert bool(torch.isnan(got[20]).all())


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows are as in a call of their own, forward and backward."""
    from bpt_b200.norm import layer_norm
    rows, dim = (1 << 31) // 512 + 5000, 512
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda")
    last = slice(rows - 6000, rows)
    part, r, w, b, gy = inputs(6000, dim, torch.bfloat16, True)
    x.zero_()
    x[last] = part
    grad = torch.zeros_like(x)
    grad[last] = gy
    leaf, weight = x.requires_grad_(True), w.clone().requires_grad_(True)
    y = layer_norm(leaf, weight, b)
    few, weight_of_few = part.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = layer_norm(few, weight_of_few, b)
    assert torch.equal(y.detach()[last], want.detach())
    y.backward(grad)
    want.backward(gy)
    assert torch.equal(leaf.grad[last], few.grad)
    full = formula(part, None, w, b, gy, 1e-5)  # the other rows add nothing
    near(weight.grad, full[0][2], full[1][2])
