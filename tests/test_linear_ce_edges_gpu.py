"""linear_cross_entropy at the edges of its number formats, against the formula in 64 bits.

Tolerances are those of test_linear_ce_gpu's note (u = 2^-24, Ez, Ep), which hold for every entry with the absolute values of
its own row and column; what is added to them stands at each test."""
import pytest
import torch

from test_linear_ce_gpu import DTYPES, IGNORE, U, check, inputs, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("down", [12, 40, 52, 90])
@pytest.mark.parametrize("of", ["x", "w", "x up, w down"])
def test_fp32_columns_of_very_different_size(of, down):
    """One feature far below the others: its column of d w has what that column of x keeps, its column of d x what that of w
    does.  One far above the others in x and as far below in w: the logits have what the other columns of x keep."""
    for n, dim in ((300, 72), (70, 73), (90, 1100)):
        x, w, b, t = inputs(n, 500, dim, torch.float32, padded=0.1)
        for c in (5, dim - 100) if dim > 512 else (5,):
            if of == "x":
                x[:, c] *= 2.0 ** -down
            elif of == "w":
                w[:, c] *= 2.0 ** -down
            else:
                x[:, c] *= 2.0 ** down
                w[:, c] *= 2.0 ** -down
        check(x, w, b, t, smoothing=0.1)


@pytest.mark.parametrize("up", [100, 108, 110, -100, -108, -110])
def test_fp32_sizes_far_from_one(up):
    """x times 2^up and w times 2^-up: the same logits."""
    x, w, b, t = inputs(300, 500, 72, torch.float32, padded=0.1)
    check(x * 2.0 ** up, w * 2.0 ** -up, b, t, smoothing=0.1)
