"""The training operators' torch extension: what autograd may ask of layer_norm and linear_cross_entropy beyond a backward."""
import pytest
import torch
from torch.autograd import forward_ad

from bpt_b200.loss import linear_cross_entropy
from bpt_b200.norm import layer_norm

pytestmark = pytest.mark.gpu


def operands():
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, r, w = (torch.randn(*s, generator=gen, device="cuda") for s in ((12, 64), (12, 64), (50, 64)))
    g, b, wb = (torch.randn(*s, generator=gen, device="cuda") for s in ((64,), (64,), (50,)))
    return dict(x=x, r=r, g=g, b=b), dict(x=x, w=w, wb=wb), torch.randint(0, 50, (12,), generator=gen, device="cuda")


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(grad_mode):
    """A tangent on any input is an error, with and without a node, and never dropped."""
    norm, ce, target = operands()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        for leaf in (False, True):
            for call, inputs in ((lambda x, r, g, b: layer_norm(x, g, b, residual=r), norm),
                                 (lambda x, w, wb: linear_cross_entropy(x, w, target, bias=wb), ce)):
                for name in inputs:
                    given = {k: v.clone().requires_grad_(leaf) for k, v in inputs.items()}
                    given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
                    with pytest.raises(NotImplementedError, match="bpt_b200.*forward-mode"):
                        call(**given)


def test_views_that_hold_negatives():
    """Inputs and gradients that are views of their own negatives in memory (as the imaginary part of a conjugate is) give what
    the written-out numbers give."""
    norm, ce, target = operands()
    for call, inputs in ((lambda x, r, g, b: layer_norm(x, g, b, residual=r), norm),
                         (lambda x, w, wb: linear_cross_entropy(x, w, target, bias=wb, reduction="none"), ce)):
        want = [v.clone().requires_grad_(True) for v in inputs.values()]
        leaves = [v.clone().requires_grad_(True) for v in inputs.values()]
        y, z = call(*want), call(*(torch._neg_view(-v) for v in leaves))
        gy = torch.randn_like(y)
        want = [y.detach()] + list(torch.autograd.grad(y, want, gy))
        got = [z.detach()] + list(torch.autograd.grad(z, leaves, torch._neg_view(-gy)))
        assert all(torch.equal(a, e) for a, e in zip(got, want))
        with torch.no_grad():
            assert torch.equal(call(*(torch._neg_view(-v) for v in inputs.values())), want[0])
    wide = torch.complex(norm["x"], norm["r"]).conj()  # strided, too
    assert wide.imag.is_neg()
    assert torch.equal(layer_norm(wide.imag, None, None), layer_norm(-norm["r"], None, None))
    hidden = torch._neg_view(target - 2 * target)
    assert torch.equal(linear_cross_entropy(ce["x"], ce["w"], hidden), linear_cross_entropy(ce["x"], ce["w"], target))
