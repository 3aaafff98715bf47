"""Layer norm of a sum, forward and backward: host side of bpt_layer_norm_forward / bpt_layer_norm_backward.

The reference's blocks end each half with `norm(h + sublayer(h))` (modules/attention.py:79-81, 141, 168-171).
`layer_norm(x, weight, bias, eps, residual=r)` is that as one differentiable call: the forward reads x and r once
and writes y, the backward reads x, r and the gradient of y once, writes the one gradient that x and r share, and
sums the gradients of weight and bias over the rows on the way, in a fixed order (no atomics: results do not vary
from run to run).  Statistics and sums are fp32.  The autograd node is compiled (csrc_torch/train_ext.cpp).
"""
from . import train_extension


def layer_norm(x, weight, bias, eps=1e-5, residual=None):
    """LayerNorm(x + residual) over the last dimension; differentiable once in x, residual, weight and bias (a forward-mode
    tangent raises NotImplementedError).

    x: (..., dim) CUDA tensor, fp32, bf16 or fp16, dim from 1 to 8192; weight, bias: (dim,) of x's dtype or None (ones,
    zeros); residual: of x's shape and dtype or None.  Any strides (non-contiguous inputs are copied).  The sum
    x + residual is not rounded before it is normalised.  Biased variance, as torch.nn.LayerNorm.  Runs on the current
    stream of x's device; bad arguments raise RuntimeError."""
    return train_extension().layer_norm(x, weight, bias, eps, residual)
