"""Softmax cross entropy fused with the projection that makes the logits: host side of bpt_linear_ce_forward /
bpt_linear_ce_backward.

The reference's models end in a generator (modules/model.py:8-17: projection, log-softmax) whose log-probabilities the
task scripts hand to a loss: nll_loss (lm.py:120-140), or a summed KL divergence from smoothed targets
(loss/__init__.py:4-28), which is the summed cross entropy with label smoothing minus the targets' entropy.
`linear_cross_entropy(x, weight, target, bias)` is projection and cross entropy as one differentiable call.  The (tokens, vocabulary) logits
are made tile by tile and never kept: the forward keeps one number per token, the backward makes them again, a piece
of tokens x vocabulary at a time.  Results do not vary from run to run.  The autograd node is compiled
(csrc_torch/train_ext.cpp).
"""
from . import train_extension

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """cross_entropy(x @ weight.T + bias, target) without the logits in memory; differentiable once in x, weight, bias (a
    forward-mode tangent raises NotImplementedError).

    x: (..., dim) and weight: (vocab, dim), CUDA tensors of one dtype (fp32, bf16, fp16); bias: (vocab,) of that dtype
    or None; target: int64 of x's leading shape.  Returns fp32: a scalar, or target's shape for reduction="none".

    A token whose target is ignore_index has loss 0 and no gradient, whatever its features hold; the mean is over the
    other tokens (NaN if there are none).  Any other target outside [0, vocab) makes its loss NaN, and the gradients
    that it reaches (nothing is read out of range; there is no check on the host, which would have to wait for the
    device).  label_smoothing as torch.nn.functional.cross_entropy defines it.

    Rows of x and weight may have any stride; other layouts are copied.  bf16 and fp16 rows that start on 16-byte
    boundaries are read where they lie, others are copied into the workspace first; fp32 operands are split there into
    two fp16 planes, or three bf16 planes where the sizes of rows, of columns or (reduction "none") of the tokens' gradients
    differ by more than 2^24, which keeps fp32 accuracy on the tensor cores, with two limits: numbers of an operand below
    2^-110 keep fewer bits, and with two planes a logit's gradient is held to 2^-21 of itself or 2^-49 of the largest token's
    gradient, so a row of d weight whose class has a probability far below 2^-28 for every token has few bits, or is zero.
    fp16: the latter bound is 2^-39.  For more than 256 tokens of bf16 or fp16 a logit's gradient is rounded to that type before the
    products.  Forward and backward may be captured into CUDA graphs.  Runs on the current stream of x's device;
    bad arguments raise RuntimeError."""
    if reduction not in _REDUCTIONS:
        raise RuntimeError("bpt_b200: linear_cross_entropy: reduction must be none, mean or sum")
    return train_extension().linear_cross_entropy(x, weight, target, bias, ignore_index, label_smoothing, _REDUCTIONS[reduction])
