"""Softmax cross entropy fused with the projection that makes the logits: host side of bpt_linear_ce_forward /
bpt_linear_ce_backward.

The reference's models end in a generator (modules/model.py:8-17: projection, log-softmax) whose log-probabilities the
task scripts hand to a loss: nll_loss (lm.py:120-140) or label smoothing (loss/__init__.py:4-28).
`linear_cross_entropy(x, weight, target, bias)` is both as one differentiable call.  The (tokens, vocabulary) logits
are made tile by tile and never kept: the forward keeps one number per token, the backward makes them again, a piece
of tokens x vocabulary at a time.  Results do not vary from run to run.
"""
import torch

from . import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows(t):
    """(t or a copy whose rows are contiguous, row stride in elements).  The stride of a single row is free."""
    if t.size(0) == 1 and (t.size(1) == 1 or t.stride(1) == 1):
        return t, (t.size(1) + 7) // 8 * 8
    if (t.stride(1) != 1 and t.size(1) != 1) or t.stride(0) < t.size(1):
        t = t.contiguous()
    return t, max(t.stride(0), t.size(1))


def _check(x, weight, target, bias, label_smoothing, reduction):
    if not x.is_cuda:
        raise RuntimeError("bpt_b200: expected a CUDA tensor (there is no CPU path)")
    if x.dtype not in _DTYPES:
        raise RuntimeError("bpt_b200: linear_cross_entropy: unsupported dtype %s" % x.dtype)
    if weight.dim() != 2 or x.dim() < 1 or weight.size(0) < 1 or weight.size(1) < 1 or x.size(-1) != weight.size(1):
        raise RuntimeError("bpt_b200: linear_cross_entropy: x must be (..., dim) and weight (vocab, dim), got %s and %s"
                           % (tuple(x.shape), tuple(weight.shape)))
    if weight.dtype != x.dtype or weight.device != x.device:
        raise RuntimeError("bpt_b200: linear_cross_entropy: weight must be a %s tensor on %s" % (x.dtype, x.device))
    if bias is not None and (bias.dtype != x.dtype or bias.device != x.device or bias.shape != weight.shape[:1]):
        raise RuntimeError("bpt_b200: linear_cross_entropy: bias must be a %s tensor of shape (%d,) on %s"
                           % (x.dtype, weight.size(0), x.device))
    if target.dtype != torch.int64 or target.device != x.device or target.shape != x.shape[:-1]:
        raise RuntimeError("bpt_b200: linear_cross_entropy: target must be an int64 tensor of shape %s on %s"
                           % (tuple(x.shape[:-1]), x.device))
    if reduction not in _REDUCTIONS:
        raise RuntimeError("bpt_b200: linear_cross_entropy: reduction must be none, mean or sum")
    if not 0.0 <= label_smoothing <= 1.0:
        raise RuntimeError("bpt_b200: linear_cross_entropy: label_smoothing must be in [0, 1]")


def _forward(x, ldx, weight, ldw, target, bias, ignore_index, smoothing, reduction, keep):
    """(loss, lse, count); the last two None without keep."""
    lib = _lib.lib()
    n, dim = x.shape
    vocab = weight.size(0)
    dev, code = x.device, _lib.dtype_code(x.dtype)
    loss = torch.empty(n if reduction == 0 else (), dtype=torch.float32, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev) if keep else None
    count = torch.empty((), dtype=torch.float32, device=dev) if keep else None
    xp, wp = x.data_ptr(), weight.data_ptr()
    with torch.cuda.device(dev):
        nbytes = lib.bpt_linear_ce_forward_workspace_bytes(xp, ldx, wp, ldw, n, vocab, dim, code)
        ws = _lib.workspace(nbytes, dev)
        _lib.check(lib.bpt_linear_ce_forward(xp, ldx, wp, ldw, _lib.ptr(bias), target.data_ptr(), ignore_index, smoothing,
                                             reduction, loss.data_ptr(), _lib.ptr(lse), _lib.ptr(count), n, vocab, dim, code,
                                             ws.data_ptr(), nbytes, _lib.stream()))
    return loss, lse, count


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index, smoothing, reduction):
        (xr, ldx), (wr, ldw) = _rows(x), _rows(weight)
        loss, lse, count = _forward(xr, ldx, wr, ldw, target, bias, ignore_index, smoothing, reduction, True)
        ctx.save_for_backward(x, weight, bias, target, lse, count)
        ctx.options = (ignore_index, smoothing, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, bias, target, lse, count = ctx.saved_tensors
        ignore_index, smoothing, reduction = ctx.options
        (x, ldx), (weight, ldw) = _rows(x), _rows(weight)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        lib = _lib.lib()
        n, dim = x.shape
        vocab = weight.size(0)
        dev, dtype, code = x.device, x.dtype, _lib.dtype_code(x.dtype)
        grad = grad.contiguous()
        dx = torch.empty((n, dim), dtype=dtype, device=dev) if need_x else None
        dw = torch.empty((vocab, dim), dtype=dtype, device=dev) if need_w else None
        db = torch.empty(vocab, dtype=dtype, device=dev) if need_b else None
        xp, wp = x.data_ptr(), weight.data_ptr()
        with torch.cuda.device(dev):
            nbytes = lib.bpt_linear_ce_backward_workspace_bytes(xp, ldx, wp, ldw, n, vocab, dim, code, need_x, need_w, need_b)
            ws = _lib.workspace(nbytes, dev)
            _lib.check(lib.bpt_linear_ce_backward(xp, ldx, wp, ldw, _lib.ptr(bias), target.data_ptr(), ignore_index, smoothing,
                                                  reduction, lse.data_ptr(), count.data_ptr(), grad.data_ptr(), _lib.ptr(dx),
                                                  _lib.ptr(dw), _lib.ptr(db), n, vocab, dim, code, ws.data_ptr(), nbytes,
                                                  _lib.stream()))
        return dx, dw, db, None, None, None, None


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """cross_entropy(x @ weight.T + bias, target) without the logits in memory; differentiable once in x, weight, bias.

    x: (..., dim) and weight: (vocab, dim), CUDA tensors of one dtype (fp32, bf16, fp16); bias: (vocab,) of that dtype
    or None; target: int64 of x's leading shape.  Returns fp32: a scalar, or target's shape for reduction="none".

    A token whose target is ignore_index has loss 0 and no gradient, whatever its features hold; the mean is over the
    other tokens (NaN if there are none).  Any other target outside [0, vocab) makes its loss NaN, and the gradients
    that it reaches (nothing is read out of range; there is no check on the host, which would have to wait for the
    device).  label_smoothing as torch.nn.functional.cross_entropy defines it.

    Rows of x and weight may have any stride; other layouts are copied.  bf16 and fp16 rows that start on 16-byte
    boundaries are read where they lie, others are copied into the workspace first; fp32 operands are split into
    three bf16 planes there, which keeps fp32 accuracy on the tensor cores."""
    _check(x, weight, target, bias, label_smoothing, reduction)
    shape = target.shape
    x = x.reshape(-1, x.size(-1))
    target = target.reshape(-1).contiguous()
    bias = None if bias is None else bias.contiguous()
    code = _REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias is not None and bias.requires_grad):
        loss = _LinearCrossEntropy.apply(x, weight, bias, target, ignore_index, float(label_smoothing), code)
    else:
        (xr, ldx), (wr, ldw) = _rows(x), _rows(weight)
        loss = _forward(xr, ldx, wr, ldw, target, bias, ignore_index, float(label_smoothing), code, False)[0]
    return loss.view(shape) if code == 0 else loss
