"""Layer norm of a sum, forward and backward: host side of bpt_layer_norm_forward / bpt_layer_norm_backward.

The reference's blocks end each half with `norm(h + sublayer(h))` (modules/attention.py:79-81, 141, 168-171).
`layer_norm(x, weight, bias, eps, residual=r)` is that as one differentiable call: the forward reads x and r once
and writes y, the backward reads x, r and the gradient of y once, writes the one gradient that x and r share, and
sums the gradients of weight and bias over the rows on the way, in a fixed order (no atomics: results do not vary
from run to run).  Statistics and sums are fp32.
"""
import torch

from . import _lib

MAX_DIM = 8192
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, weight, bias, residual):
    if not x.is_cuda:
        raise RuntimeError("bpt_b200: expected a CUDA tensor (there is no CPU path)")
    if x.dtype not in _DTYPES:
        raise RuntimeError("bpt_b200: layer_norm: unsupported dtype %s" % x.dtype)
    if x.dim() < 1 or not 1 <= x.size(-1) <= MAX_DIM:
        raise RuntimeError("bpt_b200: layer_norm: the last dimension must be in [1, %d]" % MAX_DIM)
    for name, t, shape in (("weight", weight, x.shape[-1:]), ("bias", bias, x.shape[-1:]), ("residual", residual, x.shape)):
        if t is None:
            continue
        if t.device != x.device or t.dtype != x.dtype or t.shape != shape:
            raise RuntimeError("bpt_b200: layer_norm: %s must be a %s tensor of shape %s on %s"
                               % (name, x.dtype, tuple(shape), x.device))


def _forward(x, residual, weight, bias, eps, stats):
    """y and, with stats, the rows' (mean, rstd) as one fp32 tensor (2, rows); contiguous arguments."""
    y = torch.empty_like(x)
    dim = x.size(-1)
    rows = x.numel() // dim
    mean_rstd = torch.empty((2, rows), dtype=torch.float32, device=x.device) if stats else None
    at = None if mean_rstd is None else mean_rstd.data_ptr()
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().bpt_layer_norm_forward(x.data_ptr(), _lib.ptr(residual), _lib.ptr(weight), _lib.ptr(bias),
                                                     eps, y.data_ptr(), at, None if at is None else at + 4 * rows,
                                                     rows, dim, _lib.dtype_code(x.dtype), _lib.stream()))
    return y, mean_rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, mean_rstd = _forward(x, residual, weight, bias, eps, True)
        ctx.save_for_backward(x, residual, weight, mean_rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, residual, weight, mean_rstd = ctx.saved_tensors
        need_x, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        gy = gy.contiguous()
        dim = x.size(-1)
        rows = x.numel() // dim
        da = torch.empty_like(x) if need_x or need_r else None
        dw = torch.empty(dim, dtype=x.dtype, device=x.device) if need_w else None
        db = torch.empty(dim, dtype=x.dtype, device=x.device) if need_b else None
        with torch.cuda.device(x.device):
            nbytes = _lib.lib().bpt_layer_norm_backward_workspace_bytes(rows, dim) if need_w or need_b else 0
            ws = _lib.workspace(nbytes, x.device)
            mean = mean_rstd.data_ptr()
            _lib.check(_lib.lib().bpt_layer_norm_backward(gy.data_ptr(), x.data_ptr(), _lib.ptr(residual), _lib.ptr(weight),
                                                          mean, mean + 4 * rows, _lib.ptr(da), _lib.ptr(dw), _lib.ptr(db),
                                                          rows, dim, _lib.dtype_code(x.dtype), ws.data_ptr(), nbytes,
                                                          _lib.stream()))
        return da if need_x else None, da if need_r else None, dw, db, None


def layer_norm(x, weight, bias, eps=1e-5, residual=None):
    """LayerNorm(x + residual) over the last dimension; differentiable once in x, residual, weight and bias.

    x: (..., dim) CUDA tensor, fp32, bf16 or fp16, dim from 1 to 8192; weight, bias: (dim,) of x's dtype or None (ones,
    zeros); residual: of x's shape and dtype or None.  Any strides (non-contiguous inputs are copied).  The sum
    x + residual is not rounded before it is normalised.  Biased variance, as torch.nn.LayerNorm."""
    _check(x, weight, bias, residual)
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        return _LayerNorm.apply(x, residual, weight, bias, float(eps))
    return _forward(x, residual, weight, bias, float(eps), False)[0]
