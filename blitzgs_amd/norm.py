"""layer_norm: layer normalisation over the last dimension, with its gradients.

    y = weight (x - mean) / sqrt(var + eps) + bias

mean and var (over n, uncorrected) and every sum are fp32 whatever the type of
x; each output is rounded to its type once.  x is float32, bfloat16 or float16;
weight and bias (either may be None) have x's type or float32.  The gradients
of weight and bias are added up in a fixed order, so equal inputs give equal
bits.
"""
import torch

from . import _tensors as _t

MAX_WIDTH = 32768


def _rows(t, width):
    """t as contiguous rows, and their number and stride; a copy only where no such view exists."""
    if t.is_contiguous():
        return t, t.numel() // width, width
    t = t.reshape(-1, width)
    n, (apart, step) = t.shape[0], t.stride()
    if (width > 1 and step != 1) or (n > 1 and 0 < apart < width):
        t = t.contiguous()
        apart = width
    return t, n, apart if n > 1 else width


def _stats(stats, n):
    if stats is None:
        return None, None
    return stats.data_ptr(), stats.data_ptr() + 4 * n


def _forward(x, weight, bias, eps, grads):
    """y and, for a backward, the parameters' type and each row's mean and 1 / deviation."""
    width = x.shape[-1]
    rows, n, apart = _rows(x, width)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    params = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty((2, n), device=x.device, dtype=torch.float32) if grads else None
    mean, rstd = _stats(stats, n)
    with _t.on_device(x.device):
        _t.check(_t.load().gs_layer_norm_forward(
            _t.DTYPE_CODES[x.dtype], _t.DTYPE_CODES[params], n, width, _t.ptr(rows), apart,
            _t.ptr(w), _t.ptr(b), eps, _t.ptr(y), mean, rstd, _t.stream(x.device)),
            "gs_layer_norm_forward")
    return y, params, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, ctx.params, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.columns = weight is not None and ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        width = x.shape[-1]
        rows, n, apart = _rows(x, width)
        drows, _, dapart = _rows(dy, width)
        mean, rstd = _stats(stats, n)
        w = None if weight is None else weight.contiguous()
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        dw, db = (torch.empty(width, device=x.device, dtype=ctx.params) if c else None for c in ctx.columns)
        lib, code = _t.load(), _t.DTYPE_CODES[x.dtype]
        ws = _t.workspace(lib.gs_layer_norm_workspace_bytes(code, n, width), x.device) if any(ctx.columns) else None
        with _t.on_device(x.device):
            _t.check(lib.gs_layer_norm_backward(
                code, _t.DTYPE_CODES[ctx.params], n, width, _t.ptr(rows), apart, _t.ptr(w),
                mean, rstd, _t.ptr(drows), dapart, _t.ptr(dx), _t.ptr(dw), _t.ptr(db),
                _t.ptr(ws), _t.stream(x.device)), "gs_layer_norm_backward")
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Normalise x over its last dimension; differentiable in x, weight and bias."""
    _t.require_tensor(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise RuntimeError(f"x must have a last dimension of 1 to {MAX_WIDTH}, got shape {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _t.require_tensor(p, name, device=x.device)
        if p.shape != x.shape[-1:]:
            raise RuntimeError(f"{name} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"{name} must be {x.dtype} or torch.float32, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not 0.0 <= eps < float("inf"):
        raise RuntimeError(f"eps must be a finite number of at least 0, got {eps}")
    if _t.wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]
