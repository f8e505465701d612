"""layer_norm: layer normalisation over the last dimension, with its gradients.

    y = weight (x - mean) / sqrt(var + eps) + bias

mean and var (over n, uncorrected) and every sum are fp32 whatever the type of
x; each output is rounded to its type once.  x is float32, bfloat16 or float16;
weight and bias (either may be None) have x's type or float32.  The gradients
of weight and bias are added up in a fixed order, so equal inputs give equal
bits.
"""
import torch

from . import _lib

MAX_WIDTH = 32768


def _rows(t):
    """t as (rows, width) with contiguous rows; a copy only where no such view exists."""
    t = t.reshape(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    elif t.shape[0] > 1 and 0 < t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _forward(x, weight, bias, eps, grads):
    """y and, for a backward, (the parameters' type, mean, rstd)."""
    rows = _rows(x)
    n, width = rows.shape
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    params = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    mean, rstd = torch.empty((2, n), device=x.device, dtype=torch.float32) if grads else (None, None)
    with _lib.on_device(x.device):
        _lib.check(_lib.load().gs_layer_norm_forward(
            _lib.dtype_code(x.dtype), _lib.dtype_code(params), n, width, _lib.ptr(rows), _row_stride(rows),
            _lib.ptr(w), _lib.ptr(b), eps, _lib.ptr(y), _lib.ptr(mean), _lib.ptr(rstd), _lib.stream_of(x.device)),
            "gs_layer_norm_forward")
    return y, (params, mean, rstd)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, (ctx.params, mean, rstd) = _forward(x.detach(), weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.columns = weight is not None and ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        rows, drows = _rows(x.detach()), _rows(dy)
        n, width = rows.shape
        w = None if weight is None else weight.detach().contiguous()
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        dw, db = (torch.empty(width, device=x.device, dtype=ctx.params) if c else None for c in ctx.columns)
        lib, code = _lib.load(), _lib.dtype_code(x.dtype)
        ws = _lib.workspace(lib.gs_layer_norm_workspace_bytes(code, n, width), x.device) if any(ctx.columns) else None
        with _lib.on_device(x.device):
            _lib.check(lib.gs_layer_norm_backward(
                code, _lib.dtype_code(ctx.params), n, width, _lib.ptr(rows), _row_stride(rows), _lib.ptr(w),
                _lib.ptr(mean), _lib.ptr(rstd), _lib.ptr(drows), _row_stride(drows), _lib.ptr(dx), _lib.ptr(dw),
                _lib.ptr(db), _lib.ptr(ws), _lib.stream_of(x.device)), "gs_layer_norm_backward")
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Normalise x over its last dimension; differentiable in x, weight and bias."""
    _lib.require_tensor(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise RuntimeError(f"x must have a last dimension of 1 to {MAX_WIDTH}, got shape {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _lib.require_tensor(p, name, device=x.device)
        if p.shape != x.shape[-1:]:
            raise RuntimeError(f"{name} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"{name} must be {x.dtype} or torch.float32, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not 0.0 <= eps < float("inf"):
        raise RuntimeError(f"eps must be a finite number of at least 0, got {eps}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]
