"""layer_norm: layer normalisation over the last dimension, with its gradients.

    y = weight (x - mean) / sqrt(var + eps) + bias

mean and var (over n, uncorrected) and every sum are fp32 whatever the type of
x; each output is rounded to its type once.  x is float32, bfloat16 or float16;
weight and bias (either may be None) have x's type or float32.  The gradients
of weight and bias are added up in a fixed order, so equal inputs give equal
bits.  A row whose squared deviations pass fp32's range (deviations of 1e18 and
more) has an infinite variance and becomes bias.
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


def _forward(x, weight, bias, eps, grads):
    """y and, for a backward, each row's mean and 1 / deviation and what the backward is called with."""
    width = x.shape[-1]
    rows, n, apart = _rows(x, width)
    params = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    code, param_code = _t.DTYPE_CODES[x.dtype], _t.DTYPE_CODES[params]
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty((2, n), device=x.device, dtype=torch.float32) if grads else None
    mean = stats.data_ptr() if grads else None
    with _t.on_device(x.device):
        _t.check(_t.load().gs_layer_norm_forward(
            code, param_code, n, width, rows.data_ptr(), apart, _t.ptr(weight), _t.ptr(bias), eps, y.data_ptr(), mean,
            mean + 4 * n if grads else None, _t.stream(x.device)), "gs_layer_norm_forward")
    return y, stats, (code, param_code, n, width, params)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats, ctx.how = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.wants = weight is not None and ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]
        code, _, n, width, _ = ctx.how
        ctx.ws_bytes = _t.load().gs_layer_norm_workspace_bytes(code, n, width) if any(ctx.wants) else 0
        return y

    # The autograd engine calls this from a thread of its own, on the forward's
    # device and stream: what does not need the gradient is prepared by forward.
    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        code, param_code, n, width, params = ctx.how
        device = x.device
        # hooks on saved tensors give them back with the same values, not in the same places
        stats = stats.contiguous()
        weight = None if weight is None else weight.contiguous()
        rows, _, apart = _rows(x, width)
        drows, _, dapart = _rows(dy, width)
        dx = torch.empty(x.shape, device=device, dtype=x.dtype)
        dw = torch.empty(width, device=device, dtype=params) if ctx.wants[0] else None
        db = torch.empty(width, device=device, dtype=params) if ctx.wants[1] else None
        ws = _t.workspace(ctx.ws_bytes, device)
        mean = stats.data_ptr()
        _t.check(_t.load().gs_layer_norm_backward(
            code, param_code, n, width, rows.data_ptr(), apart, _t.ptr(weight), mean, mean + 4 * n, drows.data_ptr(),
            dapart, dx.data_ptr(), _t.ptr(dw), _t.ptr(db), _t.ptr(ws), _t.stream(device)), "gs_layer_norm_backward")
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
    weight, bias = (None if p is None else p.contiguous() for p in (weight, bias))
    if _t.wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]
