"""feed_forward: the gated feed-forward block of a token network, with its gradients.

    y = (act(x gate^T) * (x up^T)) down^T

x is (..., width), gate and up are (hidden, width), down is (out, hidden) and y is (...,
out): float32, bfloat16 or float16, one type for all; act is 'silu', a / (1 + exp(-a)),
or 'gelu', a (1 + erf(a / sqrt(2))) / 2.  One call is two kernels: both projections with
the activation and the product, and the projection down.

Sums are fp32.  Besides y, what lies between two products is rounded to the tensors'
type: act(a) * b, and the gradients of a = x gate^T and b = x up^T, so float16's range (up
to 65504, from 6e-5 at full precision) holds for those too, and for a and b.  A call that
needs gradients keeps x, the weights, a, b (in the 16-bit types with four more bits each)
and act(a) * b.  The weights' gradients are added up in a
fixed order: equal inputs give equal bits.
"""
import torch

from . import _tensors as _t

MAX_SIDE = 1 << 24
ACTIVATIONS = {"silu": 0, "gelu": 1}


def _rows(t, width):
    """t as contiguous rows at least `width` apart, and their stride; a copy only where no such view exists."""
    if t.is_contiguous():
        return t, width
    t = t.reshape(-1, width)
    n, (apart, step) = t.shape[0], t.stride()
    if (width > 1 and step != 1) or (n > 1 and apart < width):
        t = t.contiguous()
        apart = width
    return t, apart if n > 1 else width


def _forward(x, gate, up, down, activation, grads):
    """y and, for a backward, a, b, their rests, h and what it is called with."""
    (hidden, width), out = gate.shape, down.shape[0]
    n = x.numel() // width
    rows, apart = _rows(x, width)
    sizes = _t.DTYPE_CODES[x.dtype], activation, n, width, hidden, out
    lib, new = _t.load(), lambda *shape: torch.empty(shape, device=x.device, dtype=x.dtype)
    y, h = new(*x.shape[:-1], out), new(n, hidden)
    a, b = (new(n, hidden), new(n, hidden)) if grads else (None, None)
    rest = torch.empty((n, hidden), device=x.device, dtype=torch.uint8) if grads and x.dtype != torch.float32 else None
    ws = _t.workspace(lib.gs_feed_forward_workspace_bytes(sizes[0], *sizes[2:], 0), x.device)
    with _t.on_device(x.device):
        _t.check(lib.gs_feed_forward(*sizes, rows.data_ptr(), apart, gate.data_ptr(), up.data_ptr(), down.data_ptr(),
                                     _t.ptr(a), _t.ptr(b), _t.ptr(rest), h.data_ptr(), y.data_ptr(), _t.ptr(ws),
                                     _t.stream(x.device)), "gs_feed_forward")
    return y, a, b, rest, h, sizes


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, activation):
        y, a, b, rest, h, ctx.how = _forward(x.detach(), gate, up, down, activation, True)
        ctx.save_for_backward(x, gate, up, down, a, b, rest, h)
        ctx.ws_bytes = _t.load().gs_feed_forward_workspace_bytes(ctx.how[0], *ctx.how[2:], 1)
        return y

    # The autograd engine calls this from a thread of its own, on the forward's
    # device and stream.
    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        # hooks on saved tensors give them back with the same values, not in the same places
        x, *saved = ctx.saved_tensors
        gate, up, down, a, b, rest, h = (t if t is None else t.contiguous() for t in saved)
        _, _, n, width, hidden, out = ctx.how
        rows, apart = _rows(x, width)
        drows, dapart = _rows(dy, out)
        new = lambda i, like: (torch.empty(like.shape, device=x.device, dtype=x.dtype)  # noqa: E731
                               if ctx.needs_input_grad[i] else None)
        dx, dgate, dup, ddown = new(0, x), new(1, gate), new(2, up), new(3, down)
        ws = _t.workspace(ctx.ws_bytes, x.device)
        _t.check(_t.load().gs_feed_forward_backward(
            *ctx.how, rows.data_ptr(), apart, gate.data_ptr(), up.data_ptr(), down.data_ptr(), a.data_ptr(), b.data_ptr(),
            _t.ptr(rest), h.data_ptr(), drows.data_ptr(), dapart, _t.ptr(dx), _t.ptr(dgate), _t.ptr(dup), _t.ptr(ddown), _t.ptr(ws),
            _t.stream(x.device)), "gs_feed_forward_backward")
        return dx, dgate, dup, ddown, None


def feed_forward(x, gate, up, down, activation="silu"):
    """The gated block of x over its last dimension; differentiable in x and the three weights."""
    _t.require_tensor(x, "x")
    for name, w in (("gate", gate), ("up", up), ("down", down)):
        _t.require_tensor(w, name, device=x.device)
        if w.dim() != 2 or w.dtype != x.dtype or not 1 <= min(w.shape) or max(w.shape) > MAX_SIDE:
            raise RuntimeError(f"{name} must be a matrix of x's type {x.dtype} with sides of 1 to {MAX_SIDE}, got "
                               f"{tuple(w.shape)} {w.dtype}")
    if x.dim() < 1 or gate.shape != up.shape or gate.shape[1] != x.shape[-1] or down.shape[1] != gate.shape[0]:
        raise RuntimeError("gate and up must be (hidden, width) and down (out, hidden) for x (..., width), got x "
                           f"{tuple(x.shape)}, gate {tuple(gate.shape)}, up {tuple(up.shape)}, down {tuple(down.shape)}")
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    gate, up, down = (w.contiguous() for w in (gate, up, down))
    if _t.wants_grad(x, gate, up, down):
        return _FeedForward.apply(x, gate, up, down, ACTIVATIONS[activation])
    return _forward(x, gate, up, down, ACTIVATIONS[activation], False)[0]
