"""feed_forward: the gated feed-forward block of a token network, with its gradients.

    y = (act(x gate^T) * (x up^T)) down^T

x is (..., width), gate and up are (hidden, width), down is (out, hidden) and y is (...,
out): float32, bfloat16 or float16, one type for all; act is 'silu', a / (1 + exp(-a)),
or 'gelu', a (1 + erf(a / sqrt(2))) / 2.  One call is two kernels: both projections with
the activation and the product, and the projection down.

Sums are fp32.  Besides y, what lies between two products is rounded to the tensors'
type: act(a) * b, and the gradients of a = x gate^T and b = x up^T, so float16's range (up
to 65504, from 6e-5 at full precision) holds for those too: gradients of y far below 1e-3
want a loss that is scaled up.  a and b themselves may pass that range.  A
call that needs gradients keeps x, the weights, a, b (in the 16-bit types with four more
bits each; what is beyond float16's range to eight bits) and act(a) * b.  The weights'
gradients are added up in a fixed order: equal inputs give equal bits.
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


def _inner(n, hidden, x):
    """Elements and bytes of n rows of a, b or h, as the library lays them: whole pieces of 8."""
    elements = n * (-(-hidden // 8) * 8)
    return elements, -(-elements * x.element_size() // 256) * 256


def _forward(x, gate, up, down, activation, grads):
    """y, what the library is called with, and for a backward h, a, b and their rests, one after the other in bytes."""
    (hidden, width), out = gate.shape, down.shape[0]
    n, device = x.numel() // width, x.device
    rows, apart = _rows(x, width)
    code = _t.DTYPE_CODES[x.dtype]
    sizes = code, activation, n, width, hidden, out
    lib = _t.load()
    y = x.new_empty(x.shape[:-1] + (out,))
    part, (elements, each) = lib.gs_feed_forward_workspace_bytes(code, n, width, hidden, out, 0), _inner(n, hidden, x)
    if grads:
        kept = torch.empty(3 * each + (elements if code else 0), device=device, dtype=torch.uint8)
        ws = _t.workspace(part, device)
        h, wsp = kept.data_ptr(), _t.ptr(ws)
        a, b, rest = _places(h, each, code)
    else:
        kept = torch.empty(part + each, device=device, dtype=torch.uint8)
        wsp = kept.data_ptr()
        a, b, rest, h = None, None, None, wsp + part
    with _t.on_device(device):
        _t.check(lib.gs_feed_forward(*sizes, rows.data_ptr(), apart, gate.data_ptr(), up.data_ptr(), down.data_ptr(), a, b,
                                     rest, h, y.data_ptr(), wsp, _t.stream(device)), "gs_feed_forward")
    return y, sizes, kept


def _places(h, each, code):
    """a, b and, of the 16-bit types, their rests behind h."""
    return h + each, h + 2 * each, h + 3 * each if code else None


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, activation):
        y, ctx.how, kept = _forward(x, gate, up, down, activation, True)
        ctx.save_for_backward(x, gate, up, down, kept)
        return y

    # The autograd engine calls this from a thread of its own, on the forward's
    # device and stream.
    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        # hooks on saved tensors give them back with the same values, not in the same places
        x, *saved = ctx.saved_tensors
        gate, up, down, kept = (t.contiguous() for t in saved)
        code, _, n, width, hidden, out = ctx.how
        device, lib = x.device, _t.load()
        rows, apart = _rows(x, width)
        drows, dapart = _rows(dy, out)
        if kept.data_ptr() % 256:
            kept = kept.clone()
        h = kept.data_ptr()
        a, b, rest = _places(h, _inner(n, hidden, x)[1], code)
        need = ctx.needs_input_grad
        grads = (torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None,
                 torch.empty_like(gate) if need[1] else None, torch.empty_like(up) if need[2] else None,
                 torch.empty_like(down) if need[3] else None)
        ws = _t.workspace(lib.gs_feed_forward_workspace_bytes(code, n, width, hidden, out, 1), device)
        _t.check(lib.gs_feed_forward_backward(
            *ctx.how, rows.data_ptr(), apart, gate.data_ptr(), up.data_ptr(), down.data_ptr(), a, b, rest, h,
            drows.data_ptr(), dapart, *map(_t.ptr, grads), _t.ptr(ws), _t.stream(device)), "gs_feed_forward_backward")
        return *grads, None


def feed_forward(x, gate, up, down, activation="silu"):
    """The gated block of x over its last dimension; differentiable in x and the three weights."""
    _t.not_traced()
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
