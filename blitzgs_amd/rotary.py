"""rotate, norm_rotate: rotary positions of queries and keys, alone or after the RMS
norm of every head, in one pass, with their gradients.

    u = x, or weight x / sqrt(mean(x^2) + eps) over the head's D elements
    y1 = magnitude (u1 cos - u2 sin),  y2 = magnitude (u1 sin + u2 cos)

for N pairs of elements, (i, i + N) or, interleaved, (2 i, 2 i + 1), by the angle
position * frequency of the pair; elements from 2 N on are u.  q is (B, Hq, T, D), k
(B, Hk, T, D) or None, as attention takes them: float32, bfloat16 or float16, one
type for both, D from 1 to 256, any strides with the last dimension contiguous.
Results lie in memory as (B, T, H, D).  Weights have the rows' type or float32.

positions are int32 or int64, (T,) or (B, T).  Tokens of an image or a volume have
several, (T, axes) or (B, T, axes), with frequencies of shape (axes, pairs): each
axis turns pairs of its own.

frequencies are int64, in 2^-64ths of a turn per position: position * frequency is
formed modulo a turn, without error however far the position, and its cosine and sine
in float32.  rotary_frequencies makes the usual ones, also scaled for contexts longer
than those of the training, as_turns makes them from any angles.

Sums are fp32, each output is rounded to its type once.  A row whose squares are not
within fp32's range is normed by those of the row times a power of two.  The weights'
gradients are added up in a fixed order: equal inputs give equal bits.
"""
import ctypes as C
import math

import torch

from . import _tensors as _t

MAX_HEAD_DIM = 256

_Strides = C.c_int64 * 4         # of which the library reads three


def as_turns(radians, device=None):
    """Angles per position (a tensor or sequence of numbers, in radians) as frequencies."""
    if not isinstance(radians, torch.Tensor):
        radians, device = torch.tensor(radians, dtype=torch.float64), "cuda" if device is None else device
    turns = radians.detach().to("cpu", torch.float64) / (2 * math.pi)
    if not bool(torch.isfinite(turns).all()):
        raise RuntimeError("frequencies must be finite")
    # whole turns do not count: what is left, in [-1/2, 1/2), as a 64-bit integer
    turns = turns - torch.floor(turns + 0.5)
    return torch.clamp(turns * 2.0 ** 64, -2.0 ** 63, 2.0 ** 63 - 1024).to(torch.int64).to(
        radians.device if device is None else device)


def rotary_frequencies(pairs, base=10000.0, factor=1.0, trained=None, ramp=(1.0, 32.0), axes=1, device="cuda"):
    """The frequencies base^(-i / pairs) radians per position, i in 0 .. pairs - 1: (pairs,), or (axes, pairs).

    factor > 1 stretches them for contexts that much longer: all of them, or, with
    `trained` (the positions of the training), only the slow ones: a pair that turns fewer
    than ramp[0] times over them is divided by factor, one that turns more than ramp[1]
    times is left as it is, and between the two the share falls linearly."""
    if pairs < 1 or axes < 1:
        raise RuntimeError(f"pairs and axes must be at least 1, got {pairs} and {axes}")
    if not 0.0 < base < math.inf or not 0.0 < factor < math.inf:
        raise RuntimeError(f"base and factor must be positive numbers, got {base} and {factor}")
    radians = torch.tensor([base ** (-i / pairs) for i in range(pairs)], dtype=torch.float64)
    if trained is None:
        radians = radians / factor
    else:
        slow, fast = ramp
        if not trained > 0 or not 0.0 <= slow < fast:
            raise RuntimeError(f"trained must be positive and ramp two rising numbers, got {trained} and {ramp}")
        kept = ((radians * trained / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        radians = radians * (kept + (1.0 - kept) / factor)
    turns = as_turns(radians, device)
    return turns if axes == 1 else turns.expand(axes, pairs).contiguous()


def _rows(t):
    """t with its last dimension contiguous, its address and its strides; None of them for no tensor."""
    if t is None:
        return None, None, None
    strides = t.stride()
    if strides[3] != 1 and t.shape[3] > 1:
        t = t.contiguous()
        strides = t.stride()
    return t, t.data_ptr(), _Strides(*strides)


class _Out:
    """A result's layout: in memory (B, T, H, D)."""

    def __init__(self, like):
        B, H, T, D = like.shape
        self.shape, self.strides = (B, H, T, D), (T * H * D, D, H * D, 1)
        self.steps = _Strides(*self.strides)

    def beside(self, t):
        """A new one of t's type and device."""
        return t.new_empty_strided(self.shape, self.strides)


class _How:
    """What a call passes to the library beside its tensors."""

    def __init__(self, q, k, weight, frequencies, interleaved, magnitude, norm, eps):
        self.q, self.k = _Out(q), None if k is None else _Out(k)
        B, Hq, T, D = self.q.shape
        code = _t.DTYPE_CODES[q.dtype]
        axes, pairs = (1, frequencies.shape[0]) if frequencies.dim() == 1 else frequencies.shape
        self.sizes = code, B, Hq, 0 if k is None else self.k.shape[1], T, D, axes, pairs
        params = _t.DTYPE_CODES[q.dtype if weight is None else weight.dtype]
        self.norm = norm
        self.first = code, params, *self.sizes[1:], interleaved, magnitude, norm, eps

    def angles(self, positions, frequencies):
        strides = positions.stride()
        if frequencies.dim() == 1:
            strides += (0,)
        if len(strides) == 2:
            strides = (0, *strides)
        return (positions.data_ptr(), 1 if positions.dtype is torch.int64 else 0, _Strides(*strides),
                frequencies.data_ptr())


def _forward(q, k, qw, kw, positions, frequencies, how):
    """The results, and the rows as they were read."""
    device = q.device
    q, qp, qs = _rows(q)
    k, kp, ks = _rows(k)
    qy = how.q.beside(q)
    ky, kyp, kys = (None, None, None) if k is None else ((ky := how.k.beside(k)), ky.data_ptr(), how.k.steps)
    with _t.on_device(device):
        _t.check(_t.load().gs_rotary_forward(
            *how.first, qp, qs, kp, ks, _t.ptr(qw), _t.ptr(kw), *how.angles(positions, frequencies), qy.data_ptr(),
            how.q.steps, kyp, kys, _t.stream(device)), "gs_rotary_forward")
    return qy, ky, q, k


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, positions, frequencies, how):
        qy, ky, q, k = _forward(q, k, qw, kw, positions, frequencies, how)
        ctx.how = how
        if not how.norm:
            q = k = None
        ctx.save_for_backward(q, k, qw, kw, positions, frequencies)
        return qy, ky

    # The autograd engine calls this from a thread of its own, on the forward's
    # device and stream.
    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dqy, dky):
        # hooks on saved tensors give them back with the same values, not in the same places
        q, k, qw, kw, positions, frequencies = ctx.saved_tensors
        how, (need_q, need_k, need_qw, need_kw, *_) = ctx.how, ctx.needs_input_grad
        frequencies = frequencies.contiguous()
        device, lib = frequencies.device, _t.load()
        q, qp, qs = _rows(q)
        k, kp, ks = _rows(k)
        dqy, dqyp, dqys = _rows(dqy)
        dky, dkyp, dkys = _rows(dky)
        dq = dk = dqw = dkw = ws = dqp = dkp = dks = qwp = kwp = dqwp = dkwp = None
        if need_q or need_qw:
            dq = how.q.beside(dqy)
            dqp = dq.data_ptr()
        if dky is not None and (need_k or need_kw):
            dk = how.k.beside(dky)
            dkp, dks = dk.data_ptr(), how.k.steps
        if how.norm:
            if qw is not None:
                qw = qw.contiguous()
                qwp = qw.data_ptr()
            if kw is not None:
                kw = kw.contiguous()
                kwp = kw.data_ptr()
            if need_qw:
                dqw = torch.empty_like(qw)
                dqwp = dqw.data_ptr()
            if need_kw and dk is not None:
                dkw = torch.empty_like(kw)
                dkwp = dkw.data_ptr()
            if need_qw or need_kw:
                ws = _t.workspace(lib.gs_rotary_workspace_bytes(*how.sizes), device)
        _t.check(lib.gs_rotary_backward(
            *how.first, qp, qs, kp, ks, qwp, kwp, *how.angles(positions, frequencies), dqyp, dqys, dkyp, dkys,
            dqp, how.q.steps, dkp, dks, dqwp, dkwp, _t.ptr(ws), _t.stream(device)), "gs_rotary_backward")
        return dq if need_q else None, dk if need_k else None, dqw, dkw, None, None, None


def _call(q, k, qw, kw, positions, frequencies, interleaved, magnitude, norm, eps):
    _t.not_traced()
    _t.require_tensor(q, "q")
    if q.dim() != 4 or not 1 <= q.shape[3] <= MAX_HEAD_DIM:
        raise RuntimeError(f"q must have dimensions (B, H, T, D) with D of 1 to {MAX_HEAD_DIM}, got shape "
                           f"{tuple(q.shape)}")
    B, H, T, D = q.shape
    if k is not None:
        _t.require_tensor(k, "k", device=q.device)
        if k.dim() != 4 or k.dtype != q.dtype or (k.shape[0], k.shape[2], k.shape[3]) != (B, T, D):
            raise RuntimeError("k must have q's type, batch, tokens and head dimension; got q "
                               f"{tuple(q.shape)} {q.dtype}, k {tuple(k.shape)} {k.dtype}")
    if (B | H | T | (0 if k is None else k.shape[1])) >= 1 << 31:
        raise RuntimeError(f"q and k must have sizes below 2^31, got {tuple(q.shape)}")
    if (not isinstance(frequencies, torch.Tensor) or frequencies.dtype != torch.int64 or frequencies.device != q.device
            or frequencies.dim() not in (1, 2) or frequencies.numel() == 0 or 2 * frequencies.numel() > D):
        raise RuntimeError(f"frequencies must be an int64 tensor of shape (pairs,) or (axes, pairs) on {q.device}, of at "
                           f"most D / 2 = {D // 2} pairs in all")
    ends = ((T,), (B, T)) if frequencies.dim() == 1 else ((T, frequencies.shape[0]), (B, T, frequencies.shape[0]))
    if (not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64)
            or positions.device != q.device or tuple(positions.shape) not in ends):
        raise RuntimeError(f"positions must be an int32 or int64 tensor of shape {ends[0]} or {ends[1]} on {q.device}")
    if not abs(magnitude) <= 3e38:
        raise RuntimeError(f"magnitude must be a number of at most 3e38, got {magnitude}")
    if not 0.0 <= eps < math.inf:
        raise RuntimeError(f"eps must be a finite number of at least 0, got {eps}")
    for name, w in (("q_weight", qw), ("k_weight", kw)):
        if w is None:
            continue
        _t.require_tensor(w, name, device=q.device)
        if w.shape != (D,) or w.dtype not in (q.dtype, torch.float32):
            raise RuntimeError(f"{name} must have shape ({D},) and be {q.dtype} or torch.float32, got "
                               f"{tuple(w.shape)} {w.dtype}")
    if qw is not None and kw is not None and qw.dtype != kw.dtype:
        raise RuntimeError(f"q_weight and k_weight must have one type, got {qw.dtype} and {kw.dtype}")
    if kw is not None and k is None:
        raise RuntimeError("k_weight needs k")
    qw, kw = (None if w is None else w.contiguous() for w in (qw, kw))
    frequencies = frequencies.contiguous()
    how = _How(q, k, kw if qw is None else qw, frequencies, int(bool(interleaved)), float(magnitude), norm, float(eps))
    if _t.wants_grad(q, k, qw, kw):
        return _Rotary.apply(q, k, qw, kw, positions, frequencies, how)
    return _forward(q, k, qw, kw, positions, frequencies, how)[:2]


def rotate(q, k, positions, frequencies, interleaved=False, magnitude=1.0):
    """q and k (or None) rotated to their positions; differentiable in both.  Returns the two."""
    return _call(q, k, None, None, positions, frequencies, interleaved, magnitude, 0, 0.0)


def norm_rotate(q, k, q_weight, k_weight, positions, frequencies, interleaved=False, magnitude=1.0, eps=1e-6):
    """The same of each head's rows over their root mean square, times weights (D,) or None; differentiable in q, k
    and the weights."""
    return _call(q, k, q_weight, k_weight, positions, frequencies, interleaved, magnitude, 1, eps)
