"""Plain 64-bit forms of rotate, norm_rotate, feed_forward and adamw_update on the CPU,
each with a bound on the kernels' rounding error that follows from where they round
(u, U32 and STEP as in token_helpers).  Bounds multiply magnitudes along the way to an
output by the errors that its factors can have; 1.05 covers the products of two errors."""
import math

import torch

from token_helpers import STEP, U, U32


def angles_64(positions, frequencies, B, T):
    """cos and sin (B, 1, T, N): the phase is an integer product modulo 2^64."""
    axes = 1 if frequencies.dim() == 1 else frequencies.shape[0]
    p = positions.cpu().long()
    p = p[..., None] if frequencies.dim() == 1 else p
    p = p.expand(B, T, axes)
    phase = (p[..., None] * frequencies.cpu().view(axes, -1)).flatten(2)
    angle = phase.double() * (2 * math.pi / 2.0 ** 64)
    return torch.cos(angle)[:, None], torch.sin(angle)[:, None]


def _pairs(x, N, interleaved):
    if interleaved:
        return x[..., 0:2 * N:2], x[..., 1:2 * N:2]
    return x[..., :N], x[..., N:2 * N]


def _joined(one, two, rest, interleaved):
    both = torch.stack([one, two], -1).flatten(-2) if interleaved else torch.cat([one, two], -1)
    return torch.cat([both, rest], -1)


def _turned(u, e_u, cos, sin, interleaved, magnitude):
    """u rotated, and the error that u's error e_u and the rotation leave: cosine and sine are within 8 U32
    (the angle's three roundings, the series, the magnitude), two products and their sum."""
    N = cos.shape[-1]
    rest, e_rest = u[..., 2 * N:], e_u[..., 2 * N:]
    a, b = _pairs(u, N, interleaved)
    ea, eb = _pairs(e_u, N, interleaved)
    m = abs(magnitude)
    y = _joined(magnitude * (a * cos - b * sin), magnitude * (a * sin + b * cos), rest, interleaved)
    own = 8 * U32 * m * (a.abs() + b.abs())
    one = m * (ea * cos.abs() + eb * sin.abs()) + 2 * U32 * m * ((a * cos).abs() + (b * sin).abs()) + own
    two = m * (ea * sin.abs() + eb * cos.abs()) + 2 * U32 * m * ((a * sin).abs() + (b * cos).abs()) + own
    return y, _joined(one, two, e_rest, interleaved)


def rotary_64(x, w, dy, positions, frequencies, interleaved, magnitude, norm, eps):
    """{name: (value, bound)} of y and, with dy, of dx and dw."""
    t = x.dtype
    u, step = U[t], STEP[t]
    x = x.detach().double().cpu()
    B, _, T, D = x.shape
    cos, sin = angles_64(positions, frequencies, B, T)
    wd = torch.ones(D, dtype=torch.float64) if w is None else w.detach().double().cpu()
    zero = torch.zeros_like(x)
    # a row's sum of squares: at most 32 in a lane and six exchanges
    e_r = 32 * U32
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt() if norm else torch.ones_like(x[..., :1])
    z = x * r
    e_z = z.abs() * (e_r + U32) if norm else zero
    v = z * wd if norm else x
    e_v = z.abs() * wd.abs() * (e_r + 2 * U32) if norm else zero
    y, e_y = _turned(v, e_v, cos, sin, interleaved, magnitude)
    out = dict(y=(y, u * y.abs() + 1.05 * e_y + step))
    if dy is None:
        return out
    dy = dy.double().cpu()
    g, e_g = _turned(dy, zero, cos, -sin, interleaved, magnitude)
    if not norm:
        out["dx"] = (g, u * g.abs() + 1.05 * e_g + step)
        return out
    h = g * wd
    e_h = e_g * wd.abs() + U32 * h.abs()
    mean = (h * z).mean(-1, keepdim=True)
    e_mean = (40 * U32 * (h * z).abs() + e_h * z.abs() + h.abs() * e_z).mean(-1, keepdim=True)
    dx = r * (h - z * mean)
    inner = e_h + z.abs() * e_mean + e_z * mean.abs() + 2 * U32 * (h.abs() + (z * mean).abs())
    out["dx"] = (dx, u * dx.abs() + 1.05 * (r * inner + e_r * dx.abs()) + step)
    rows = lambda q: q.reshape(-1, D).sum(0)  # noqa: E731
    dw = rows(g.transpose(1, 2) * z.transpose(1, 2))
    p = t if w is None else w.dtype
    chain = x.numel() // D + 64
    e_dw = rows(e_g * z.abs() + g.abs() * e_z) + chain * U32 * rows((g * z).abs())
    out["dw"] = (dw, U[p] * dw.abs() + 1.05 * e_dw + STEP[p])
    return out


def activation_64(name, a):
    """The activation, its slope, and the largest absolute slope and second derivative there can be."""
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s)), 1.1, 0.5
    phi = 0.5 * torch.erfc(-a / math.sqrt(2))
    return a * phi, phi + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi), 1.13, 0.8


def feed_forward_64(x, gate, up, down, activation, dy=None):
    """{name: (value, bound)} of y and, with dy, of the four gradients.  x (M, W)."""
    t = x.dtype
    u, step = U[t], STEP[t]
    x, gate, up, down = (v.detach().double().cpu() for v in (x, gate, up, down))
    (M, W), H, O = x.shape, gate.shape[0], down.shape[0]
    s = lambda n: (n + 16) * U32  # noqa: E731     a sum of n products
    a, b = x @ gate.T, x @ up.T
    e_a, e_b = s(W) * (x.abs() @ gate.T.abs()), s(W) * (x.abs() @ up.T.abs())
    act, slope, most, bend = activation_64(activation, a)

    def hidden(e_a, e_b):
        e_act = most * e_a + 8 * U32 * act.abs() + 2 * U32 * a.abs() * (slope.abs() + U32)
        return e_act, 1.05 * (e_act * b.abs() + act.abs() * e_b)

    h = act * b
    e_h = hidden(e_a, e_b)[1] + u * h.abs() + step
    y = h @ down.T
    out = dict(y=(y, u * y.abs() + 1.05 * ((e_h + s(H) * h.abs()) @ down.T.abs()) + step))
    if dy is None:
        return out
    dy = dy.double().cpu()
    # the backward's a and b are rounded, to a sixteenth of the last bit
    near_u = u if t == torch.float32 else u / 8          # a half of the last bit is held as 7 sixteenths
    e_a, e_b = e_a + near_u * a.abs() + step, e_b + near_u * b.abs() + step
    e_act, _ = hidden(e_a, e_b)
    dh = dy @ down
    e_dh = s(O) * (dy.abs() @ down.abs())
    e_slope = bend * e_a + 16 * U32
    da, db = dh * b * slope, dh * act
    e_da = 1.05 * (e_dh * (b * slope).abs() + (dh * slope).abs() * e_b + (dh * b).abs() * e_slope) + u * da.abs() + step
    e_db = 1.05 * (e_dh * act.abs() + dh.abs() * e_act) + u * db.abs() + step
    dx = da @ gate + db @ up
    e_dx = (e_da + s(2 * H) * da.abs()) @ gate.abs() + (e_db + s(2 * H) * db.abs()) @ up.abs()
    out["dx"] = (dx, u * dx.abs() + 1.05 * e_dx + step)
    for name, d, e in (("dgate", da, e_da), ("dup", db, e_db)):
        v = d.T @ x
        out[name] = (v, u * v.abs() + 1.05 * ((e + s(M) * d.abs()).T @ x.abs()) + step)
    v = dy.T @ h
    out["ddown"] = (v, u * v.abs() + 1.05 * (dy.abs().T @ (e_h + s(M) * h.abs())) + step)
    return out


def near(got, want, t, depth, what):
    """The error's length against the result's: up to four independent roundings on the way, each of a length of
    at most u / sqrt(3) of what it rounds, make 1.2 u; 2 u allows for what they round being longer than the result by
    cancellation; fp32 sums of `depth` terms add up to 4 sqrt(depth) U32."""
    got, want = got.detach().double().cpu(), want.double()
    if want.numel() and want.norm() > 0:
        rel = ((got - want).norm() / want.norm()).item()
        assert rel <= 2 * U[t] + 4 * math.sqrt(depth + 16) * U32, f"{what}: off by {rel:.3g}"


PHI = 0x9E3779B9


def scrambled(x):
    """The hash of 32 bits (int64 tensor or int)."""
    x = x ^ (x >> 16)
    x = x * 0x6A09E667 & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = x * 0xBB67AE85 & 0xFFFFFFFF
    return x ^ (x >> 16)


def draws(n, place, step, seed):
    """32 bits for each of n elements of the tensor at a place in a call."""
    key = scrambled((place * PHI + scrambled((step * PHI + seed) & 0xFFFFFFFF)) & 0xFFFFFFFF)
    return scrambled((torch.arange(n) * PHI + key) & 0xFFFFFFFF)


def values_8(codes, scales, top):
    """What 8-bit moments stand for, float64; codes (n,), scales (ceil(n / 128),)."""
    c, e = codes.cpu().long(), scales.cpu().double().repeat_interleave(128)[:codes.numel()] - 127
    size = c & 127 if top == 14 else c
    field, m = size >> 3, size & 7
    v = torch.where(field > 0, m + 8, m).double() * torch.exp2(torch.clamp(field, min=1) - top - 3 + e)
    v = torch.where(size == (127 if top == 14 else 255), math.nan, v)
    return torch.where(c >= 128, -v, v) if top == 14 else v


def codes_8(x, draw, top, error):
    """The lowest and highest code that x (float64, within `error` of the kernel's) may have, and the scales."""
    n = x.numel()
    pad = -n % 128
    size = torch.nn.functional.pad(x.abs(), (0, pad)).view(-1, 128)
    largest = size.amax(1)
    e = torch.where(largest > 0, torch.clamp(torch.frexp(largest)[1] - 1, min=-127), -127)
    unit = torch.exp2(e.double()).repeat_interleave(128)[:n]

    def code(v):
        y = v.clamp(min=0) / unit
        field = torch.where(y > 0, torch.clamp(torch.frexp(y)[1] - 1 + top, min=1), 1)
        return (torch.floor(y * torch.exp2((top - field + 3).double()) + draw / 65536.0) + (field - 1) * 8).long()

    # a subnormal code's rest is rounded to 2^-20 of a step before it is looked at
    slack = error + unit * 2.0 ** (1 - top - 3 - 20)
    return code(x.abs() - slack), code(x.abs() + slack), (e + 127)


def adamw_64(p, g, m, v, step, lr, betas, eps, decay):
    """(value, bound) of p, m, v after the step; m and v float64 as they are before."""
    t = p.dtype
    b1, b2 = betas
    p, g = p.detach().double().cpu(), g.double().cpu()
    m1 = b1 * m + (1 - b1) * g
    e_m = 4 * U32 * ((b1 * m).abs() + ((1 - b1) * g).abs()) + STEP[torch.float32]
    v1 = b2 * v + (1 - b2) * g * g
    e_v = 5 * U32 * v1 + 2 * STEP[torch.float32]
    root = torch.sqrt(v1 / (1 - b2 ** step))
    den = root + eps
    rate = lr / (1 - b1 ** step)
    new = p * (1 - lr * decay) - rate * m1 / den
    e = rate * e_m / den + (rate * m1 / den).abs() * (10 * U32 + e_v / (2 * v1).clamp(min=1e-300)) + 3 * U32 * p.abs()
    return (new, U[t] * new.abs() + 1.05 * e + STEP[t]), (m1, e_m), (v1, e_v)
