"""Plain 64-bit forms of the token operators on the CPU, each with a bound on
the kernels' rounding error that follows from where they round.

u(type) is half the spacing of the type relative to the value; U32 is fp32's.
An fp32 sum of n terms in the kernels is a chain of at most `chain` additions
per lane and a tree over lanes, so its error is at most (chain + 16) U32 times
the sum of the terms' magnitudes."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24
# the smallest step below the normal range, which bounds what underflow loses
STEP = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0.0, f"{what}: {worst:.3g} beyond the bound at {int(over.argmax())} of {over.numel()}"


def layer_norm_64(x, weight, bias, eps, dy, rows_chain):
    """{name: (value, bound)} of y, dx, dweight, dbias."""
    t, p = x.dtype, (weight if weight is not None else bias)
    p = t if p is None else p.dtype
    x, dy = x.detach().double().cpu(), dy.double().cpu()
    n = x.shape[-1]
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    u, g = U[t], 64 * U32          # a lane adds at most 32 elements of a row
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    var = (d * d).mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    z = d * rstd
    e_mean = g * x.abs().mean(-1, keepdim=True)
    e_rstd = g + (e_mean * rstd) ** 2 + 4 * U32          # relative
    e_z = z.abs() * (e_rstd + 4 * U32) + e_mean * rstd
    y = z * w + b
    out = dict(y=(y, u * y.abs() + 1.01 * e_z * w.abs() + 2 * U32 * ((z * w).abs() + b.abs()) + STEP[t]))
    h = dy * w
    mh, mhz = h.mean(-1, keepdim=True), (h * z).mean(-1, keepdim=True)
    dx = rstd * (h - mh - z * mhz)
    e_mh = g * h.abs().mean(-1, keepdim=True)
    e_mhz = g * (h * z).abs().mean(-1, keepdim=True) + (h.abs() * e_z).mean(-1, keepdim=True)
    inner = 4 * U32 * (h.abs() + mh.abs() + (z * mhz).abs()) + e_mh + z.abs() * e_mhz + e_z * (mhz.abs() + e_mhz)
    out["dx"] = (dx, u * dx.abs() + 1.01 * rstd * inner + e_rstd * dx.abs() + STEP[t])
    rows = lambda v: v.reshape(-1, n).sum(0)  # noqa: E731
    gr = (rows_chain + 64) * U32
    dw, db = rows(dy * z), rows(dy)
    out["dweight"] = (dw, U[p] * dw.abs() + 1.01 * (gr * rows((dy * z).abs()) + rows(dy.abs() * e_z)) + STEP[p])
    out["dbias"] = (db, U[p] * db.abs() + gr * rows(dy.abs()) + STEP[p])
    return out


def attention_64(q, k, v, causal, key_lengths, query_start, scale, do=None):
    """{name: (value, bound)} of o and, with do, of dq, dk, dv."""
    t = q.dtype
    u, step = U[t], STEP[t]
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1:3]
    G = Hq // Hkv
    j = torch.arange(Tk)
    lengths = torch.full((B,), Tk) if key_lengths is None else key_lengths.cpu().clamp(0, Tk)
    held = (j[None] < lengths[:, None])[:, None, :, None]
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    start = torch.full((B,), Tk - Tq) if query_start is None else query_start.cpu()
    sees = (j[None, None] < lengths[:, None, None]).expand(B, Tq, Tk)
    if causal:
        sees = sees & (j[None, None] <= torch.arange(Tq)[None, :, None] + start[:, None, None])
    sees = sees[:, None]
    ke, ve = (x.repeat_interleave(G, 1) for x in (k, v))
    kt, vt = ke.transpose(2, 3), ve.transpose(2, 3)
    S = (q @ kt * scale).masked_fill(~sees, -math.inf)
    top = S.amax(-1, keepdim=True) if Tk else S.new_zeros((B, Hq, Tq, 1))
    E = torch.exp(S - top.masked_fill(top == -math.inf, 0.0))
    total = E.sum(-1, keepdim=True)
    P = E / total.masked_fill(total == 0, 1.0)
    # relative error of a probability: its score's (an fp32 dot product, then a
    # multiplication by log2(e) and a subtraction of numbers of its size), the
    # exponential's, and the same again in the sum; a chain of Tk / 64 rescalings
    size = (q.abs() @ kt.abs() * scale).masked_fill(~sees, 0.0)
    most = size.amax(-1, keepdim=True) if Tk else size.new_zeros((B, Hq, Tq, 1))
    e_p = 2 * (U32 * (D + 8) * (size + most) + (Tk / 8 + 32) * U32)
    g = (Tk + 32) * U32
    o = P @ ve
    mass = P @ ve.abs()
    under = step * ve.abs().sum(2, keepdim=True)
    out = dict(o=(o, u * o.abs() + 1.01 * ((u + g) * mass + (P * e_p) @ ve.abs()) + under + step))
    if do is None:
        return out
    do = do.double().cpu()
    fold = lambda x: x.view(B, Hkv, G, Tk, D).sum(2)  # noqa: E731
    g_rows = (G * Tq + 32) * U32
    dv = fold(P.transpose(2, 3) @ do)
    # P as an operand: rounded to the type, and recomputed from the rounded lse
    e_dv = fold(((u + 2 * e_p + g_rows) * P + step).transpose(2, 3) @ do.abs())
    out["dv"] = (dv, u * dv.abs() + 1.01 * e_dv + step)
    dP = do @ vt
    delta = (do * o).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    e_o = u * u * o.abs() + 1.01 * (u * mass + g * mass + (P * e_p) @ ve.abs()) + under + step
    if t == torch.float32:
        e_o = e_o + u * o.abs()
    e_delta = (do.abs() * (e_o + (D + 8) * U32 * o.abs())).sum(-1, keepdim=True)
    e_dp = (D + 8) * U32 * (do.abs() @ vt.abs())
    e_ds = u * dS.abs() + 1.01 * (P * (e_dp + e_delta) + 2 * e_p * dS.abs()) + step
    dq, dk = dS @ ke * scale, fold(dS.transpose(2, 3) @ q) * scale
    out["dq"] = (dq, u * dq.abs() + 1.01 * scale * ((e_ds + g * dS.abs()) @ ke.abs()) + step)
    out["dk"] = (dk, u * dk.abs() + 1.01 * scale * fold((e_ds + g_rows * dS.abs()).transpose(2, 3) @ q.abs()) + step)
    return out


QUINTIC = (3.4445, -4.7750, 2.0315)


def orthogonalise_64(update, steps):
    """The value, and a bound on the Frobenius norm of each matrix's error.

    A step multiplies an error by at most 4.3, the largest slope of the quintic
    (and of its divided differences) on [0, 1.21].  A product of K terms adds
    about sqrt(K) U32 from its fp32 sums and 12 U32 from its operands' 22 bits,
    relative to the factors' norms; three products a step, |B| up to 3.5."""
    a, b, c = QUINTIC
    G = update.detach().double().cpu()
    tall = G.shape[-2] > G.shape[-1]
    X = G.transpose(-1, -2) if tall else G
    X = X / (torch.linalg.matrix_norm(X, keepdim=True) + 1e-7)
    per_step = 3 * 3.5 * (math.sqrt(max(X.shape[-2:])) + 12) * U32
    error = torch.zeros(X.shape[:-2], dtype=torch.float64)
    for _ in range(steps):
        A = X @ X.transpose(-1, -2)
        error = 4.3 * error + per_step * torch.linalg.matrix_norm(X)
        X = a * X + (b * A + c * (A @ A)) @ X
    error = error + U[update.dtype] * torch.linalg.matrix_norm(X) + 1e-30
    return (X.transpose(-1, -2) if tall else X), error
