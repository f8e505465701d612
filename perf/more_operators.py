"""The remaining operators of a token network in front of the rasterizer, as measurable cases.

A block of such a network rotates (and mostly normalises) its queries and keys
before attention and ends in a gated feed-forward; what is no weight matrix takes
AdamW.  Four kinds of work:
  rotate       rotary positions of queries and keys
  norm_rotate  the RMS norm of every head's queries and keys, with the rotation
  feed         the gated feed-forward block: three products, the activation
  adamw        an AdamW step over all tensors of a network, moments in 32 or 8 bits
the first three forward, and with `train` with their gradients.

listed() holds the sizes; draw() takes more from the same ranges."""
import math

import torch

DEV = "cuda"
own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BASE = 10000.0
EPS = 1e-6
# the optimiser's settings
LR, BETAS, ADAM_EPS, DECAY, STEP, SEED = 1e-3, (0.9, 0.999), 1e-8, 0.01, 7, 12345
BLOCK = 128            # elements that share a power of two, in 8 bits

# ------------------------------------------------------------------- the cases


def listed():
    return [
        # the queries and keys of two long sequences whose heads share keys in fours, from a fused projection
        dict(name="rotate_train_2x8192x20x128", kind="rotate", B=2, Hq=16, Hkv=4, T=8192, D=128, axes=1, pairs=64,
             interleaved=False, factor=1.0, far=1, dtype="bfloat16", params="bfloat16", train=True),
        # one new token for each of 64 sequences far into their contexts, half of each head rotated, frequencies scaled
        dict(name="rotate_64x1x40x128", kind="rotate", B=64, Hq=32, Hkv=8, T=1, D=128, axes=1, pairs=32,
             interleaved=True, factor=8.0, far=1 << 20, dtype="float16", params="float16", train=False),
        # the image tokens of a large batch: a row and a column, parameters kept in 32 bits
        dict(name="norm_rotate_train_16x2048x24x64", kind="norm_rotate", B=16, Hq=16, Hkv=8, T=2048, D=64, axes=2,
             pairs=16, interleaved=False, factor=1.0, far=1, dtype="bfloat16", params="float32", train=True),
        # an odd head, an odd number of tokens, all in 32 bits
        dict(name="norm_rotate_train_3x1021x9x75", kind="norm_rotate", B=3, Hq=6, Hkv=3, T=1021, D=75, axes=1,
             pairs=35, interleaved=True, factor=1.0, far=1, dtype="float32", params="float32", train=True),
        # one new token for each of 16 sequences: latency
        dict(name="norm_rotate_16x1x40x128", kind="norm_rotate", B=16, Hq=32, Hkv=8, T=1, D=128, axes=1, pairs=64,
             interleaved=False, factor=1.0, far=32768, dtype="bfloat16", params="bfloat16", train=False),
        # a training step's block over a batch of image tokens
        dict(name="feed_train_8192x1024x4096", kind="feed", rows=8192, width=1024, hidden=4096, out=1024,
             dtype="bfloat16", train=True),
        # the predictor's own block, two scenes of two views, in 32 bits
        dict(name="feed_train_1024x256x512", kind="feed", rows=1024, width=256, hidden=512, out=256,
             dtype="float32", train=True),
        # odd sizes everywhere
        dict(name="feed_train_1337x251x683", kind="feed", rows=1337, width=251, hidden=683, out=251,
             dtype="float16", train=True),
        # one token through a wide block: the weights' bytes
        dict(name="feed_1x2048x8192", kind="feed", rows=1, width=2048, hidden=8192, out=2048, dtype="bfloat16",
             train=False),
        # the parameters of a network of 8 blocks, all in 32 bits
        dict(name="adamw_32_8x1024", kind="adamw", depth=8, width=1024, bits=32, dtype="float32"),
        # weights and gradients in 16 bits, moments in 8
        dict(name="adamw_8_12x1024", kind="adamw", depth=12, width=1024, bits=8, dtype="bfloat16"),
        # a small odd network: latency
        dict(name="adamw_8_3x61", kind="adamw", depth=3, width=61, bits=8, dtype="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _up_to(x, most):
    return max(1, min(x, int(most)))


def draw(rng):
    kind = rng.choice(["rotate", "norm_rotate", "norm_rotate", "feed", "feed", "feed", "adamw", "adamw"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind == "adamw":
        return dict(kind=kind, depth=rng.randint(1, 12), width=_log(rng, 16, 1000), bits=rng.choice([8, 32]),
                    dtype=dtype)
    if kind == "feed":
        width, hidden = _log(rng, 24, 1500), _log(rng, 32, 4000)
        if rng.random() < 0.6:
            width, hidden = width // 8 * 8, hidden // 8 * 8
        train = rng.random() < 0.6
        most = 3e10 / (width * hidden) / (16 if dtype == "float32" else 1)
        rows = _up_to(_log(rng, 1, 8192), most) if train else _up_to(_log(rng, 1, 512), most)
        out = width if rng.random() < 0.8 else _log(rng, 16, 1500)
        return dict(kind=kind, rows=rows, width=width, hidden=hidden, out=out, dtype=dtype, train=train)
    D = rng.choice([24, 33, 48, 64, 64, 75, 80, 96, 128, 128])
    axes = rng.choice([1, 1, 2])
    pairs = max(1, D // 2 // axes // rng.choice([1, 1, 2]))
    Hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5])
    train = rng.random() < 0.6
    T = _log(rng, 1, 8192) if train else rng.choice([1, 1, 1, 2, 7, 600])
    B = _up_to(_log(rng, 1, 64), 4e7 / (Hkv * (group + 1) * T * D))
    return dict(kind=kind, B=B, Hq=Hkv * group, Hkv=Hkv, T=T, D=D, axes=axes, pairs=pairs,
                interleaved=rng.random() < 0.4, factor=rng.choice([1.0, 1.0, 4.0]),
                far=rng.choice([1, 4096, 1 << 20]) if axes == 1 else 1, dtype=dtype,
                params=rng.choice([dtype, "float32"]), train=train)


def _shapes(case):
    """The parameters of a network of gated blocks: matrices, norms, a table of positions."""
    w = case["width"]
    one = [(w,), (w,), (64,), (64,), (w + w // 2, w), (w, w), (4 * w, w), (4 * w, w), (w, 4 * w)]
    return one * case["depth"] + [(257, w), (w,), (w,), (56, w)]


def _layout(case):
    """(first element, elements) of each tensor in one flat buffer, and the buffer's size: tensors begin at whole blocks."""
    at, places = 0, []
    for shape in _shapes(case):
        n = math.prod(shape)
        places.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return places, at


# ------------------------------------------------------------------ the inputs


def _normal(g, shape, dtype, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale + mean).to(dtype)


def _frequencies(case):
    """Radians a position of each pair."""
    return [BASE ** (-i / case["pairs"]) / case["factor"] for i in range(case["pairs"])]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "feed":
        M, W, H, O = (case[k] for k in ("rows", "width", "hidden", "out"))
        s["x"] = _normal(g, (M, W), t)
        s["gate"], s["up"] = (_normal(g, (H, W), t, 1 / math.sqrt(W)) for _ in range(2))
        s["down"] = _normal(g, (O, H), t, 1 / math.sqrt(H))
        if case["train"]:
            s["dy"] = _normal(g, (M, O), t)
            for k in ("x", "gate", "up", "down"):
                s[k].requires_grad_(True)
        return s
    if case["kind"] == "adamw":
        places, size = _layout(case)
        real = torch.zeros(size, device=DEV, dtype=torch.bool)
        for at, n in places:
            real[at:at + n] = True
        flat = {k: torch.where(real, torch.randn(size, generator=g, device=DEV), 0.0) for k in "pgmv"}
        del real
        flat["p"], flat["g"] = (flat["p"] * 0.05).to(t), (flat["g"] * 1e-3).to(t)
        flat["m"] *= 3e-4
        flat["v"] = (flat["v"] * 4e-4).square_()
        if case["bits"] == 8:
            # moments as an earlier step left them, rounded with some random bits
            m, v = flat["m"], flat["v"]
            draw = torch.randint(0, 65536, (2, size), generator=g, device=DEV)
            (flat["m"], sm), (flat["v"], sv) = _pack(m, draw[0], 14), _pack(v, draw[1], 30)
            s["scales"] = torch.stack([sm, sv])
            del m, v, draw
        s.update(flat)
        view = lambda k: [flat[k][at:at + n] for at, n in places]  # noqa: E731
        s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"] = (view(k) for k in "pgmv")
        if case["bits"] == 8:
            s["scale_list"] = [s["scales"][:, at // BLOCK:-(-(at + n) // BLOCK)] for at, n in places]
        return s
    B, Hq, Hkv, T, D, A = (case[k] for k in ("B", "Hq", "Hkv", "T", "D", "axes"))
    # slices of a fused projection: (B, T, H, D) in memory, seen as (B, H, T, D)
    fused = _normal(g, (B, T, Hq + 2 * Hkv, D), t)
    s["q"], s["k"] = fused[:, :, :Hq].transpose(1, 2), fused[:, :, Hq:Hq + Hkv].transpose(1, 2)
    s["frequencies"] = torch.tensor([round(f / (2 * math.pi) * 2.0 ** 64) for f in _frequencies(case)], device=DEV)
    first = torch.randint(0, case["far"], (B, 1), generator=g, device=DEV)
    at = torch.arange(T, device=DEV)
    if A == 1:
        s["positions"] = (first + at).int()
    else:
        # tokens of an image of 37 columns: a row and a column
        s["positions"] = torch.stack([at // 37, at % 37], -1)[None].expand(B, T, 2).int()
        s["frequencies"] = s["frequencies"].expand(A, -1).contiguous()
    if case["kind"] == "norm_rotate":
        p = TYPES[case["params"]]
        s["qw"], s["kw"] = (_normal(g, (D,), p, 0.1, 1.0) for _ in range(2))
    if case["train"]:
        s["dq"], s["dk"] = (_normal(g, (B, T, H, D), t).transpose(1, 2) for H in (Hq, Hkv))
        for k in ("q", "k", "qw", "kw"):
            if k in s:
                s[k].requires_grad_(True)
    return s


# --------------------------------------------------------------------- running


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotate": _own_rotate, "norm_rotate": _own_rotate, "feed": _own_feed, "adamw": _own_adamw}[kind](state)
    with torch.no_grad():
        return {"rotate": _plain_rotate, "norm_rotate": _plain_rotate, "feed": _plain_feed,
                "adamw": _plain_adamw}[kind](state)


def _own_rotate(s):
    from blitzgs_amd.rotary import norm_rotate, rotate
    c = s["case"]
    if c["kind"] == "rotate":
        q, k = rotate(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=c["interleaved"])
        leaves = (s["q"], s["k"])
    else:
        q, k = norm_rotate(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["frequencies"],
                           interleaved=c["interleaved"], eps=EPS)
        leaves = (s["q"], s["k"], s["qw"], s["kw"])
    if not c["train"]:
        return [q, k]
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"]))]


def _own_feed(s):
    from blitzgs_amd.feedforward import feed_forward
    y = feed_forward(s["x"], s["gate"], s["up"], s["down"], activation="silu")
    if not s["case"]["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, (s["x"], s["gate"], s["up"], s["down"]), s["dy"])]


def _own_adamw(s):
    from blitzgs_amd.adamw import adamw_update, moment_values
    adamw_update(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], step=STEP, lr=LR, betas=BETAS, eps=ADAM_EPS,
                 weight_decay=DECAY, scales=s.get("scale_list"), seed=SEED)
    if s["case"]["bits"] == 32:
        return [s["p"], s["m"], s["v"]]
    m, v = moment_values(s["m"], s["v"], s["scales"], dtype=torch.bfloat16)
    return [s["p"], m, v]


# cos and sin of position x frequency, formed modulo a turn of 2^64; (B, 1, T, pairs of all axes)
def _turned(s):
    positions = s["positions"].long()
    if s["case"]["axes"] == 1:
        positions = positions[..., None]
    phase = positions[..., None] * s["frequencies"].view(s["case"]["axes"], -1)
    angle = phase.flatten(2).double() * (2 * math.pi / 2.0 ** 64)
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _rotated(x, cos, sin, interleaved):
    R = 2 * cos.shape[-1]
    y = x.clone()
    one, two = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y[..., one] = x[..., one] * cos - x[..., two] * sin
    y[..., two] = x[..., one] * sin + x[..., two] * cos
    return y


# u = w x / sqrt(mean(x^2) + eps) or x, y = rotated(u); g = dy rotated back, h = g w,
# z = x r, dx = r (h - z mean(h z)), dw = sum over rows g z
def _plain_rotate(s):
    c = s["case"]
    cos, sin = _turned(s)
    norm, t = c["kind"] == "norm_rotate", s["q"].dtype
    out, dx, dw = [], [], []
    # queries, then keys: two calls of the same few operations
    for x, w, dy in ((s["q"], s.get("qw"), s.get("dq")), (s["k"], s.get("kw"), s.get("dk"))):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) if norm else None
        z = x * r if norm else x
        out.append(_rotated(z * w.float() if norm else z, cos, sin, c["interleaved"]).to(t))
        if not c["train"]:
            continue
        g = _rotated(dy.float(), cos, -sin, c["interleaved"])
        if norm:
            dw.append((g * z).sum((0, 1, 2)).to(w.dtype))
            h = g * w.float()
            g = r * (h - z * (h * z).mean(-1, keepdim=True))
        dx.append(g.to(t))
    return out + dx + dw


# a = x G^T, b = x U^T, h = a sigmoid(a) b, y = h D^T; dh = dy D,
# da = dh b act'(a), db = dh act(a), dx = da G + db U, dG = da^T x, dU = db^T x, dD = dy^T h
def _plain_feed(s):
    t = s["x"].dtype
    x, gate, up, down = (s[k].float() for k in ("x", "gate", "up", "down"))
    a, b = x @ gate.t(), x @ up.t()
    sig = 1 / (1 + torch.exp(-a))
    act = a * sig
    h = act * b
    y = (h @ down.t()).to(t)
    if not s["case"]["train"]:
        return y
    dy = s["dy"].float()
    dh = dy @ down
    da, db = dh * b * (sig * (1 + a * (1 - sig))), dh * act
    return [y, (da @ gate + db @ up).to(t), (da.t() @ x).to(t), (db.t() @ x).to(t), (dy.t() @ h).to(t)]


# What decides how a number is rounded: 32 bits for each element from its key and its
# index, of which the first moment takes the lower half and the second the upper.
def _scrambled(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _keys(count, device):
    """Of each tensor of a call, from the seed, the step and the tensor's place."""
    place = torch.arange(count, device=device)
    return _scrambled((place * 0x9E3779B9 + _scrambled((STEP * 0x9E3779B9 + SEED) & 0xFFFFFFFF)) & 0xFFFFFFFF)


def _power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


# Eight bits: numbers of a block over the power of two at or below its largest are of [0, 2);
# `top` is the exponent field of [1, 2), three bits follow it, fields of 0 are subnormal.
# Rounded up where the rest and draw / 2^16 make a whole step.  First moments (top 14) have a
# sign in bit 7, second ones (top 30) have none.
def _pack(x, draw, top):
    size = x.abs().double().view(-1, BLOCK)
    largest = size.amax(1, keepdim=True)
    e = torch.where(largest > 0, torch.clamp(torch.frexp(largest)[1] - 1, min=-127), -127)
    y = (size * _power(-e)).view(-1)
    field = torch.where(y > 0, torch.clamp(torch.frexp(y)[1] - 1 + top, min=1), 1)
    code = torch.floor(y * _power(top - field + 3) + draw / 65536.0).long() + ((field - 1) << 3)
    code = torch.where(torch.logical_and(x < 0, code > 0), code + 128, code) if top == 14 else code
    return code.to(torch.uint8), (e + 127).view(-1).to(torch.uint8)


def _values(codes, scales, top):
    c = codes.int()
    sign = torch.where(c >= 128, -1.0, 1.0) if top == 14 else 1.0
    c = c & 127 if top == 14 else c
    field = c >> 3
    mantissa = torch.where(field > 0, 8 + (c & 7), c & 7)
    e = (scales.int() - 127).repeat_interleave(BLOCK)
    return (mantissa * sign * _power(torch.clamp(field, min=1) - top - 3 + e)).float()


def _plain_adamw(s):
    c = s["case"]
    eight = c["bits"] == 8
    m, v = (_values(s["m"], s["scales"][0], 14), _values(s["v"], s["scales"][1], 30)) if eight else (s["m"], s["v"])
    p, g = s["p"].float(), s["g"].float()
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g * g
    root = torch.sqrt(v / (1 - BETAS[1] ** STEP)) + ADAM_EPS
    s["p"].copy_(p * (1 - LR * DECAY) - LR * (m / (1 - BETAS[0] ** STEP)) / root)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return [s["p"], s["m"], s["v"]]
    first = torch.tensor([at for at, _ in _layout(c)[0]], device=p.device)
    at = torch.arange(p.numel(), device=p.device)
    which = torch.searchsorted(first, at, right=True) - 1
    draw = _scrambled(((at - first[which]) * 0x9E3779B9 + _keys(len(first), p.device)[which]) & 0xFFFFFFFF)
    for k, x, d, top, row in (("m", m, draw & 65535, 14, 0), ("v", v, draw >> 16, 30, 1)):
        codes, scales = _pack(x, d, top)
        s[k].copy_(codes)
        s["scales"][row].copy_(scales)
    # four significant bits and a power of two: whole in 16 bits
    return [s["p"], _values(s["m"], s["scales"][0], 14).bfloat16(), _values(s["v"], s["scales"][1], 30).bfloat16()]


# ------------------------------------------------------------------------ work


def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    e = _size(case["dtype"])
    if case["kind"] == "feed":
        M, W, H, O = (case[k] for k in ("rows", "width", "hidden", "out"))
        weights, rows = (2 * W + O) * H * e, (W + O) * M * e
        # forward three products; backward twice as many; x, dy and the weights in, y and the gradients out
        return dict(bytes=2 * (weights + rows) if case["train"] else weights + rows,
                    flops=2 * M * H * (2 * W + O) * (3 if case["train"] else 1))
    if case["kind"] == "adamw":
        n = sum(n for _, n in _layout(case)[0])
        # p, g and the moments in, p and the moments out, those of 8 bits as the values they stand for too
        moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
        return dict(bytes=n * (3 * e + moments), flops=n * (16 if case["bits"] == 32 else 40))
    n = case["B"] * case["T"] * (case["Hq"] + case["Hkv"]) * case["D"]
    # forward: x in, y out; backward: dy in, dx out, and under a norm x again
    norm = case["kind"] == "norm_rotate"
    times = (5 if norm else 4) if case["train"] else 2
    return dict(bytes=n * e * times + case["B"] * case["T"] * case["axes"] * 4, flops=n * times * (4 if norm else 3))


# ------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    if case["kind"] == "feed" and case["train"] and case["rows"] * case["width"] * case["hidden"] > 4e10:
        return None
    with torch.no_grad():
        s = prepare(case, seed)
        return {"rotate": _exact_rotate, "norm_rotate": _exact_rotate, "feed": _exact_feed,
                "adamw": _exact_adamw}[case["kind"]](s)


def _exact_rotate(s):
    c = s["case"]
    # a pair is a complex number, the rotation a factor exp(i position frequency)
    frequency = torch.tensor(_frequencies(c), device=DEV, dtype=torch.float64)
    angle = torch.outer(s["positions"].reshape(-1).double(), frequency)
    turn = torch.polar(torch.ones_like(angle), angle).view(c["B"], 1, c["T"], -1)
    N = turn.shape[-1]

    def rotated(x, turn):
        R = x[..., :2 * N]
        if c["interleaved"]:
            y = torch.view_as_real(torch.complex(R[..., 0::2], R[..., 1::2]) * turn).flatten(-2)
        else:
            z = torch.complex(R[..., :N].contiguous(), R[..., N:].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
        return torch.cat([y, x[..., 2 * N:]], -1)

    outs, grads, weights = [], [], []
    for x, w, dy in (("q", "qw", "dq"), ("k", "kw", "dk")):
        x = s[x].double()
        if c["kind"] == "norm_rotate":
            w = s[w].double()
            length = torch.sqrt(x.square().sum(-1, keepdim=True) / c["D"] + EPS)
            outs.append(rotated(x / length * w, turn))
        else:
            outs.append(rotated(x, turn))
        if not c["train"]:
            continue
        g = rotated(s[dy].double(), turn.conj())
        if c["kind"] == "norm_rotate":
            weights.append(torch.einsum("bhtd,bhtd->d", g, x / length))
            g = g * w
            g = g / length - x * (torch.linalg.vecdot(g, x)[..., None] / (c["D"] * length ** 3))
        grads.append(g)
    return outs + grads + weights


def _exact_feed(s):
    x, gate, up, down = (s[k].double() for k in ("x", "gate", "up", "down"))
    a, b = torch.nn.functional.linear(x, gate), torch.nn.functional.linear(x, up)
    act = a * torch.sigmoid(a)
    y = torch.nn.functional.linear(act * b, down)
    if not s["case"]["train"]:
        return y
    dy = s["dy"].double()
    dh = dy.mm(down)
    da = dh * b * (torch.sigmoid(a) + act * torch.sigmoid(-a))
    db = dh * act
    return [y, da.mm(gate) + db.mm(up), da.t().mm(x), db.t().mm(x), dy.t().mm(act * b)]


def _exact_adamw(s):
    c = s["case"]
    n = s["p"].numel()

    def decoded(codes, scales, signed):
        # every code's value, looked up
        top = 14 if signed else 30
        table = [((i & 7) + 8 * ((i >> 3) > 0)) * 2.0 ** (max(i >> 3, 1) - top - 3) for i in range(128 if signed else 256)]
        table = torch.tensor(table + [-x for x in table] if signed else table, device=DEV, dtype=torch.float64)
        return table[codes.long()] * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK)

    eight = c["bits"] == 8
    m, v = (decoded(s["m"], s["scales"][0], True), decoded(s["v"], s["scales"][1], False)) if eight \
        else (s["m"].double(), s["v"].double())
    p, g = s["p"].double(), s["g"].double()
    m = torch.lerp(g, m, BETAS[0])
    v = torch.lerp(g.square(), v, BETAS[1])
    p = p - LR * (DECAY * p + m / (1 - BETAS[0] ** STEP) / ((v / (1 - BETAS[1] ** STEP)).sqrt() + ADAM_EPS))
    if not eight:
        return [p, m, v]

    def mix(x):
        for shift, times in ((16, 0x6A09E667), (15, 0xBB67AE85), (16, 1)):
            x = torch.bitwise_xor(x, torch.bitwise_right_shift(x, shift)) * times % 2 ** 32
        return x

    phi = 0x9E3779B9
    start = mix(torch.tensor((STEP * phi + SEED) % 2 ** 32, device=DEV))
    bits = torch.zeros(n, device=DEV, dtype=torch.int64)
    for i, (at, size) in enumerate(_layout(c)[0]):
        key = mix((start + i * phi) % 2 ** 32)
        bits[at:at + size] = mix((torch.arange(size, device=DEV) * phi + key) % 2 ** 32)

    def stored(x, draw, top):
        largest = x.abs().view(-1, BLOCK).amax(1)
        unit = torch.exp2(torch.floor(torch.log2(largest.clamp(min=1e-300)))).repeat_interleave(BLOCK)
        y = x.abs() / unit
        # the step between neighbouring values about y
        step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** (1 - top))))) / 8
        return torch.copysign(torch.floor(y / step + draw / 65536.0) * step * unit, x)

    return [p, stored(m, bits % 65536, 14), stored(v, bits // 65536, 30)]
