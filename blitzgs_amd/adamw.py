"""adamw_update, AdamW: an AdamW step over many tensors at once, with moments in 32
bits or in 8.

    m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
    p = (1 - lr weight_decay) p - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)

Parameters and gradients are float32, bfloat16 or float16, of one type; all arithmetic
is fp32 and a parameter is rounded to its type once.  SparseGaussianAdam updates the
per-Gaussian tensors of a scene, OrthogonalMomentum the weight matrices of a network in
front of it, AdamW what is left of the network, or all of it.

Moments in 8 bits are uint8 tensors of the parameter's shape and one of scales, (2,
ceil(n / 128)): 128 elements in a row share a power of two, over which a first moment
is a small float of a sign, four bits of exponent and three of mantissa, a second one
of five and three.  They are rounded up with the probability of the rest, by bits that
follow from seed, step, the tensor's place in the call and the element's: equal inputs
give equal bits.  A step uses the moments before they are rounded.  A moment that is
infinite or NaN is NaN in 8 bits.  A second moment that is not zero is not rounded to
zero: an element whose gradients are below 2^-16 of the largest of its 128 moves as if
they were measured by that, which is on average less than with 32 bits.
"""
import ctypes as C
import math
import operator
from array import array

import torch

from . import _tensors as _t
from ._lib import AdamWSettings

BLOCK = 128


def new_moments(param, bits=32):
    """(exp_avg, exp_avg_sq, scales) of a parameter at the start; scales is None with 32 bits."""
    if bits not in (8, 32):
        raise RuntimeError(f"moments have 8 or 32 bits, got {bits!r}")
    zeros = lambda *shape, dtype: torch.zeros(shape, device=param.device, dtype=dtype)  # noqa: E731
    if bits == 32:
        return zeros(*param.shape, dtype=torch.float32), zeros(*param.shape, dtype=torch.float32), None
    return (zeros(*param.shape, dtype=torch.uint8), zeros(*param.shape, dtype=torch.uint8),
            zeros(2, -(-param.numel() // BLOCK), dtype=torch.uint8))


# over whole lists, without a line of Python for each tensor: a call over many is bound by these
_SHAPE, _DTYPE = operator.attrgetter("shape"), operator.attrgetter("dtype")
_CONTIGUOUS, _DEVICE, _NUMEL = torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.numel
_ADDRESS, _STRIDE = torch.Tensor.data_ptr, torch.Tensor.stride


def _are(ts, dtype, device, shapes=None):
    """Whether ts are tensors of a type, on a device and of these shapes."""
    try:
        return (set(map(_DTYPE, ts)) == {dtype} and set(map(_DEVICE, ts)) == {device.index}
                and (shapes is None or list(map(_SHAPE, ts)) == shapes))
    except (AttributeError, TypeError):        # no tensor
        return False


def _contiguous(ts):
    """Whether all are; what is no dense tensor is not."""
    try:
        return all(map(_CONTIGUOUS, ts))
    except (TypeError, RuntimeError):
        return False


def _checked(ts, name, dtype, device, shapes):
    """Contiguous tensors of a type and of the parameters' shapes."""
    if len(ts) != len(shapes):
        raise RuntimeError(f"{name} must hold a tensor for each of {len(shapes)} parameters, got {len(ts)}")
    if not (_are(ts, dtype, device, shapes) and _contiguous(ts)):
        raise RuntimeError(f"{name} must hold contiguous {dtype} tensors of the parameters' shapes on {device}")


def _settings(lr, betas, eps, weight_decay):
    beta1, beta2 = betas
    if not (0.0 <= lr < math.inf and 0.0 <= eps < math.inf and 0.0 <= weight_decay < math.inf
            and 0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise RuntimeError("lr, eps and weight_decay must be finite and not negative and the betas in [0, 1), got "
                           f"{lr}, {eps}, {weight_decay}, {betas}")
    return float(lr), float(beta1), float(beta2), float(eps), float(weight_decay)


@torch.no_grad()
def adamw_update(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 scales=None, seed=0):
    """Step number `step` (from 1 on), in place, over lists of tensors on one device.

    exp_avgs, exp_avg_sqs: float32, or uint8 with a list of scales, as new_moments makes
    them.  A tensor may not come twice, nor overlap another, nor a gradient one of them
    (gradients may be one tensor).  In a captured graph every replay is the step, with
    the rates and the seed, that was captured: its 8-bit moments are rounded by the same
    bits each time."""
    _t.not_traced()
    params, grads = list(params), list(grads)
    how = _settings(lr, betas, eps, weight_decay)
    if not isinstance(step, int) or not 1 <= step < 2 ** 53:
        raise RuntimeError(f"step must be an integer from 1 to 2^53, got {step!r}")
    if not isinstance(seed, int):
        raise RuntimeError(f"seed must be an integer, got {seed!r}")
    if not params:
        return
    first = params[0]
    _t.require_tensor(first, "params")
    dtype, device = first.dtype, first.device
    if not (_are(params, dtype, device) and _contiguous(params)):
        raise RuntimeError(f"params must hold contiguous {dtype} tensors on {device}")
    shapes = list(map(_SHAPE, params))
    if not _contiguous(grads):
        if not all([isinstance(g, torch.Tensor) and g.layout is torch.strided for g in grads]):
            raise RuntimeError("grads must hold dense tensors")
        grads = [g.contiguous() for g in grads]
    if not _are(grads, dtype, device, shapes):
        raise RuntimeError(f"grads must hold a {dtype} tensor of each parameter's shape on {device}")
    moment = torch.float32 if scales is None else torch.uint8
    _checked(exp_avgs, "exp_avgs", moment, device, shapes)
    _checked(exp_avg_sqs, "exp_avg_sqs", moment, device, shapes)
    n, sizes = len(params), list(map(_NUMEL, params))
    pointers = lambda addresses: (C.c_void_p * n).from_buffer(array("Q", addresses))  # noqa: E731
    written = [list(map(_ADDRESS, ts)) for ts in (params, exp_avgs, exp_avg_sqs)]
    low = high = None
    if scales is not None:
        if len(scales) != n:
            raise RuntimeError(f"scales must hold a tensor for each of {n} parameters, got {len(scales)}")
        blocks = [-(-size // BLOCK) for size in sizes]
        strides = list(map(_STRIDE, scales)) if _are(scales, torch.uint8, device, [(2, b) for b in blocks]) else []
        if not strides or not all([row >= b and (one == 1 or b < 2) for b, (row, one) in zip(blocks, strides)]):
            raise RuntimeError(f"scales must hold uint8 tensors of shape (2, ceil(n / {BLOCK})) with contiguous rows on "
                               f"{device}")
        first_rows = list(map(_ADDRESS, scales))
        written += [first_rows, [a + row for a, (row, _) in zip(first_rows, strides)]]
        low, high = (pointers(a) for a in written[3:])
    with _t.on_device(device):
        _t.check(_t.load().gs_adamw_update(
            _t.DTYPE_CODES[dtype], 32 if scales is None else 8, n, (C.c_int64 * n).from_buffer(array("q", sizes)),
            pointers(written[0]), pointers(list(map(_ADDRESS, grads))), pointers(written[1]), pointers(written[2]), low, high,
            C.byref(AdamWSettings(*how, step, seed & 0xFFFFFFFF)), _t.stream(device)), "gs_adamw_update")
    # written through their addresses: graphs that saved them are told
    torch.autograd.graph.increment_version(params)


@torch.no_grad()
def moment_values(exp_avg, exp_avg_sq, scales, dtype=torch.float32):
    """The values that 8-bit moments stand for, float32 or (which holds them whole) bfloat16."""
    _t.not_traced()
    for name, t in (("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq), ("scales", scales)):
        if (not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.uint8 or t.device != exp_avg.device):
            raise RuntimeError(f"{name} must be a uint8 HIP device tensor (of exp_avg's device)")
    n = exp_avg.numel()
    if exp_avg_sq.shape != exp_avg.shape or scales.shape != (2, -(-n // BLOCK)):
        raise RuntimeError(f"exp_avg_sq must have exp_avg's shape and scales (2, {-(-n // BLOCK)}), got "
                           f"{tuple(exp_avg_sq.shape)} and {tuple(scales.shape)}")
    if dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError(f"dtype must be torch.float32 or torch.bfloat16, got {dtype}")
    m, v, scales = exp_avg.contiguous(), exp_avg_sq.contiguous(), scales.contiguous()
    out = [torch.empty(exp_avg.shape, device=exp_avg.device, dtype=dtype) for _ in range(2)]
    with _t.on_device(exp_avg.device):
        _t.check(_t.load().gs_adamw_values(
            _t.DTYPE_CODES[dtype], n, m.data_ptr(), v.data_ptr(), scales.data_ptr(), scales.data_ptr() + scales.stride(0),
            out[0].data_ptr(), out[1].data_ptr(), _t.stream(exp_avg.device)), "gs_adamw_values")
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW whose step takes all tensors of a group through the device together.

    bits: 32 or 8, of the moments.  State per parameter: 'step' (an integer), 'exp_avg',
    'exp_avg_sq' and, with 8 bits, 'scales'; a state with another number of bits than the
    group's is refused by the step.  Steps are counted on the host, so a step cannot be
    captured in a graph; adamw_update can."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, bits=32, seed=0):
        try:
            _settings(lr, betas, eps, weight_decay)
        except RuntimeError as e:
            raise ValueError(str(e)) from None
        if bits not in (8, 32) or not isinstance(seed, int):
            raise ValueError(f"bits must be 8 or 32 and seed an integer, got {bits!r} and {seed!r}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits, seed=seed))

    def load_state_dict(self, state_dict):
        """Takes a state of torch's AdamW and Adam too, moments of 16 bits as float32, unless its groups ask for
        another step than this one."""
        def take(state, loaded, p):
            for name in ("exp_avg", "exp_avg_sq", "scales"):
                t = loaded.get(name)
                if isinstance(t, torch.Tensor):
                    dtype = torch.float32 if t.is_floating_point() else t.dtype
                    state[name] = t.detach().to(p.device, dtype, copy=True).contiguous()
            if "step" in loaded:
                state["step"] = int(loaded["step"])

        def fit(saved):
            groups = []
            for group in saved["param_groups"]:
                for name in ("lr", "betas", "eps", "weight_decay"):
                    if name not in group:
                        raise ValueError(f"a group of the loaded state has no {name}")
                for name in ("amsgrad", "maximize"):
                    if group.get(name):
                        raise ValueError(f"AdamW has no {name}, which the loaded state asks for")
                if group["weight_decay"] and not group.get("decoupled_weight_decay", True):
                    raise ValueError("the loaded state's weight_decay is part of its gradients; AdamW's is not")
                # what says nothing of bits has those of its moments
                held = [saved["state"][k] for k in group["params"] if k in saved["state"]]
                bits = 8 if any("scales" in s for s in held) else 32 if held else self.defaults["bits"]
                groups.append({"bits": bits, "seed": self.defaults["seed"], **group})
            return {**saved, "param_groups": groups}

        _t.load_uncast(self, super().load_state_dict, state_dict, take, fit)

    @torch.no_grad()
    def step(self, closure=None):
        # before anything is made: a capture records new moments' zeros, it does not write them
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW counts its steps on the host and cannot be captured; adamw_update can")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = []
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["step"] = 0
                    state["exp_avg"], state["exp_avg_sq"], scales = new_moments(p, group["bits"])
                    if scales is not None:
                        state["scales"] = scales
                if ("scales" in state) != (group["bits"] == 8):
                    raise RuntimeError(f"a parameter's state has not the {group['bits']} bits of its group")
                alike.setdefault((p.device, p.dtype, state["step"]), []).append((p, state))
            calls += [(group, *key, pairs) for key, pairs in alike.items()]
        for i, (group, _, _, step, pairs) in enumerate(calls):
            params, states = zip(*pairs)
            adamw_update(params, [p.grad for p in params], [s["exp_avg"] for s in states],
                         [s["exp_avg_sq"] for s in states], step + 1, group["lr"], group["betas"], group["eps"],
                         group["weight_decay"], [s["scales"] for s in states] if group["bits"] == 8 else None,
                         group["seed"] + i)
            for s in states:
                s["step"] = step + 1
        return loss
