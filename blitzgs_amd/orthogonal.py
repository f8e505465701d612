"""orthogonalise: the orthogonalised update of weight matrices, and the
optimiser that takes it.

A matrix G = U S V^T is replaced by a matrix near U V^T, through steps of

    A = X X^T,  X <- a X + (b A + c A A) X,  a, b, c = 3.4445, -4.7750, 2.0315

from X = G / (|G| + 1e-7) on the shorter side's rows.  Singular values do not
end at 1 but within about 0.7 to 1.2.  Products keep fp32's accuracy whatever
the matrices' type; the result is rounded to it once.

SparseGaussianAdam updates the per-Gaussian tensors of a scene;
OrthogonalMomentum updates the weight matrices of a network in front of it.
"""
import ctypes as C

import torch

from . import _tensors as _t

_MAX_PER_CALL = 32      # tensors per gs_momentum_* call


def _orthogonalise(stack, steps):
    count, m, n = stack.shape
    lib = _t.load()
    out = torch.empty_like(stack)
    ws = _t.workspace(lib.gs_orthogonalise_workspace_bytes(count, m, n), stack.device)
    with _t.on_device(stack.device):
        _t.check(lib.gs_orthogonalise(_t.DTYPE_CODES[stack.dtype], count, m, n, _t.ptr(stack), steps,
                                        _t.ptr(out), _t.ptr(ws), _t.stream(stack.device)), "gs_orthogonalise")
    return out


@torch.no_grad()
def orthogonalise(update, steps=5):
    """The orthogonalised matrices of update (..., m, n), in its shape and type.

    All matrices of one call go through the device together.  Not
    differentiable.  steps: 1 to 32."""
    _t.not_traced()
    _t.require_tensor(update, "update")
    if update.dim() < 2 or max(update.shape[-2:]) > 65536:
        raise RuntimeError(f"update must hold matrices with sides of up to 65536, got shape {tuple(update.shape)}")
    if not isinstance(steps, int) or not 1 <= steps <= 32:
        raise RuntimeError(f"steps must be an integer from 1 to 32, got {steps!r}")
    if update.numel() == 0:
        return torch.empty_like(update)
    stack = update.reshape(-1, *update.shape[-2:]).contiguous()
    if stack.shape[0] > 65535:
        raise RuntimeError(f"update may hold at most 65535 matrices, got {stack.shape[0]}")
    return _orthogonalise(stack, steps).view(update.shape)


class OrthogonalMomentum(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised, for weight matrices (two dimensions).

        m = momentum m + g,   u = g + momentum m (nesterov) or m
        p = (1 - lr weight_decay) p - lr sqrt(max(1, rows / columns)) orthogonalise(u)

    The state is one fp32 tensor per parameter, 'momentum_buffer', in a saved
    state too.  Parameters of one shape and type in a group go through the device
    together."""

    def __init__(self, params, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5):
        if not lr >= 0.0 or not 0.0 <= momentum < 1.0 or not weight_decay >= 0.0:
            raise ValueError(f"lr and weight_decay must not be negative and momentum in [0, 1), got {lr}, "
                             f"{weight_decay}, {momentum}")
        if not isinstance(steps, int) or not 1 <= steps <= 32:
            raise ValueError(f"steps must be an integer from 1 to 32, got {steps!r}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps))

    def load_state_dict(self, state_dict):
        def take(state, loaded, p):
            buffer = loaded.get("momentum_buffer")
            if isinstance(buffer, torch.Tensor):
                state["momentum_buffer"] = buffer.detach().to(p.device, torch.float32, copy=True).contiguous()

        _t.load_uncast(self, super().load_state_dict, state_dict, take)

    def _buffer(self, p):
        state = self.state[p]
        if "momentum_buffer" not in state:
            state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
        m = state["momentum_buffer"]
        if (not isinstance(m, torch.Tensor) or m.dtype != torch.float32 or m.shape != p.shape or m.device != p.device
                or not m.is_contiguous()):
            raise RuntimeError(f"momentum_buffer must be a contiguous float32 tensor of shape {tuple(p.shape)} on "
                               f"{p.device}")
        return m

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                _t.require_tensor(p, "param")
                if p.dim() != 2:
                    raise RuntimeError(f"OrthogonalMomentum takes matrices, got shape {tuple(p.shape)}")
                if not p.is_contiguous() or p.grad.dtype != p.dtype or p.grad.is_sparse:
                    raise RuntimeError("parameters must be contiguous, with dense gradients of their type")
                alike.setdefault((p.device, p.dtype, tuple(p.shape)), []).append((p, self._buffer(p)))
            for (device, dtype, shape), pairs in alike.items():
                for i in range(0, len(pairs), _MAX_PER_CALL):
                    with _t.on_device(device):
                        self._update(group, *zip(*pairs[i:i + _MAX_PER_CALL]), device, dtype, shape)
        return loss

    def _update(self, group, params, momenta, device, dtype, shape):
        lib, code, n = _t.load(), _t.DTYPE_CODES[dtype], len(params)
        stream, size = _t.stream(device), shape[0] * shape[1]
        grads = [p.grad.contiguous() for p in params]
        pointers = lambda ts: (C.c_void_p * n)(*(t.data_ptr() for t in ts))  # noqa: E731
        update = torch.empty((n, *shape), device=device, dtype=torch.float32)
        _t.check(lib.gs_momentum_update(code, n, size, pointers(grads), pointers(momenta), group["momentum"],
                                          int(group["nesterov"]), _t.ptr(update), stream), "gs_momentum_update")
        update = _orthogonalise(update, group["steps"])
        scale = max(1.0, shape[0] / shape[1]) ** 0.5
        _t.check(lib.gs_momentum_apply(code, n, size, pointers(params), 1.0 - group["lr"] * group["weight_decay"],
                                         group["lr"] * scale, _t.ptr(update), stream), "gs_momentum_apply")
        # written through their addresses: graphs that saved them are told
        torch.autograd.graph.increment_version(params)
