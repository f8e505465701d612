"""What the token operators' Python entry points share: element types, checks of
tensor arguments, streams and workspaces."""
import contextlib

import torch
from torch.autograd import forward_ad

from . import _lib

# the C ABI's element types (GS_F32, GS_BF16, GS_F16)
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HERE = contextlib.nullcontext()


def require_tensor(t, name, device=None):
    """t is a float32, bfloat16 or float16 HIP device tensor (on `device`)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a HIP device tensor (blitzgs_amd has no CPU path)")
    if t.dtype not in DTYPE_CODES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")


_tracing = torch._C._get_tracing_state


def not_traced():
    """A trace would hold the results' memory and not the kernels, or the kernels without the checks of their
    arguments, on tensors of other sizes."""
    if _tracing() is not None:
        raise RuntimeError("the operators of blitzgs_amd cannot be traced")


def ptr(t):
    """A tensor's address; None (NULL) for no tensor."""
    return None if t is None else t.data_ptr()


# The current stream's handle.  torch.cuda.current_stream wraps it in an object,
# which costs more than the rest of a small backward's work on the host (13 us in
# the autograd engine's thread); it stays the fallback.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream(device):
    return _raw_stream(device.index) if _raw_stream else torch.cuda.current_stream(device).cuda_stream


def on_device(device):
    """A context in which `device` is the current one: launches go to the current device."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def workspace(nbytes, device):
    """A byte buffer of a *_bytes query's size; None where nothing is needed."""
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


def wants_grad(*tensors):
    """Whether a call has to go through its autograd function: a backward may follow, or
    a tensor has a forward-mode tangent, which that function refuses.  A call that does not
    is not traced."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    # -1 outside all dual levels, where no tensor has a tangent
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        return True
    not_traced()
    return False


def load_uncast(optimizer, load, state_dict, take, fit=None):
    """load(state_dict) of an optimiser whose state keeps its own types: torch's loading
    casts a state to its parameter's type, so take(state, loaded, parameter) takes from
    what was loaded once more: after all hooks that may change that, and before any that
    look at the result.  fit(state_dict) may refuse what is loaded, or give it otherwise."""
    loaded = {}

    def look(_, state):
        state = state if fit is None else fit(state)
        loaded.update(state)
        return state

    def restore(_):
        ours = (p for group in optimizer.param_groups for p in group["params"])
        for key, p in zip((k for group in loaded["param_groups"] for k in group["params"]), ours):
            if key in loaded["state"]:
                take(optimizer.state[p], loaded["state"][key], p)

    hooks = [optimizer.register_load_state_dict_pre_hook(look),
             optimizer.register_load_state_dict_post_hook(restore, prepend=True)]
    try:
        load(state_dict)
    finally:
        for hook in hooks:
            hook.remove()


check = _lib.check
load = _lib.load
