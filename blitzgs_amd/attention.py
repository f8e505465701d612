"""attention: scaled dot-product attention with a backward that recomputes the
probabilities.

    o = softmax(scale q k^T) v, per head, over the keys that a query sees

q and o are (B, Hq, Tq, D), k and v (B, Hkv, Tk, D); Hq is a multiple of Hkv,
and query head h reads key head h // (Hq // Hkv).  float32, bfloat16 or
float16, one type for all; D from 1 to 128.  Any strides are taken as they are
as long as the last dimension is contiguous, so projections of shape (B, T, H, D)
and slices of a fused projection are passed as transposed views.

Query i of batch b sees key j when j < key_lengths[b] and, with causal,
j <= i + query_start[b].  By default the last query sees the last of Tk keys.
A query that sees no key gives zeros and no gradient, and keys from
key_lengths on are never read, nor are those that no query sees.  A NaN or an
infinity reaches the queries that see its key and, in the backward, the keys that
its query sees, and no others.

Scores, softmax and all sums are fp32; probabilities are rounded to the
tensors' type for the product with v.  The sums come before their division by the
softmax's, so values of v beyond 1e36 / Tk may pass fp32's range; float16's values
never do.  Nothing of size Tq x Tk is stored: a call that needs gradients keeps q,
k, v, o, one number per query, and in the 16-bit types a second part of o.  Equal
inputs give equal bits.
"""
import ctypes as C
import math

import torch

from . import _tensors as _t

MAX_HEAD_DIM = 128


_Strides = C.c_int64 * 3


def _strides(t):
    return _Strides(*t.stride()[:3])


def _last_contiguous(t):
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _token_major(like):
    """An empty (B, H, T, D) tensor that lies as (B, T, H, D), ready for the next projection."""
    B, H, T, D = like.shape
    return torch.empty_strided((B, H, T, D), (T * H * D, D, H * D, 1), device=like.device, dtype=like.dtype)


def _forward(q, k, v, causal, key_lengths, query_start, scale, grads):
    """o and, for a backward, what rounding o left, lse, and what the backward is called with."""
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1:3]
    lib, sizes = _t.load(), (_t.DTYPE_CODES[q.dtype], B, Hq, Hkv, Tq, Tk, D)
    unequal = int(causal or key_lengths is not None)
    o = _token_major(q)
    lse = torch.empty((B, Hq, Tq), device=q.device, dtype=torch.float32) if grads else None
    rest = _token_major(q) if grads and q.dtype != torch.float32 else None
    ws = _t.workspace(lib.gs_attention_workspace_bytes(*sizes, unequal, 0), q.device)
    laid = q.stride(), k.stride(), v.stride(), o.stride()
    strides = [_Strides(*s[:3]) for s in laid]
    with _t.on_device(q.device):
        _t.check(lib.gs_attention_forward(
            *sizes, q.data_ptr(), strides[0], k.data_ptr(), strides[1], v.data_ptr(), strides[2], scale, int(causal),
            _t.ptr(key_lengths), _t.ptr(query_start), o.data_ptr(), strides[3], _t.ptr(rest), _t.ptr(lse),
            _t.ptr(ws), _t.stream(q.device)), "gs_attention_forward")
    return o, rest, lse, (sizes, strides, laid, unequal, scale, int(causal))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, key_lengths, query_start, scale):
        q, k, v = (_last_contiguous(t.detach()) for t in (q, k, v))
        o, rest, lse, ctx.how = _forward(q, k, v, causal, key_lengths, query_start, scale, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, key_lengths, query_start)
        ctx.ws_bytes = _t.load().gs_attention_workspace_bytes(*ctx.how[0], ctx.how[3], 1)
        return o

    # The autograd engine calls this from a thread of its own, on the forward's
    # device and stream: what does not need the gradient is prepared by forward.
    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, rest, lse, key_lengths, query_start = ctx.saved_tensors
        sizes, (qs, ks, vs, os), laid, _, scale, causal = ctx.how
        do = _last_contiguous(do)
        dq, dk, dv, beside = _token_major(q), None, None, ks
        dqs = os
        if ((q.stride(), k.stride(), v.stride(), o.stride()) != laid or (rest is not None and rest.stride() != laid[3])
                or not lse.is_contiguous() or (key_lengths is not None and not key_lengths.is_contiguous())
                or (query_start is not None and not query_start.is_contiguous())):
            # hooks on saved tensors give them back with the same values, not in the same places
            q, k, v, o, lse = (t.contiguous() for t in (q, k, v, o, lse))
            rest, key_lengths, query_start = (t if t is None else t.contiguous()
                                              for t in (rest, key_lengths, query_start))
            qs, ks, vs, os, dqs = (_strides(t) for t in (q, k, v, o, dq))
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dk, dv = _token_major(k), _token_major(v)
            beside = _strides(dk)
        ws = _t.workspace(ctx.ws_bytes, q.device)
        _t.check(_t.load().gs_attention_backward(
            *sizes, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, scale, causal, _t.ptr(key_lengths),
            _t.ptr(query_start), o.data_ptr(), os, _t.ptr(rest), lse.data_ptr(), do.data_ptr(), _strides(do),
            dq.data_ptr(), dqs, _t.ptr(dk), beside, _t.ptr(dv), beside, _t.ptr(ws), _t.stream(q.device)),
            "gs_attention_backward")
        return dq, dk, dv, None, None, None, None


def _per_batch(t, name, q):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.device != q.device or t.dtype != torch.int32 or t.shape != q.shape[:1]:
        raise RuntimeError(f"{name} must be an int32 tensor of shape ({q.shape[0]},) on {q.device}")
    return t.contiguous()


def attention(q, k, v, causal=False, key_lengths=None, query_start=None, scale=None):
    """Attention of q over k and v; differentiable in the three.

    key_lengths, query_start: int32 (B,) on q's device, or None.
    scale: a positive number; None for 1 / sqrt(D)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _t.require_tensor(t, name, device=None if name == "q" else q.device)
        if t.dim() != 4:
            raise RuntimeError(f"{name} must have dimensions (B, H, T, D), got shape {tuple(t.shape)}")
        if t.dtype != q.dtype:
            raise RuntimeError(f"{name} must be {q.dtype} like q, got {t.dtype}")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise RuntimeError("k and v must have one shape, with q's batch and head dimension; got q "
                           f"{tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise RuntimeError(f"q's {q.shape[1]} heads must be a multiple of k's {k.shape[1]}")
    if not 1 <= q.shape[3] <= MAX_HEAD_DIM:
        raise RuntimeError(f"the head dimension must be in 1 to {MAX_HEAD_DIM}, got {q.shape[3]}")
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise RuntimeError(f"scale must be a positive number, got {scale}")
    if query_start is not None and not causal:
        raise RuntimeError("query_start needs causal=True")
    how = bool(causal), _per_batch(key_lengths, "key_lengths", q), _per_batch(query_start, "query_start", q), scale
    if _t.wants_grad(q, k, v):
        return _Attention.apply(q, k, v, *how)
    return _forward(*(_last_contiguous(t) for t in (q, k, v)), *how, False)[0]
