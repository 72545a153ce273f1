"""The wide categorical head: log-probability, entropy and cross entropy of given classes for logits = hidden weight^T + bias that are never
stored, with gradients (q1env_head_forward / _backward, include/q1env.h).

It is what policy.CategoricalN is over logits that exist (the reference's discrete mouse, Discrete(2S+1): q1physrl/action_dist.py:221-222,
q1physrl_env/q1physrl_env/env.py:216-219).  A minibatch of B samples against 2S+1 classes keeps B x (2S+1) logits, their log-softmax, its
exponential and the gradient of each alive there; here a float or two per sample are kept, and the backward pass works through pieces of the classes.

    logp, entropy = linear_categorical(hidden, weight, actions, bias)      # both float32 (B,), both differentiable
    loss = linear_cross_entropy(hidden, weight, target, bias)              # minus the mean log-probability
    loss, dhidden, dweight, dbias = linear_cross_entropy_grad(...)         # the same with its gradients, without autograd

hidden (..., D), weight (V, D) and bias (V,) are float32, bfloat16 or float16 CUDA tensors of one type; actions / target (...) int32 or int64.  Rows may be
strided; a last dimension that is not contiguous is copied.  Rows whose target is ignore_index are padding: log-probability, entropy and gradients
are zero whatever the hidden row holds.  A target outside 0 .. V-1 gives NaN.  There is no forward-mode derivative and no second one: both raise.  Work runs on the tensors' device, on its current stream.

A captured graph: the forward calls and linear_cross_entropy_grad can be captured; the autograd forms cannot (a capture that meets an eager graph of
the same leaves ends the process), and say so."""
import ctypes as C
import functools

import torch

from . import _lib
from .clip import refuse_tangents

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _rows(x):
    """x (..., D) as (rows, D) with a contiguous last dimension; a copy only where no strided view is one."""
    if x.dim() == 2 and x.is_contiguous():
        return x
    x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


@functools.lru_cache(maxsize=256)
def _state_bytes(n):
    return _lib.load().q1env_head_state_bytes(n)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(dtype, n, d, v, backward):
    return _lib.load().q1env_head_workspace_bytes(dtype, n, d, v, backward)


def _check(hidden, weight, target, bias, ignore_index):
    if not (torch.is_tensor(hidden) and torch.is_tensor(weight) and torch.is_tensor(target) and (bias is None or torch.is_tensor(bias))):
        raise TypeError("hidden, weight, target (and bias) must be tensors")
    if hidden.dtype not in _DTYPES:
        raise TypeError(f"hidden must be float32, bfloat16 or float16, got {hidden.dtype}")
    if weight.dtype != hidden.dtype or (bias is not None and bias.dtype != hidden.dtype):
        raise TypeError("hidden, weight and bias must have one dtype")
    if target.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"classes must be int32 or int64, got {target.dtype}")
    if weight.dim() != 2 or hidden.dim() < 1 or weight.shape[0] < 1 or weight.shape[1] < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden (..., D) and weight (V, D) do not fit: {tuple(hidden.shape)}, {tuple(weight.shape)}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"one class per row of hidden: {tuple(target.shape)} against {tuple(hidden.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"bias must be ({weight.shape[0]},), got {tuple(bias.shape)}")
    if not isinstance(ignore_index, int) or not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must be an int of 64 bits")
    refuse_tangents([t for t in (hidden, weight, bias) if t is not None], "the wide categorical head")
    if not hidden.is_cuda:
        raise _lib.Q1EnvError("the wide categorical head runs on an MI355X only: there is no CPU fallback")
    for t in (weight, target, bias):
        if t is not None and t.device != hidden.device:
            raise ValueError("all tensors must be on one device")


def _head(hidden, weight, target, bias, ignore_index, backward):
    """The C struct of a head without its state, and the tensors it points at: they are referenced until the launches are queued, and the caching allocator keeps
    freed blocks to the stream they were used on."""
    h, w = _rows(hidden), _rows(weight)
    b = None if bias is None else bias.contiguous()
    n, d, v, dtype = h.shape[0], h.shape[1], w.shape[0], _DTYPES[h.dtype]
    nbytes = _workspace_bytes(dtype, n, d, v, backward)
    if not nbytes:
        raise ValueError(f"sizes out of range: {n} rows (2^22), width {d} (2^16), {v} classes (2^22)")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
    s = _lib.Q1Head(dtype, 64 if target is None or target.dtype == torch.int64 else 32, n, d, v, ignore_index, h.data_ptr(), _stride(h), w.data_ptr(), _stride(w),
                    None if b is None else b.data_ptr(), None if target is None else target.data_ptr(), None, ws.data_ptr(), nbytes)
    return s, (h, w, b, target, ws)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _forward(hidden, weight, target, bias, ignore_index, reduction):
    """(logp (n,), entropy (n,), state) without a reduction, (loss (), state) with one"""
    target = target.reshape(-1).contiguous()
    s, keep = _head(hidden, weight, target, bias, ignore_index, 0)
    device, n = hidden.device, s.rows
    state = torch.empty(_state_bytes(n), dtype=torch.uint8, device=device)
    s.state_dev = state.data_ptr()
    logp = torch.empty(n, dtype=torch.float32, device=device)
    ent = loss = None
    if reduction is None:
        ent = torch.empty(n, dtype=torch.float32, device=device)
    else:
        loss = torch.empty((), dtype=torch.float32, device=device)
    _lib.check(_lib.load().q1env_head_forward(device.index, _stream(device), C.byref(s), _lib.REDUCE_SUM if reduction == "sum" else _lib.REDUCE_MEAN, logp.data_ptr(),
                                              None if ent is None else ent.data_ptr(), None if loss is None else loss.data_ptr()))
    del keep
    return (logp, ent, state) if reduction is None else (loss, state)


def _upstream(g):
    return g if g is None or (g.dtype == torch.float32 and g.is_contiguous()) else g.to(torch.float32).contiguous()


def _backward(hidden, weight, bias, state, dlogp, dentropy, dloss, need):
    """need: which of (hidden, weight, bias) to differentiate; their gradients or None"""
    s, keep = _head(hidden, weight, None, bias, 0, 1)
    s.state_dev = state.data_ptr()
    dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if need[0] else None
    dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if need[1] else None
    db = torch.empty(bias.shape, dtype=bias.dtype, device=bias.device) if need[2] and bias is not None else None
    if dh is None and dw is None and db is None:
        return dh, dw, db
    up = _upstream(dlogp), _upstream(dentropy), _upstream(dloss)
    _lib.check(_lib.load().q1env_head_backward(hidden.device.index, _stream(hidden.device), C.byref(s), *[None if g is None else g.data_ptr() for g in up],
                                               None if dh is None else dh.data_ptr(), s.width, None if dw is None else dw.data_ptr(), s.width,
                                               None if db is None else db.data_ptr()))
    del keep
    return dh, dw, db


class _Categorical(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, bias, ignore_index, reduction):
        *out, state = _forward(hidden, weight, target, bias, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, bias, state)
        ctx.reduction = reduction
        ctx.set_materialize_grads(False)
        return tuple(out) if reduction is None else out[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the backward pass of the wide categorical head cannot be captured into a graph: capture linear_cross_entropy_grad")
        if all(g is None for g in grads):
            return None, None, None, None, None, None
        hidden, weight, bias, state = ctx.saved_tensors
        up = (grads[0], grads[1], None) if ctx.reduction is None else (None, None, grads[0])
        need = ctx.needs_input_grad
        dh, dw, db = _backward(hidden, weight, bias, state, *up, (need[0], need[1], need[3]))
        return dh, dw, None, db, None, None


def _apply(hidden, weight, target, bias, ignore_index, reduction):
    _check(hidden, weight, target, bias, ignore_index)
    if not (torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))):
        return _forward(hidden, weight, target, bias, ignore_index, reduction)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the differentiable forms cannot be captured into a graph: capture linear_cross_entropy_grad, or the forward under torch.no_grad()")
    out = _Categorical.apply(hidden, weight, target, bias, ignore_index, reduction)
    return out if reduction is None else (out,)


def linear_categorical(hidden, weight, actions, bias=None, *, ignore_index=-100):
    """(log-probability, entropy) of the given actions, float32, in actions' shape."""
    logp, ent = _apply(hidden, weight, actions, bias, ignore_index, None)[:2]
    return (logp, ent) if actions.dim() == 1 else (logp.view(actions.shape), ent.view(actions.shape))


def linear_cross_entropy(hidden, weight, target, bias=None, *, ignore_index=-100, reduction="mean"):
    """Minus the log-probability of the targets: its mean over the rows that are not ignored (0 when all are), "sum", or "none" (per row)."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if reduction == "none":
        return -_apply(hidden, weight, target, bias, ignore_index, None)[0].view(target.shape)
    return _apply(hidden, weight, target, bias, ignore_index, reduction)[0]


@torch.no_grad()
def linear_cross_entropy_grad(hidden, weight, target, bias=None, *, ignore_index=-100, reduction="mean", grad_scale=None):
    """(loss, dhidden, dweight, dbias or None) without autograd.  grad_scale: optional float32 device scalar the gradients are multiplied by."""
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean' or 'sum', got {reduction!r}")
    _check(hidden, weight, target, bias, ignore_index)
    if grad_scale is not None and not (torch.is_tensor(grad_scale) and grad_scale.numel() == 1 and grad_scale.dtype == torch.float32 and grad_scale.device == hidden.device):
        raise ValueError("grad_scale must be one float32 on hidden's device")
    loss, state = _forward(hidden, weight, target, bias, ignore_index, reduction)
    one = torch.ones((), dtype=torch.float32, device=hidden.device) if grad_scale is None else grad_scale
    return loss, *_backward(hidden, weight, bias, state, None, None, one, (True, True, True))
