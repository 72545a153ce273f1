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
are zero whatever the hidden row holds.  A target outside 0 .. V-1 gives NaN.  Work runs on the tensors' device, on its current stream.

A captured graph: the forward calls and linear_cross_entropy_grad can be captured; the autograd forms cannot (a capture that meets an eager graph of
the same leaves ends the process), and say so."""
import ctypes as C

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _rows(x):
    """x (..., D) as (rows, D) with a contiguous last dimension; a copy only where no strided view is one."""
    x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


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
    if not hidden.is_cuda:
        raise _lib.Q1EnvError("the wide categorical head runs on an MI355X only: there is no CPU fallback")
    for t in (weight, target, bias):
        if t is not None and t.device != hidden.device:
            raise ValueError("all tensors must be on one device")


class _Call:
    """One head's tensors as the C struct wants them.  Everything it points at stays referenced here until the launches are queued; the caching
    allocator keeps freed blocks to the stream they were used on."""

    def __init__(self, hidden, weight, target, bias, ignore_index, state=None):
        self.lib = _lib.load()
        self.hidden, self.weight = _rows(hidden.detach()), _rows(weight.detach())
        self.bias = None if bias is None else bias.detach().contiguous()
        self.target = None if target is None else target.reshape(-1).contiguous()
        self.dtype = _DTYPES[hidden.dtype]
        self.n, self.d, self.v = self.hidden.shape[0], self.hidden.shape[1], self.weight.shape[0]
        self.device = hidden.device
        nstate = self.lib.q1env_head_state_bytes(self.n)
        if not nstate:
            raise ValueError(f"{self.n} rows are more than the head takes (2^22)")
        self.state = torch.empty((nstate,), dtype=torch.uint8, device=self.device) if state is None else state
        self.ignore_index = ignore_index

    def struct(self, backward):
        nbytes = self.lib.q1env_head_workspace_bytes(self.dtype, self.n, self.d, self.v, backward)
        if not nbytes:
            raise ValueError(f"sizes out of range: {self.n} rows, width {self.d}, {self.v} classes")
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=self.device)
        return ws, _lib.Q1Head(self.dtype, 64 if self.target is None or self.target.dtype == torch.int64 else 32, self.n, self.d, self.v, self.ignore_index,
                               self.hidden.data_ptr(), _stride(self.hidden), self.weight.data_ptr(), _stride(self.weight),
                               0 if self.bias is None else self.bias.data_ptr(), 0 if self.target is None else self.target.data_ptr(),
                               self.state.data_ptr(), ws.data_ptr(), nbytes)

    def _at(self):
        return self.device.index, torch.cuda.current_stream(self.device).cuda_stream

    def forward(self, entropy, reduction):
        """logp (n,), entropy (n,) or None, loss () or None"""
        ws, s = self.struct(0)
        f32 = dict(dtype=torch.float32, device=self.device)
        logp = torch.empty((self.n,), **f32)
        ent = torch.empty((self.n,), **f32) if entropy else None
        loss = torch.empty((), **f32) if reduction is not None else None
        dev, stream = self._at()
        _lib.check(self.lib.q1env_head_forward(dev, stream, C.byref(s), _lib.REDUCE_SUM if reduction == "sum" else _lib.REDUCE_MEAN, logp.data_ptr(),
                                               ent.data_ptr() if entropy else None, loss.data_ptr() if reduction is not None else None))
        return logp, ent, loss

    def backward(self, dlogp, dentropy, dloss, need):
        """need: which of (hidden, weight, bias) to differentiate; their gradients ((n, d), (v, d), (v,)) or None"""
        ws, s = self.struct(1)
        opt = dict(dtype=self.hidden.dtype, device=self.device)
        dh = torch.empty((self.n, self.d), **opt) if need[0] else None
        dw = torch.empty((self.v, self.d), **opt) if need[1] else None
        db = torch.empty((self.v,), **opt) if need[2] and self.bias is not None else None
        if dh is None and dw is None and db is None or (dlogp is None and dentropy is None and dloss is None):
            return dh, dw, db
        f = [None if g is None else g.to(torch.float32).reshape(-1).contiguous() for g in (dlogp, dentropy, dloss)]
        dev, stream = self._at()
        _lib.check(self.lib.q1env_head_backward(dev, stream, C.byref(s), *[None if g is None else g.data_ptr() for g in f],
                                                None if dh is None else dh.data_ptr(), self.d, None if dw is None else dw.data_ptr(), self.d,
                                                None if db is None else db.data_ptr()))
        return dh, dw, db


def _refuse_capture(tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the differentiable forms cannot be captured into a graph: capture linear_cross_entropy_grad, or the forward under torch.no_grad()")


class _Categorical(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, bias, ignore_index, reduction):
        call = _Call(hidden, weight, target, bias, ignore_index)
        logp, ent, loss = call.forward(reduction is None, reduction)
        ctx.save_for_backward(hidden, weight, bias, call.state)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        ctx.set_materialize_grads(False)
        return (logp, ent) if reduction is None else loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        hidden, weight, bias, state = ctx.saved_tensors
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the backward pass of the wide categorical head cannot be captured into a graph: capture linear_cross_entropy_grad")
        need = (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3])
        if all(g is None for g in grads):
            return None, None, None, None, None, None
        call = _Call(hidden, weight, None, bias, ctx.ignore_index, state)
        up = (grads[0], grads[1], None) if ctx.reduction is None else (None, None, grads[0])
        dh, dw, db = call.backward(*up, need)
        return (None if dh is None else dh.view(hidden.shape)), dw, None, db, None, None


def linear_categorical(hidden, weight, actions, bias=None, *, ignore_index=-100):
    """(log-probability, entropy) of the given actions, float32, in actions' shape."""
    _check(hidden, weight, actions, bias, ignore_index)
    _refuse_capture((hidden, weight, bias))
    logp, ent = _Categorical.apply(hidden, weight, actions, bias, ignore_index, None)
    return logp.view(actions.shape), ent.view(actions.shape)


def linear_cross_entropy(hidden, weight, target, bias=None, *, ignore_index=-100, reduction="mean"):
    """Minus the log-probability of the targets: its mean over the rows that are not ignored (0 when all are), "sum", or "none" (per row)."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    _check(hidden, weight, target, bias, ignore_index)
    _refuse_capture((hidden, weight, bias))
    if reduction == "none":
        return -_Categorical.apply(hidden, weight, target, bias, ignore_index, None)[0].view(target.shape)
    return _Categorical.apply(hidden, weight, target, bias, ignore_index, reduction)


@torch.no_grad()
def linear_cross_entropy_grad(hidden, weight, target, bias=None, *, ignore_index=-100, reduction="mean", grad_scale=None):
    """(loss, dhidden, dweight, dbias or None) without autograd.  grad_scale: optional float32 device scalar the gradients are multiplied by."""
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean' or 'sum', got {reduction!r}")
    _check(hidden, weight, target, bias, ignore_index)
    if grad_scale is not None and not (torch.is_tensor(grad_scale) and grad_scale.numel() == 1 and grad_scale.dtype == torch.float32 and grad_scale.device == hidden.device):
        raise ValueError("grad_scale must be one float32 on hidden's device")
    call = _Call(hidden, weight, target, bias, ignore_index)
    _, _, loss = call.forward(False, reduction)
    one = torch.ones((), dtype=torch.float32, device=call.device) if grad_scale is None else grad_scale
    dh, dw, db = call.backward(None, None, one, (True, True, True))
    return loss, dh.view(hidden.shape), dw, db
