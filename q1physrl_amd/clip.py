"""The global norm of many gradients, and clipping by it (q1env_grad_norm / q1env_grad_clip, include/q1env.h): RLlib's `grad_clip`, which its TF
policies apply with tf.clip_by_global_norm; the reference's trainer config leaves it unset (data/params.yml:2-13).

    norm = clip_grad_norm_([p.grad for p in params], 0.5)          # in place; norm: float32 () on the device, no synchronisation
    norm = clip_grad_norm_(bucket_views, 0.5, scale=1 / world, out=[p.grad for p in params])

Tensors: CUDA, one device, float32 / bfloat16 / float16 (mixed as they come), any shape; dense ones in any order of dimensions, or rows of contiguous
values at a pitch (a column slice).  Results carry no graph, as those of torch's own clipping do not: a norm is no loss term, and forward-mode tangents are refused.  Squares are summed in float64 in an order that the sizes alone fix: the same bits every time."""
import functools
import operator
from array import array

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_T = torch.Tensor
_PLAIN = {torch.Tensor, torch.nn.Parameter}
_dtype, _shape = operator.attrgetter("dtype"), operator.attrgetter("shape")


@functools.lru_cache(maxsize=64)
def _workspace_bytes(count):
    return _lib.load().q1env_grad_norm_workspace_bytes(count)


def refuse_tangents(tensors, what):
    """Raises where a tensor carries a forward-mode tangent: the kernels would drop it without a word."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _address(a):
    return None if a is None else a.buffer_info()[0]


def _pitched(t):
    """(columns, pitch) of a tensor that is rows of contiguous values at a pitch, (0, 0) of a dense one; None of anything else."""
    dims = sorted(((st, n) for n, st in zip(t.shape, t.stride()) if n != 1), reverse=True)
    if any(st <= 0 for st, _ in dims):
        return None
    run = 1                                              # values that lie one behind the other, from the innermost dimension out
    while dims and dims[-1][0] == run:
        run *= dims.pop()[1]
    if not dims:
        return 0, 0
    pitch = dims[-1][0]
    rows = pitch
    while dims and dims[-1][0] == rows:
        rows *= dims.pop()[1]
    return (run, pitch) if not dims and pitch > run else None


def _order(t):
    """the dimensions of more than one value, outermost in memory first"""
    return sorted((d for d in range(t.dim()) if t.shape[d] != 1), key=t.stride, reverse=True)


def _layouts(tensors, out):
    """The cols / src_pitch / dst_pitch arrays of tensors that are not all contiguous."""
    cols, sp, dp = (array("q", bytes(8 * len(tensors))) for _ in range(3))
    for i, t in enumerate(tensors):
        o = t if out is None else out[i]
        if t.numel() == 0:
            continue
        if t.is_neg() != o.is_neg():
            raise ValueError(f"tensor {i} or its out is a lazily negated view (of a conjugate): call resolve_neg() first")
        a, b = _pitched(t), _pitched(o)
        c = 0 if a is None or b is None else min((x for x in (a[0], b[0]) if x), default=0)
        if a is None or b is None or (out is not None and _order(t) != _order(o)) or (a[0] or c) != c or (b[0] or c) != c:
            raise ValueError(f"tensor {i} of shape {tuple(t.shape)}: strides {t.stride()}" + ("" if out is None else f", out {o.stride()}")
                             + " are neither dense nor rows of contiguous values at a pitch, in one order")
        if c:
            cols[i], sp[i], dp[i] = c, a[1] or c, b[1] or c
    return cols, sp, dp


def _tensors(tensors, what):
    tensors = [tensors] if isinstance(tensors, _T) else list(tensors)
    if not _PLAIN.issuperset(map(type, tensors)) and not all(map(torch.is_tensor, tensors)):
        raise TypeError(f"{what}: tensors only")
    return tensors


def _run(tensors, out, max_norm, scale):
    tensors = _tensors(tensors, "gradients")
    scale = float(scale)
    if not (0.0 < scale < float("inf")):
        raise ValueError("scale must be positive and finite")
    if max_norm is not None and not float(max_norm) >= 0.0:
        raise ValueError("max_norm must not be negative or NaN")
    n = len(tensors)
    if n == 0:
        raise ValueError("no tensors: there is no device to put the norm on")
    if n > 65536:
        raise ValueError("more than 65536 tensors")
    refuse_tangents(tensors, "the gradient norm")
    kinds = list(map(_dtype, tensors))
    if not _DTYPES.keys() >= set(kinds):
        raise TypeError(f"gradients must be float32, bfloat16 or float16, got {set(kinds) - set(_DTYPES)}")
    values = list(map(_T.numel, tensors))
    devices = set(map(_T.get_device, tensors))
    plain = all(map(_T.is_contiguous, tensors))
    if out is not None:
        out = _tensors(out, "out")
        if len(out) != n:
            raise ValueError(f"{len(out)} tensors in out for {n} gradients")
        if list(map(_dtype, out)) != kinds:
            raise TypeError("out must have the gradients' dtypes")
        plain = plain and all(map(_T.is_contiguous, out))
        if list(map(_T.numel, out)) != values or (not plain and list(map(_shape, out)) != list(map(_shape, tensors))):
            raise ValueError("out must have the gradients' shapes (their numbers of values where all are contiguous)")
        devices |= set(map(_T.get_device, out))
    if min(devices) < 0:
        raise _lib.Q1EnvError("gradient clipping runs on an MI355X only: there is no CPU fallback")
    if len(devices) != 1:
        raise ValueError("all tensors must be on one device")
    cols = sp = dp = None
    if not plain:
        if out is not None or max_norm is None:          # only read: a broadcast gradient (stride 0) counts as the values it stands for
            tensors = [t if t.is_contiguous() or _pitched(t) is not None else t.contiguous() for t in tensors]
        cols, sp, dp = _layouts(tensors, out)
    src = array("Q", map(_T.data_ptr, tensors))
    sizes = array("q", values)
    dtype = array("i", map(_DTYPES.__getitem__, kinds))
    dev = devices.pop()
    device = tensors[0].device
    lib = _lib.load()
    nbytes = _workspace_bytes(n)
    buf = torch.empty(nbytes, dtype=torch.uint8, device=device)                          # the partial sums, and a long list's table
    norm = torch.empty((), dtype=torch.float32, device=device)
    stream = torch.cuda.current_stream(device).cuda_stream
    p = _address
    if max_norm is None:
        _lib.check(lib.q1env_grad_norm(dev, stream, n, p(src), p(sizes), p(dtype), p(cols), p(sp), scale, norm.data_ptr(), buf.data_ptr(), nbytes))
    else:
        dst = src if out is None else array("Q", map(_T.data_ptr, out))
        _lib.check(lib.q1env_grad_clip(dev, stream, n, p(src), p(dst), p(sizes), p(dtype), p(cols), p(sp), p(dp), scale, float(max_norm), norm.data_ptr(),
                                       buf.data_ptr(), nbytes))
        written = tensors if out is None else out
        try:
            torch.autograd.graph.increment_version(written)                              # autograd has to know what was written
        except RuntimeError:
            if not any(map(_T.is_inference, written)):                                   # (tensors made in inference mode have no version)
                raise
    return norm


def grad_norm(grads, *, scale=1.0):
    """|scale| x the 2-norm over all tensors: float32 () on their device."""
    return _run(grads, None, None, scale)


def clip_grad_norm_(grads, max_norm, *, scale=1.0, out=None):
    """grads <- grads x scale x min(1, max_norm / norm), norm = grad_norm(grads, scale=scale); returns the norm.  out: where the results go instead
    (tensors of the same shapes - or, where all are contiguous, sizes - and dtypes that overlap nothing but, each, its own source); the gradients stay as they are.  A NaN gradient makes the norm and every
    result NaN, an infinite one turns finite values to zero.  A norm past float32's range is returned as inf; the gradients are clipped by its float64 value."""
    return _run(grads, out, max_norm, scale)
