"""The global gradient norm and clipping by it (q1physrl_amd/clip.py, q1env_grad_norm / q1env_grad_clip) against float64, and its refusals.

Tolerances: the norm is a float64 sum rounded once: 2^-24 relative, and 2^-40 for the sum.  A clipped value is one float32 factor (2^-24) times the value, one
rounding in float32 and one to the type: 3 x 2^-24 + the type's half step, relative; in float16 its subnormal half step 2^-25."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from q1physrl_amd import _lib, clip

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(sizes, dtypes, seed=0, amp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * amp).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def truth(grads, max_norm, scale):
    norm = scale * math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in grads))
    c = scale * (1.0 if norm <= max_norm else max_norm / norm)
    return norm, [g.double() * c for g in grads]


def check(got_norm, got, grads, max_norm, scale):
    norm, ref = truth(grads, max_norm, scale)
    assert abs(float(got_norm) - norm) <= norm * (2.0 ** -24 + 2.0 ** -40)
    for x, r in zip(got, ref):
        tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
        tol = r.abs() * (3 * 2.0 ** -24 + HALF[x.dtype] * 1.01) + tiny
        assert x.shape == r.shape and bool(((x.double() - r).abs() <= tol).all())


SETS = [[(1,)], [(3,), (1,), (5, 7)], [(256, 6), (256,), (256, 256), (256,), (10, 256), (10,)], [(1,)] * 700, [(9001,), (0,), (8191,), (8193,), (0, 3), (16384,)],
        [(3_000_001,), (2,), (1_000_003,)], [(i % 97 + 1,) for i in range(230)]]


@gpu
@pytest.mark.parametrize("dtypes", [[d] for d in DTYPES] + [DTYPES], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("sizes", SETS, ids=range(len(SETS)))
@pytest.mark.parametrize("max_norm,scale", [(0.5, 1.0), (1e9, 1.0), (0.25, 0.125)])
def test_against_float64(sizes, dtypes, max_norm, scale):
    grads = make(sizes, dtypes, seed=len(sizes))
    kept = [g.clone() for g in grads]
    out = [torch.full_like(g, 7.0) for g in grads]
    n1 = clip.clip_grad_norm_(grads, max_norm, scale=scale, out=out)
    assert n1.dtype == torch.float32 and n1.shape == ()
    assert all(map(torch.equal, grads, kept))                       # out of place: the gradients stay
    check(n1, out, kept, max_norm, scale)
    n2 = clip.clip_grad_norm_(grads, max_norm, scale=scale)         # in place: the same bits
    assert torch.equal(n1, n2) and all(map(torch.equal, grads, out))
    assert torch.equal(clip.grad_norm(kept, scale=scale), n1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_views_of_a_bucket_and_odd_addresses(dtype):
    sizes = [1, 2, 3, 5, 1023, 4097, 64, 20001]
    src, dst = torch.randn(sum(sizes) + 1, device="cuda").to(dtype), torch.zeros(sum(sizes) + 3, device="cuda", dtype=dtype)
    a, b, at = [], [], 0
    for s in sizes:
        a.append(src[1 + at:1 + at + s])
        b.append(dst[at:at + s])
        at += s
    n = clip.clip_grad_norm_(a, 0.5, out=b)
    check(n, b, [x.clone() for x in a], 0.5, 1.0)
    assert not bool(dst[at:].any())                                 # what lies behind the last one is left as it was


@gpu
def test_strides():
    base = torch.randn(64, 96, device="cuda")
    grads = [base[:, :40], base[:, 40:96], torch.randn(30, 50, device="cuda").t(), torch.randn(4, 6, 5, 7, device="cuda").to(memory_format=torch.channels_last)]
    kept = [g.clone() for g in grads]
    out = [torch.zeros(64, 40, device="cuda"), torch.zeros(64, 200, device="cuda")[:, 3:59], torch.zeros(30, 50, device="cuda").t(),
           torch.zeros(4, 6, 5, 7, device="cuda").to(memory_format=torch.channels_last)]
    n = clip.clip_grad_norm_(grads, 2.0, out=out)
    check(n, out, kept, 2.0, 1.0)
    n2 = clip.clip_grad_norm_(grads, 2.0)
    check(n2, grads, kept, 2.0, 1.0)
    assert torch.equal(n, n2) and torch.equal(base[:, :40], out[0])
    wide = torch.ones(1, device="cuda").expand(100)                 # a broadcast gradient is read as the values it stands for
    assert float(clip.grad_norm([wide])) == 10.0
    with pytest.raises(ValueError):
        clip.clip_grad_norm_([wide], 1.0)                           # ... and cannot be clipped in place
    with pytest.raises(ValueError):
        clip.clip_grad_norm_([base[::2, ::2]], 1.0)
    with pytest.raises(ValueError):
        clip.clip_grad_norm_([torch.zeros(30, 50, device="cuda")], 1.0, out=[torch.zeros(50, 30, device="cuda").t()])


@gpu
def test_values_whose_squares_do_not_fit_float32():
    big = [torch.full((1000,), 1e30, device="cuda"), torch.full((77,), -3e37, device="cuda")]
    check(clip.clip_grad_norm_([g.clone() for g in big], 1.0), [], big, 1.0, 1.0)
    got = [g.clone() for g in big]
    check(clip.clip_grad_norm_(got, 1.0), got, big, 1.0, 1.0)
    small = [torch.full((1000,), 1e-30, device="cuda")]
    assert abs(float(clip.grad_norm(small)) / (float(small[0][0]) * math.sqrt(1000)) - 1) < 1e-6


@gpu
def test_what_is_not_finite_is_not_hidden():
    a = [torch.ones(5000, device="cuda"), torch.ones(3, device="cuda")]
    a[0][4999] = float("nan")
    n = clip.clip_grad_norm_(a, 0.5)
    assert math.isnan(float(n)) and bool(torch.isnan(a[0]).all()) and bool(torch.isnan(a[1]).all())
    a = [torch.ones(5000, device="cuda"), torch.ones(3, device="cuda")]
    a[1][0] = float("inf")
    n = clip.clip_grad_norm_(a, 0.5)
    assert math.isinf(float(n)) and not bool(a[0].any()) and math.isnan(float(a[1][0])) and float(a[1][1]) == 0.0


@gpu
def test_more_than_32_bits_of_values():
    """a tensor of more than 2^31 values (2^32 bytes), and rows of one further apart than that in all"""
    n = 2 ** 31 + 77
    g = torch.full((n,), 0.25, device="cuda", dtype=torch.bfloat16)
    g[-1] = 3.0
    norm = clip.clip_grad_norm_([g], 1.0)
    true = math.sqrt((n - 1) * 0.0625 + 9.0)
    assert abs(float(norm) - true) <= 2.0 ** -23 * true
    want = torch.tensor([0.25 / true, 3.0 / true], dtype=torch.float64)
    got = torch.stack([g[0], g[-1]]).double().cpu()
    assert bool(((got - want).abs() <= want * (2.0 ** -8 + 2.0 ** -22)).all()) and bool((g[:-1] == g[0]).all())
    rows = g[:2 ** 31].view(2 ** 11, 2 ** 20)[:, 5:9]
    rows.fill_(2.0)
    assert abs(float(clip.grad_norm([rows])) - math.sqrt(4.0 * 4 * 2 ** 11)) <= 2.0 ** -23 * 200
    clip.clip_grad_norm_([rows], 0.0)
    assert not bool(rows.any()) and float(g[4]) == float(g[0]) and float(g[9]) == float(g[0])


@gpu
def test_zero_gradients_and_a_zero_bound():
    z = [torch.zeros(100, device="cuda"), torch.zeros(0, device="cuda")]
    assert float(clip.clip_grad_norm_(z, 0.0)) == 0.0 and not bool(z[0].any())
    o = [torch.ones(100, device="cuda")]
    assert float(clip.clip_grad_norm_(o, 0.0)) == 10.0 and not bool(o[0].any())
    assert float(clip.grad_norm([torch.zeros(0, device="cuda")])) == 0.0
    assert float(clip.clip_grad_norm_([torch.zeros(0, device="cuda")], 1.0)) == 0.0
    u = torch.ones(4, device="cuda")
    assert float(clip.clip_grad_norm_(u, 2.0)) == 2.0 and bool((u == 1).all())      # exactly at the bound: not touched; a single tensor


@gpu
def test_captured_and_replayed_and_side_streams():
    grads = make([(1000,), (37, 9), (50001,)], [torch.float32, torch.bfloat16])
    out = [torch.zeros_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip.clip_grad_norm_(grads, 0.5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for bound in (0.5, 3.0):
        g = torch.cuda.CUDAGraph()
        o = [torch.zeros_like(x) for x in grads]
        with torch.cuda.graph(g):
            n = clip.clip_grad_norm_(grads, bound, out=o)
        graphs.append((g, n, o, bound))
    for k in range(4):
        for x, y in zip(grads, make([(1000,), (37, 9), (50001,)], [torch.float32, torch.bfloat16], seed=30 + k)):
            x.copy_(y)
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, n, o, bound in graphs:
            want = [torch.zeros_like(x) for x in grads]
            assert torch.equal(n, clip.clip_grad_norm_(grads, bound, out=want)) and all(map(torch.equal, o, want))


@gpu
def test_autograd_learns_of_the_write_and_inference_tensors_are_taken():
    x = torch.randn(10, device="cuda", requires_grad=True)
    y = x * 2
    z = y.exp()                                                     # saves its result
    clip.clip_grad_norm_([z.detach()], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.sum().backward()
    with torch.inference_mode():
        g = torch.full((16,), 2.0, device="cuda")
        assert float(clip.clip_grad_norm_([g], 4.0)) == 8.0 and bool((g == 1.0).all())


@gpu
def test_the_same_tensor_twice_and_overlaps_are_refused():
    g = torch.randn(100, device="cuda")
    with pytest.raises(_lib.Q1EnvError, match="overlap"):
        clip.clip_grad_norm_([g, g], 1.0)
    with pytest.raises(_lib.Q1EnvError, match="overlap"):
        clip.clip_grad_norm_([g[:60], g[50:]], 1.0)
    with pytest.raises(_lib.Q1EnvError, match="overlap"):
        clip.clip_grad_norm_([g[:50]], 1.0, out=[g[10:60]])
    assert float(clip.grad_norm([g, g])) == pytest.approx(math.sqrt(2) * float(g.double().norm()), rel=1e-6)       # reading twice is fine
    o = [torch.zeros(60, device="cuda"), torch.zeros(50, device="cuda")]
    clip.clip_grad_norm_([g[:60], g[50:]], 1.0, out=o)


# ---- refusals: no GPU needed

def test_refuses_what_it_does_not_take():
    t = torch.zeros(3)
    with pytest.raises(_lib.Q1EnvError):
        clip.clip_grad_norm_([t], 1.0)
    with pytest.raises(TypeError):
        clip.clip_grad_norm_([torch.zeros(3, dtype=torch.float64)], 1.0)
    with pytest.raises(TypeError):
        clip.clip_grad_norm_([t, None], 1.0)
    with pytest.raises(ValueError):
        clip.clip_grad_norm_([], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            clip.clip_grad_norm_([t], bad)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            clip.clip_grad_norm_([t], 1.0, scale=bad)
    with pytest.raises(ValueError):
        clip.clip_grad_norm_([t], 1.0, out=[t, t])
    with pytest.raises(TypeError):
        clip.clip_grad_norm_([t], 1.0, out=[t.half()])
    with pytest.raises(ValueError):
        clip.clip_grad_norm_([t], 1.0, out=[torch.zeros(4)])


@pytest.mark.parametrize("shape,strides,want", [((4, 5), (5, 1), (0, 0)), ((5, 4), (1, 5), (0, 0)), ((4, 5), (9, 1), (5, 9)), ((4, 5), (10, 2), (1, 2)), ((3,), (0,), None), ((7,), (1,), (0, 0)),
                                                ((1, 5), (77, 1), (0, 0)), ((2, 3, 4), (24, 8, 1), (4, 8)), ((2, 3, 4), (30, 8, 1), None), ((), (), (0, 0)), ((4, 5), (3, 1), None)])
def test_layouts(shape, strides, want):
    t = torch.zeros(200).as_strided(shape, strides)
    assert clip._pitched(t) == want


def call(lib, src, dst, values, **kw):
    n = len(src)
    a = dict(dtype=[0] * n, cols=None, sp=None, dp=None, scale=1.0, max_norm=1.0, norm=4096, ws=4096, nbytes=1 << 20)
    a.update(kw)
    arr = lambda x, t: None if x is None else np.array(x, t)  # noqa: E731
    keep = [arr(src, np.uint64), arr(dst, np.uint64), arr(values, np.int64), arr(a["dtype"], np.int32), arr(a["cols"], np.int64), arr(a["sp"], np.int64), arr(a["dp"], np.int64)]
    return lib.q1env_grad_clip(0, None, n, *[_lib.ptr(x) for x in keep], a["scale"], a["max_norm"], a["norm"], a["ws"], a["nbytes"])


def test_the_library_refuses():
    lib = _lib.load()
    ok = dict(src=[4096, 8192], dst=[4096, 8192], values=[10, 10])
    for kw in (dict(dtype=[0, 3]), dict(values=[-1, 10]), dict(values=[1 << 41, 10]), dict(src=[0, 8192]), dict(dst=[4096, 0]), dict(src=[4097, 8192]), dict(scale=0.0), dict(scale=float("inf")),
               dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(norm=None), dict(ws=None), dict(nbytes=8), dict(cols=[3, 0], sp=[3, 0], dp=[3, 0]), dict(cols=[5, 0], sp=[4, 0], dp=[5, 0]),
               dict(cols=[5, 0], sp=[5, 0], dp=[4, 0]), dict(cols=[5, 0]), dict(dst=[4096, 4100]), dict(dst=[4096, 4096]), dict(dst=[4100, 8192]), dict(dst=[8192, 12288])):
        args = dict(ok)
        args.update(kw)
        assert call(lib, **args) == -1, kw
    # a destination over another tensor's source, and interleaved columns that do touch
    assert call(lib, src=[4096, 8192], dst=[16384, 4096], values=[10, 10]) == -1
    assert call(lib, src=[4096, 4096 + 12], dst=[4096, 4096 + 12], values=[20, 20], cols=[4, 4], sp=[10, 10], dp=[10, 10]) == -1
    assert b"overlap" in lib.q1env_last_error()
    assert lib.q1env_grad_norm_workspace_bytes(-1) == 0 and lib.q1env_grad_norm_workspace_bytes(12) > 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_factors_outside_float32s_range(dtype):
    """A norm past float32's largest value is reported as inf, but the gradients are clipped by it as by any other: the factor, below float32's normal range here (and above it for
    the tiny gradients), keeps its bits.  A value is one float64 product, a rounding to float32 and one to the type."""
    tol = 2.0 ** -24 + HALF[dtype] + 2.0 ** -40
    for n, amp, scale, bound in ((1_000_003, 3e38, 1.0, 0.5), (5, 2.5e38, 1.0, 1e-6), (3001, 1e-30, 1e40, 1e300), (3001, 1e-35, 1e42, 1e5)):
        g = torch.full((n,), amp, device="cuda").to(dtype)
        a = float(g[0])
        norm = math.sqrt(n) * a * scale
        want = a * scale * min(1.0, bound / norm)
        for pitched in (False, True):
            src = torch.zeros(n, 3, device="cuda", dtype=dtype)[:, 1:2] if pitched else torch.empty(n, 1, device="cuda", dtype=dtype)
            src.copy_(g[:, None])
            got = clip.clip_grad_norm_([src], bound, scale=scale)
            assert (math.isinf(float(got)) if norm > 3.5e38 else abs(float(got) / norm - 1) <= 2.0 ** -23)
            assert bool(((src.double() - want).abs() <= want * tol).all()), (n, amp, float(src[0, 0]), want)


def test_refuses_forward_mode_tangents():
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        x = fwad.make_dual(torch.ones(3), torch.ones(3))
        for f in (lambda: clip.grad_norm([torch.ones(2), x]), lambda: clip.clip_grad_norm_([x], 1.0), lambda: clip.clip_grad_norm_([x], 1.0, out=[torch.zeros(3)])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()


@gpu
def test_results_carry_no_graph():
    x = torch.randn(50, device="cuda", requires_grad=True)
    g = x * 3.0
    out = [torch.zeros(50, device="cuda")]
    assert not clip.grad_norm([g]).requires_grad and not clip.clip_grad_norm_([g], 1.0, out=out).requires_grad and not out[0].requires_grad


@gpu
def test_autograd_learns_of_the_write_beside_inference_tensors():
    """a list that begins with a tensor made in inference mode: the others' versions count all the same"""
    with torch.inference_mode():
        first = torch.full((16,), 2.0, device="cuda")
    x = torch.randn(10, device="cuda", requires_grad=True)
    z = (x * 2).exp()
    clip.clip_grad_norm_([first, z.detach()], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.sum().backward()
    out = [torch.zeros(16, device="cuda"), torch.zeros(10, device="cuda")]
    before = out[1]._version
    clip.clip_grad_norm_([first, x.detach()], 0.1, out=out)
    assert out[1]._version > before


def test_the_library_refuses_a_norm_or_workspace_over_a_tensor():
    lib = _lib.load()
    a, b, ws, norm = 1 << 20, 1 << 21, 1 << 24, 1 << 23

    def norm_only(src, values, **kw):
        k = dict(norm=norm, ws=ws, cols=None, sp=None, device=0)
        k.update(kw)
        arr = lambda x, t: None if x is None else np.array(x, t)  # noqa: E731
        keep = [arr(src, np.uint64), arr(values, np.int64), arr([0] * len(src), np.int32), arr(k["cols"], np.int64), arr(k["sp"], np.int64)]
        return lib.q1env_grad_norm(k["device"], None, len(src), *[_lib.ptr(x) for x in keep], 1.0, k["norm"], k["ws"], 1 << 20)
    for kw in (dict(norm=a + 36), dict(ws=a - 16), dict(norm=b), dict(norm=ws + 16)):
        assert call(lib, src=[a, b], dst=[a, b], values=[10, 10], **{"ws": ws, "norm": norm, **kw}) == -1 and b"the norm or the workspace" in lib.q1env_last_error(), kw
        assert norm_only([a, b], [10, 10], **kw) == -1 and b"the norm or the workspace" in lib.q1env_last_error(), kw
    assert call(lib, src=[a], dst=[b], values=[10], ws=ws, norm=b + 4) == -1 and b"the norm or the workspace" in lib.q1env_last_error()
    assert norm_only([a], [20], cols=[4], sp=[10], norm=a + 12) == -1 and b"the norm or the workspace" in lib.q1env_last_error()
    # beside them: on to the next check (no such device)
    for kw in (dict(src=[a, b], values=[10, 10], norm=a + 40), dict(src=[a, 0], values=[10, 0])):
        assert norm_only(device=99, **kw) != 0 and b"the norm or the workspace" not in lib.q1env_last_error()


def test_lazily_negated_views_are_not_taken_for_their_memory():
    """the imaginary part of a conjugate holds the opposite of what its memory does"""
    x = torch.randn(5, 3, dtype=torch.complex64).conj().imag
    assert x.is_neg()
    with pytest.raises(ValueError, match="negated"):
        clip._layouts([x], [torch.zeros(5, 6)[:, ::2]])
    with pytest.raises(ValueError, match="negated"):
        clip._layouts([torch.zeros(5, 6)[:, ::2]], [x])
    clip._layouts([x], None)                                        # in place a factor commutes with the sign
