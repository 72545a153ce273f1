"""The wide categorical head (q1physrl_amd/categorical.py, q1env_head_*): against the definition in float64, at the sizes, masks, strides and types
where tiles end, and its refusals (those need no GPU).

Tolerances, from the arithmetic alone (u = 2^-24, float32's half step; ut = the type's half step):
  a logit: D products and sums in float32, the accumulator possibly truncating: at most (D + 8) 2u S with S = sum_k |h_k w_k| + |b| -> el
  log-sum-exp: the largest el, the sum of the exponentials with at most 256 + V / 2048 additions in a chain and one exponential of 4u per term,
    the logarithm and the final sums at their own magnitude: el + (256 + V / 2048 + 16) 2u + 8u |lse|
  log-probability: that and el again; entropy: each p (log p) to the relative error e of p plus the error of log p
  a gradient of a logit: its parts to e relative, and half a step ut of the type it is stored in (float32: 2^-24); a product over K of them: (K + 8) 2u of
    the sum of the absolute products more, half a step ut of the result, and in float16 the subnormal step 2^-25 of the result and of the scaled store."""
import ctypes as C
import math

import pytest
import torch

from q1physrl_amd import _lib, categorical

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
IGN = -100
gpu = pytest.mark.gpu


def make(n, d, v, dtype, bias=True, seed=0, ignored=0.1, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.tanh(torch.randn(n, d, device="cuda", generator=g)).to(dtype)
    w = (torch.randn(v, d, device="cuda", generator=g) * (spread / math.sqrt(d))).to(dtype)
    b = torch.randn(v, device="cuda", generator=g).to(dtype) if bias else None
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    t[torch.rand(n, device="cuda", generator=g) < ignored] = IGN
    return h, w, b, t


class Truth:
    """The definition in float64, and how far each result may be off."""

    def __init__(self, h, w, b, t, ignore=IGN):
        self.dtype, self.d, self.v = h.dtype, h.shape[1], w.shape[0]
        self.ok = t != ignore
        self.t = torch.where(self.ok, t.long(), 0)
        self.h = torch.where(self.ok[:, None], h.detach().double(), 0.0)       # what an ignored row holds does not matter
        self.w = w.detach().double()
        self.b = torch.zeros(self.v, dtype=torch.float64, device=h.device) if b is None else b.detach().double()
        z = self.h @ self.w.T + self.b
        self.lse = torch.logsumexp(z, 1)
        self.lp = z - self.lse[:, None]
        self.p = self.lp.exp()
        self.lp = torch.where(self.p > 0, self.lp, 0.0)                        # a class at -inf takes no part
        self.logp = torch.where(self.ok, z.gather(1, self.t[:, None])[:, 0] - self.lse, 0.0)
        self.entropy = torch.where(self.ok, -(self.p * self.lp).sum(1), 0.0)
        fin = torch.where(torch.isfinite(self.b), self.b.abs(), 0.0)
        self.el = ((self.d + 8) * 2 * U * (self.h.abs() @ self.w.abs().T + fin)).amax(1)
        self.elogp = 2 * self.el + (256 + self.v / 2048 + 16) * 2 * U + 8 * U * (self.lse.abs() + self.logp.abs() + 1)
        self.e = 2 * self.elogp                                                # relative error of a probability
        self.eent = self.e * (self.p * (self.lp.abs() + 1)).sum(1) + self.elogp

    def grads(self, A, E):
        """(dh, dw, db) and their tolerances for upstream A = d/dlogp, E = d/dentropy (rows)."""
        A, E = (torch.where(self.ok, x.double(), 0.0) for x in (A, E))
        g = -self.p * (A[:, None] + E[:, None] * (self.lp + self.entropy[:, None]))
        g.scatter_add_(1, self.t[:, None], A[:, None])
        size = self.p * (A.abs()[:, None] + E.abs()[:, None] * (self.lp.abs() + self.entropy[:, None] + 1))
        ut = HALF[self.dtype]
        n = self.h.shape[0]
        off = size * self.e[:, None] + g.abs() * ut + 4 * U * size.scatter_add(1, self.t[:, None], A.abs()[:, None])
        if self.dtype == torch.float16:                                        # the scaled store's smallest step: at most 2^-25 of 2^-13 of the largest bound
            off = off + torch.where(self.ok, 2.0 ** -38 * (A.abs() + 16 * E.abs()).max(), 0.0)[:, None]
        tiny = 2.0 ** -25 if self.dtype == torch.float16 else 0.0

        def tol(k, err, size_, ref):
            return err * (1 + 1e-3) + (k + 8) * 2 * U * size_ + ut * ref.abs() * 1.01 + tiny + 1e-30
        dh, dw, db = g @ self.w, g.T @ self.h, g.sum(0)
        return ((dh, tol(self.v, off @ self.w.abs(), (g.abs() + off) @ self.w.abs(), dh)), (dw, tol(n, off.T @ self.h.abs(), (g.abs() + off).T @ self.h.abs(), dw)),
                (db, tol(n, off.sum(0), (g.abs() + off).sum(0), db)))


def near(got, ref, tol, what):
    got = got.detach().double()
    assert got.shape == ref.shape, what
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - ref).abs() - tol
    assert float(over.max() if over.numel() else -1.0) <= 0.0, f"{what}: {float((got - ref).abs().max()):.3g} off, {float(over.max()):.3g} over what the arithmetic allows"


SIZES = [(1, 1, 1), (1, 16, 2), (3, 5, 7), (1, 256, 721), (33, 64, 129), (127, 256, 361), (130, 200, 1000), (257, 72, 65), (64, 128, 5003), (5, 1000, 300), (2001, 40, 34),
         (700, 264, 520), (300, 65, 255), (256, 64, 256)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_rows_and_gradients(n, d, v, dtype):
    h, w, b, t = make(n, d, v, dtype, bias=(n % 2 == 1), seed=n + v)
    leaves = [x.requires_grad_() for x in (h, w, b) if x is not None]
    logp, ent = categorical.linear_categorical(h, w, t, b)
    assert logp.dtype == ent.dtype == torch.float32
    T = Truth(h, w, b, t)
    near(logp, T.logp, T.elogp, "logp")
    near(ent, T.entropy, T.eent, "entropy")
    g = torch.Generator(device="cuda").manual_seed(7)
    A, E = torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g) * 0.1
    got = torch.autograd.grad((logp, ent), leaves, (A, E))
    ref = T.grads(A, E)
    for name, x, (r, tol) in zip(("dh", "dw", "db"), got, ref):
        assert x.dtype == dtype
        near(x, r, tol, name)
    assert bool((got[0][t == IGN] == 0).all()) and bool((logp[t == IGN] == 0).all()) and bool((ent[t == IGN] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(20001, 72, 2049), (3000, 136, 2100), (1500, 300, 9000), (5000, 520, 3000), (2047, 1001, 8200), (4100, 1024, 5000), (8200, 1040, 8300), (70, 4095, 60000), (400, 4094, 45000)])
def test_sizes_of_every_tile(n, d, v, dtype):
    """sizes at which every tile, whole and split sums, and both backward products together and apart take their turn, with partial tiles on every side; and laid-out
    weights of every type in several pieces"""
    h, w, b, t = make(n, d, v, dtype, seed=v, ignored=0.2)
    h = torch.where((t == IGN)[:, None], float("nan"), h)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    logp, ent = categorical.linear_categorical(h, w, t, b)
    T = Truth(h, w, b, t)
    near(logp, T.logp, T.elogp, "logp")
    near(ent, T.entropy, T.eent, "entropy")
    g = torch.Generator(device="cuda").manual_seed(9)
    A, E = torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g) * 0.1
    for name, x, (r, tol) in zip(("dh", "dw", "db"), torch.autograd.grad((logp, ent), leaves, (A, E)), T.grads(A, E)):
        near(x, r, tol, name)
    loss, *got = categorical.linear_cross_entropy_grad(h, w, t, b)
    k = T.ok.double().sum()
    near(loss, -T.logp.sum() / k, (T.elogp * T.ok).sum() / k + 2 * U * T.logp.abs().sum() / k, "loss")
    for name, x, (r, tol) in zip(("dh", "dw", "db"), got, T.grads((-1.0 / k).expand(n), torch.zeros(n, device="cuda"))):
        near(x, r, tol, name)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(1, 16, 3), (200, 256, 361), (129, 100, 1025)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy(n, d, v, dtype, reduction):
    h, w, b, t = make(n, d, v, dtype, seed=3)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    loss = categorical.linear_cross_entropy(h, w, t, b, reduction=reduction)
    T = Truth(h, w, b, t)
    live = T.ok.double()
    count = live.sum().clamp(min=1)
    if reduction == "none":
        near(loss, -T.logp, T.elogp, "loss")
        up = torch.linspace(0.5, 1.5, n, device="cuda")
        A = -up
    else:
        k = count if reduction == "mean" else torch.ones((), device="cuda", dtype=torch.float64)
        near(loss, -T.logp.sum() / k, (T.elogp * live).sum() / k + 2 * U * T.logp.abs().sum() / k, "loss")
        up = torch.tensor(0.75, device="cuda")
        A = (-0.75 / k).expand(n)
    got = torch.autograd.grad(loss, leaves, up)
    for name, x, (r, tol) in zip(("dh", "dw", "db"), got, T.grads(A, torch.zeros(n, device="cuda"))):
        near(x, r, tol, name)
    if reduction != "none":
        l2, dh, dw, db = categorical.linear_cross_entropy_grad(h, w, t, b, reduction=reduction, grad_scale=up)
        assert torch.equal(l2, loss.detach()) and all(map(torch.equal, (dh, dw, db), got))


@gpu
def test_pieces_of_the_classes_and_splits():
    """more classes x rows than one piece holds (float32: 256 MiB), and a sum split over many workgroups"""
    n, d, v = 30000, 24, 3000
    h, w, b, t = make(n, d, v, torch.float32)
    T = Truth(h, w, b, t)
    loss, dh, dw, db = categorical.linear_cross_entropy_grad(h, w, t, b)
    live = T.ok.double()
    near(loss, -T.logp.sum() / live.sum(), (T.elogp * live).mean() + 4 * U * T.logp.abs().mean(), "loss")
    for name, x, (r, tol) in zip(("dh", "dw", "db"), (dh, dw, db), T.grads((-1.0 / live.sum()).expand(n), torch.zeros(n, device="cuda"))):
        near(x, r, tol, name)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_what_padding_rows_hold_does_not_matter(dtype):
    h, w, b, t = make(150, 96, 333, dtype, seed=5, ignored=0.3)
    a = categorical.linear_cross_entropy_grad(h, w, t, b)
    bad = h.clone()
    bad[t == IGN] = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dtype, device="cuda").repeat(32)
    c = categorical.linear_cross_entropy_grad(bad, w, t, b)
    assert all(map(torch.equal, a, c))
    h2 = bad.requires_grad_()
    logp, ent = categorical.linear_categorical(h2, w, t, b)
    (g,) = torch.autograd.grad((logp, ent), (h2,), (torch.ones_like(logp), torch.ones_like(ent)))
    assert bool(torch.isfinite(logp).all() & torch.isfinite(ent).all() & torch.isfinite(g).all()) and bool((g[t == IGN] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_all_rows_ignored_and_no_rows(dtype):
    h, w, b, t = make(40, 32, 70, dtype)
    loss, dh, dw, db = categorical.linear_cross_entropy_grad(h, w, torch.full_like(t, IGN), b)
    assert float(loss) == 0.0 and not any(bool(x.any()) for x in (dh, dw, db))
    e = h[:0].requires_grad_()
    w.requires_grad_(), b.requires_grad_()
    loss = categorical.linear_cross_entropy(e, w, t[:0], b)
    gs = torch.autograd.grad(loss, (e, w, b))
    assert float(loss) == 0.0 and gs[0].shape == (0, 32) and not bool(gs[1].any()) and not bool(gs[2].any())
    logp, ent = categorical.linear_categorical(e, w, t[:0], b)
    assert logp.shape == ent.shape == (0,)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_masked_classes(dtype):
    """a bias of -inf takes a class out; the type's lowest value does the same to rounding; whole tiles of them, and a row's own class"""
    n, d, v = 60, 64, 700
    h, w, b, t = make(n, d, v, dtype, seed=11, ignored=0.0)
    b[128:400] = -float("inf")
    b[500] = -float("inf")
    t = torch.where((t >= 128) & (t < 400) | (t == 500), 3, t)
    T = Truth(h, w, b, t)
    loss, dh, dw, db = categorical.linear_cross_entropy_grad(h, w, t, b)
    for name, x, (r, tol) in zip(("dh", "dw", "db"), (dh, dw, db), T.grads(torch.full((n,), -1.0 / n, device="cuda"), torch.zeros(n, device="cuda"))):
        near(x, r, tol, name)
    assert not bool(dw[128:400].any()) and not bool(db[128:400].any())
    logp, ent = categorical.linear_categorical(h, w, t, b)
    near(logp, T.logp, T.elogp, "logp")
    near(ent, T.entropy, T.eent, "entropy")
    low = b.clone()
    low[torch.isinf(low)] = torch.finfo(dtype).min
    logp2, ent2 = categorical.linear_categorical(h, w, t, low)
    near(logp2, T.logp, T.elogp, "logp, lowest value")
    near(ent2, T.entropy, T.eent, "entropy, lowest value")
    own = t.clone()
    own[0] = 200                                                              # a class that takes no part: no chance at all
    assert float(categorical.linear_categorical(h, w, own, b)[0][0]) == -float("inf")
    nothing = torch.full_like(b, -float("inf"))
    assert bool(torch.isnan(categorical.linear_categorical(h, w, t, nothing)[0]).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n,d,v", [(2, 73, 2), (1, 64, 40), (31, 48, 70), (60, 200, 130), (100, 64, 300), (256, 136, 257)])
def test_few_rows_of_16_bits_keep_the_gradient_finer_than_their_type(n, d, v, dtype):
    """The few roundings of a gradient of few rows need not even out, so it is held in two pieces: ut^2 of it is lost, not ut (ut the type's half step), and the results are off by
    their own rounding and what float32 leaves: the bounds of the other tests with ut^2 for the stored gradient."""
    h, w, b, t = make(n, d, v, dtype, seed=n, ignored=0.0)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    got = torch.autograd.grad(categorical.linear_categorical(h, w, t, b), leaves, (torch.ones(n, device="cuda"), torch.full((n,), 0.25, device="cuda")))
    T = Truth(h, w, b, t)
    A, E = torch.ones(n, device="cuda", dtype=torch.float64), torch.full((n,), 0.25, device="cuda", dtype=torch.float64)
    g = -T.p * (A[:, None] + E[:, None] * (T.lp + T.entropy[:, None]))
    g.scatter_add_(1, T.t[:, None], A[:, None])
    size = T.p * (1 + 0.25 * (T.lp.abs() + T.entropy[:, None] + 1))
    ut = HALF[dtype]
    # the second piece's smallest step in float16: half of 2^-24 at a scale that brings the largest possible value to 2^13 at least
    off = size * T.e[:, None] + g.abs() * ut * ut + 4 * U * (size + g.abs()) + (2.0 ** -38 * 5 if dtype == torch.float16 else 0.0)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for name, x, ref, err, part, k in (("dh", got[0], g @ T.w, off @ T.w.abs(), g.abs() @ T.w.abs(), 2 * v), ("dw", got[1], g.T @ T.h, off.T @ T.h.abs(), g.abs().T @ T.h.abs(), 2 * n)):
        near(x, ref, err * 1.01 + (k + 8) * 2 * U * (part + err) + ut * ref.abs() * 1.01 + tiny, name)


SKINNY = [(1, 1, 1), (5, 3, 2), (9, 4, 3), (1, 7, 33), (2, 300, 31), (31, 130, 1000), (32, 64, 32), (32, 1000, 4099), (33, 61, 32), (500, 8, 1), (1000, 257, 15), (3001, 128, 32), (700, 2171, 5), (33, 70, 33)]


@gpu
@pytest.mark.parametrize("n,d,v", SKINNY)
@pytest.mark.parametrize("how", ["whole", "views", "odd"])
def test_few_rows_or_classes_of_float32(n, d, v, how):
    """At most 32 rows or classes of float32 are read straight from memory: whole rows, rows with a pitch (in and out), and rows that start at any 4 bytes."""
    h, w, b, t = make(n, d, v, torch.float32, seed=n + d + v)
    if how != "whole":
        pad = 4 if how == "views" else 3

        def laid(x):
            wide = torch.full((x.shape[0], x.shape[1] + 2 * pad), float("nan"), device="cuda")
            wide[:, pad:pad + x.shape[1]] = x
            return wide[:, pad:pad + x.shape[1]]
        h, w = laid(h), laid(w)
    if n > 1 and bool((t != IGN).any()):
        dead = (t == IGN).nonzero()[:, 0]
        h[dead] = float("nan")                                                 # what ignored rows hold
    leaves = [x.requires_grad_() for x in (h, w, b)]
    logp, ent = categorical.linear_categorical(h, w, t, b)
    T = Truth(h, w, b, t)
    near(logp, T.logp, T.elogp, "logp")
    near(ent, T.entropy, T.eent, "entropy")
    g = torch.Generator(device="cuda").manual_seed(5)
    A, E = torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g)
    for entropy in (True, False):
        if entropy:
            got = torch.autograd.grad((logp, ent), leaves, (A, E), retain_graph=True)
        else:
            got = torch.autograd.grad(logp, leaves, A)
        for name, x, (r, tol) in zip(("dh", "dw", "db"), got, T.grads(A, E if entropy else torch.zeros_like(E))):
            near(x, r, tol, name)
        assert bool((got[0][t == IGN] == 0).all())


@gpu
@pytest.mark.parametrize("n,d,v", [(20, 64, 700), (300, 64, 31), (1, 36, 90)])
def test_masked_classes_of_few_rows_or_classes(n, d, v):
    h, w, b, t = make(n, d, v, torch.float32, seed=4, ignored=0.0)
    off = torch.zeros(v, dtype=torch.bool, device="cuda")
    off[3:v // 2] = True
    off[v - 1] = True
    t = torch.where(off[t], 1, t)
    for low in (-float("inf"), torch.finfo(torch.float32).min):
        bias = torch.where(off, low, b)
        T = Truth(h, w, torch.where(off, -float("inf"), b), t)
        logp, ent = categorical.linear_categorical(h, w, t, bias)
        near(logp, T.logp, T.elogp, "logp")
        near(ent, T.entropy, T.eent, "entropy")
        leaves = [x.clone().requires_grad_() for x in (h, w, bias)]
        A, E = torch.linspace(-1, 1, n, device="cuda"), torch.linspace(0.5, 0.1, n, device="cuda")
        got = torch.autograd.grad(categorical.linear_categorical(leaves[0], leaves[1], t, leaves[2]), leaves, (A, E))
        for name, x, (r, tol) in zip(("dh", "dw", "db"), got, T.grads(A, E)):
            near(x, r, tol, name)
        assert not bool(got[1][off].any()) and not bool(got[2][off].any())
    nothing = torch.full_like(b, -float("inf"))
    assert bool(torch.isnan(categorical.linear_categorical(h, w, t, nothing)[0]).all())


@gpu
@pytest.mark.parametrize("bad", [-1, 700, 2 ** 40])
def test_classes_that_do_not_exist_are_nan(bad):
    h, w, b, t = make(20, 64, 700, torch.float32, ignored=0.0)
    good = categorical.linear_categorical(h, w, t, b)
    t2 = t.clone()
    t2[7] = bad
    h.requires_grad_()
    logp, ent = categorical.linear_categorical(h, w, t2, b)
    keep = torch.arange(20, device="cuda") != 7
    assert math.isnan(float(logp[7])) and math.isnan(float(ent[7])) and torch.equal(logp[keep], good[0][keep]) and torch.equal(ent[keep], good[1][keep])
    (dh,) = torch.autograd.grad(logp.sum(), h)
    assert bool(torch.isnan(dh[7]).all()) and bool(torch.isfinite(dh[keep]).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d", [64, 61, 8])
def test_strides_and_alignment(dtype, d):
    """rows at a pitch, a base address one element off, a transposed weight (copied), leading dimensions, int32 classes"""
    n, v = 77, 190
    h, w, b, t = make(n, d, v, dtype, seed=2)
    ref = categorical.linear_cross_entropy_grad(h, w, t, b)
    wide = torch.zeros(n, 2 * d + 3, dtype=dtype, device="cuda")
    wide[:, 1:d + 1] = h
    flat = torch.zeros(v * d + 1, dtype=dtype, device="cuda")
    flat[1:] = w.reshape(-1)
    b1 = torch.zeros(v + 1, dtype=dtype, device="cuda")
    b1[1:] = b
    for args in ((wide[:, 1:d + 1], w, t, b), (h, flat[1:].view(v, d), t, b), (h, w.t().contiguous().t(), t, b1[1:]), (wide[:, 1:d + 1], flat[1:].view(v, d), t.int(), b1[1:])):
        got = categorical.linear_cross_entropy_grad(*args)
        assert all(map(torch.equal, got, ref))
    got = categorical.linear_cross_entropy_grad(h.view(7, 11, d), w, t.view(7, 11), b)
    assert got[1].shape == (7, 11, d) and torch.equal(got[1].view(n, d), ref[1]) and torch.equal(got[2], ref[2])
    logp, ent = categorical.linear_categorical(h.view(7, 11, d), w, t.view(7, 11), b)
    assert logp.shape == ent.shape == (7, 11)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_offsets_past_32_bits(dtype):
    """a weight of more than 2^32 bytes, and rows of hidden further apart than the loads into the LDS reach (they are laid out first)"""
    n, d, v = (40, 32776, 66001) if dtype == torch.bfloat16 else (33, 16392, 66001)
    g = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randn(v, d, device="cuda", generator=g, dtype=torch.float32) * (2.0 / math.sqrt(d))).to(dtype)
    h = torch.randn(n, d, device="cuda", generator=g).to(dtype)
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    t[:4] = torch.tensor([v - 1, v - 2, 0, IGN], device="cuda")
    z = torch.cat([h.double() @ c.double().T for c in w.split(4096)], 1)
    absz = torch.cat([h.double().abs() @ c.double().abs().T for c in w.split(4096)], 1)
    ok = t != IGN
    lse = torch.logsumexp(z, 1)
    el = ((d + 8) * 2 * U * absz).amax(1)
    logp = torch.where(ok, z.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse, 0.0)
    e = 2 * (2 * el + (256 + v / 2048 + 16) * 2 * U + 8 * U * (lse.abs() + logp.abs() + 1))
    loss, dh, dw, _ = categorical.linear_cross_entropy_grad(h, w, t)
    k = ok.double().sum()
    near(loss, -logp.sum() / k, (e / 2 * ok).sum() / k + 2 * U * logp.abs().sum() / k, "loss")
    p = torch.exp(z - lse[:, None])
    q = p.clone()
    q[ok.nonzero()[:, 0], t[ok]] -= 1.0
    q = torch.where(ok[:, None], q / k, 0.0)
    off = torch.where(ok[:, None], p * (e[:, None] + 4 * U) / k, 0.0) + (HALF[dtype] + 4 * U) * q.abs()
    for part in (slice(0, 64), slice(v - 64, v)):
        ref = q[:, part].T @ h.double()
        near(dw[part], ref, off[:, part].T @ h.double().abs() * 1.01 + (n + 8) * 2 * U * (q[:, part].abs().T @ h.double().abs()) + HALF[dtype] * ref.abs() * 1.01 + 1e-30, "dw")
    ref = sum(q[:, c0:c0 + 4096] @ w[c0:c0 + 4096].double() for c0 in range(0, v, 4096))
    size = sum(off[:, c0:c0 + 4096] @ w[c0:c0 + 4096].double().abs() for c0 in range(0, v, 4096))
    total = sum(q[:, c0:c0 + 4096].abs() @ w[c0:c0 + 4096].double().abs() for c0 in range(0, v, 4096))
    near(dh, ref, size * 1.01 + (v + 8) * 2 * U * total + HALF[dtype] * ref.abs() * 1.01 + 1e-30, "dh")
    del w, dw
    wide = torch.zeros(n, 2 ** 21 + 16, dtype=dtype, device="cuda")
    wide[:, 8:8 + 512] = h[:, :512]
    w2, b2 = torch.randn(300, 512, device="cuda", generator=g).to(dtype), None
    got, want = categorical.linear_cross_entropy_grad(wide[:, 8:520], w2, t % 300, b2), categorical.linear_cross_entropy_grad(h[:, :512].contiguous(), w2, t % 300, b2)
    assert all(torch.equal(x, y) for x, y in zip(got, want) if x is not None)


@gpu
def test_gradients_against_differences():
    """central differences of the float32 loss in float64-summed directions: step 2^-6 along a unit direction, third-order term and two roundings of the loss"""
    n, d, v = 40, 32, 50
    h, w, b, t = make(n, d, v, torch.float32, seed=9, ignored=0.2)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    c = torch.linspace(-1, 1, n, device="cuda")

    def f(h_, w_, b_):
        logp, ent = categorical.linear_categorical(h_, w_, t, b_)
        return (logp * c).double().sum() + 0.3 * ent.double().sum()
    grads = torch.autograd.grad(f(*leaves), leaves)
    step = 2.0 ** -6
    for i, g in enumerate(grads):
        gen = torch.Generator(device="cuda").manual_seed(i)
        u = torch.randn(g.shape, device="cuda", generator=gen)
        u = u / u.norm()
        with torch.no_grad():
            up, dn = ([x + s * step * u if k == i else x for k, x in enumerate(leaves)] for s in (1, -1))
            diff = float(f(*up) - f(*dn)) / (2 * step)
        want = float((g.double() * u.double()).sum())
        # the loss: n rows of about log(v) + |l| each to 2^-20; the third derivative of n rows along a unit direction is below n x 8 |h or w|^3 / n^0
        assert abs(diff - want) <= n * 8 * 2.0 ** -20 / (2 * step) + step * step / 6 * n * 8, (i, diff, want)


@gpu
def test_only_what_is_asked_for_and_partial_upstreams():
    h, w, b, t = make(90, 64, 200, torch.float32, seed=4)
    T = Truth(h, w, b, t)
    w.requires_grad_()
    logp, ent = categorical.linear_categorical(h, w, t, b)
    (dw,) = torch.autograd.grad(ent.sum(), (w,))
    r, tol = T.grads(torch.zeros(90, device="cuda"), torch.ones(90, device="cuda"))[1]
    near(dw, r, tol, "dw of the entropy alone")
    logp, ent = categorical.linear_categorical(h, w, t, b)
    (dw,) = torch.autograd.grad(logp.sum(), (w,))
    r, tol = T.grads(torch.ones(90, device="cuda"), torch.zeros(90, device="cuda"))[1]
    near(dw, r, tol, "dw of logp alone")
    with pytest.raises(RuntimeError):
        x = categorical.linear_cross_entropy(h, w, t, b)
        (g,) = torch.autograd.grad(x, (w,), create_graph=True)
        g.sum().backward()


@gpu
def test_same_bits_every_time_and_two_streams_at_once():
    h, w, b, t = make(500, 128, 3001, torch.bfloat16, seed=6)
    h2, w2, b2, t2 = make(333, 256, 900, torch.bfloat16, seed=8)
    ref, ref2 = categorical.linear_cross_entropy_grad(h, w, t, b), categorical.linear_cross_entropy_grad(h2, w2, t2, b2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    s1.wait_stream(torch.cuda.current_stream()), s2.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = categorical.linear_cross_entropy_grad(h, w, t, b)
        with torch.cuda.stream(s2):
            c = categorical.linear_cross_entropy_grad(h2, w2, t2, b2)
        torch.cuda.synchronize()
        assert all(map(torch.equal, a, ref)) and all(map(torch.equal, c, ref2))


@gpu
def test_captured_and_replayed():
    h, w, b, t = make(200, 64, 777, torch.float32, seed=1)
    other = make(200, 64, 777, torch.float32, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        categorical.linear_cross_entropy_grad(h, w, t, b)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                                       # two graphs of the same call share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = categorical.linear_cross_entropy_grad(h, w, t, b)
        graphs.append((g, out))
    with torch.no_grad():
        for k in range(4):
            src = other if k % 2 else make(200, 64, 777, torch.float32, seed=20 + k)
            for x, y in zip((h, w, b, t), src):
                x.copy_(y)
            want = categorical.linear_cross_entropy_grad(h, w, t, b)
            for g, out in graphs:
                g.replay()
            torch.cuda.synchronize()
            for g, out in graphs:
                assert all(map(torch.equal, out, want))
    w.requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="captured"):
            categorical.linear_cross_entropy(h, w, t, b)
        keep = torch.zeros(1, device="cuda")
    assert keep is not None


# ---- refusals: no GPU needed

def test_refuses_what_does_not_fit():
    h, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    f = categorical.linear_categorical
    for args, err in (((h, w.double(), t), TypeError), ((h.double(), w.double(), t), TypeError), ((h, w, t.float()), TypeError), ((h, w.bfloat16(), t), TypeError),
                      ((h, w[:, :7], t), ValueError), ((h, w[:0], t), ValueError), ((h, w, t[:3]), ValueError), ((h, w, t, torch.zeros(4)), ValueError),
                      ((h, w, t, torch.zeros(5, dtype=torch.float16)), TypeError), ((h, None, t), TypeError), ((h, w, t), _lib.Q1EnvError)):
        with pytest.raises(err):
            f(*args)
    with pytest.raises(ValueError):
        categorical.linear_cross_entropy(h, w, t, reduction="avg")
    with pytest.raises(ValueError):
        f(h, w, t, ignore_index=0.5)


def test_sizes_are_host_arithmetic():
    lib = _lib.load()
    assert lib.q1env_head_state_bytes(-1) == 0 and lib.q1env_head_state_bytes(2 ** 22 + 1) == 0 and lib.q1env_head_state_bytes(0) > 0
    ws = lib.q1env_head_workspace_bytes
    assert ws(0, 100, 64, 1000, 0) > 0 and ws(1, 100, 64, 1000, 1) > 0 and ws(2, 0, 64, 1000, 1) > 0
    for bad in ((3, 1, 1, 1), (0, -1, 1, 1), (0, 1, 0, 1), (0, 1, 2 ** 16 + 1, 1), (0, 1, 1, 0), (0, 1, 1, 2 ** 22 + 1), (0, 2 ** 22 + 1, 1, 1)):
        assert ws(*bad, 0) == 0
    # the logits are not in it: 8192 x 131072 float32 logits are 4.3 GB
    assert ws(1, 8192, 2048, 131072, 0) < 2 ** 28 and ws(1, 8192, 2048, 131072, 1) < 2 ** 30


def head(**kw):
    a = dict(dtype=0, target_bits=64, rows=4, width=8, classes=5, ignore_index=-100, hidden_dev=4096, hidden_stride=8, weight_dev=4096, weight_stride=8, bias_dev=None, target_dev=4096,
             state_dev=4096, ws_dev=4096, ws_bytes=1 << 30)
    a.update(kw)
    return _lib.Q1Head(*[a[k] for k, _ in _lib.Q1Head._fields_])


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(width=0), dict(classes=0), dict(hidden_dev=None), dict(weight_dev=None), dict(hidden_stride=7),
                                dict(weight_stride=7), dict(state_dev=None), dict(ws_dev=None), dict(ws_bytes=16), dict(target_bits=16), dict(target_dev=None), dict(hidden_dev=4097),
                                dict(rows=2 ** 22 + 1)])
def test_the_library_refuses(kw):
    lib = _lib.load()
    assert lib.q1env_head_forward(0, None, C.byref(head(**kw)), 0, 4096, None, None) == -1
    if not {"target_bits", "target_dev"} & set(kw):
        assert lib.q1env_head_backward(0, None, C.byref(head(**kw)), 4096, None, None, 4096, 8, None, 8, None) == -1


def test_the_library_refuses_results():
    lib = _lib.load()
    h = head()
    assert lib.q1env_head_forward(0, None, None, 0, 4096, None, None) == -1
    assert lib.q1env_head_forward(0, None, C.byref(h), 2, 4096, None, None) == -1
    assert lib.q1env_head_forward(0, None, C.byref(h), 0, None, None, None) == -1
    b = lib.q1env_head_backward
    assert b(0, None, C.byref(h), None, None, None, 4096, 8, None, 8, None) == -1           # no upstream gradient
    assert b(0, None, C.byref(h), 4096, None, 4096, 4096, 8, None, 8, None) == -1           # two kinds of it
    assert b(0, None, C.byref(h), 4096, None, None, None, 8, None, 8, None) == -1           # nothing asked for
    assert b(0, None, C.byref(h), 4096, None, None, 4096, 7, None, 8, None) == -1
    assert b(0, None, C.byref(h), 4096, None, None, None, 8, 4096, 7, None) == -1
    assert b(0, None, C.byref(h), 4096, None, None, 4098, 8, None, 8, None) == -1
    assert b"alignment" in lib.q1env_last_error() or b"aligned" in lib.q1env_last_error()


def test_the_library_refuses_overlaps_and_odd_addresses():
    """what a call writes may not overlap what it reads, its workspace or another result; rows of one pitch may interleave (that call goes on to the device)"""
    lib = _lib.load()
    rows, width, classes, base = 64, 8, 5, 1 << 24
    at = dict(hidden_dev=base, weight_dev=base + (1 << 16), bias_dev=base + (2 << 16), target_dev=base + (3 << 16), state_dev=base + (4 << 16), ws_dev=base + (1 << 20))
    free = base + (8 << 16)
    f, b = lib.q1env_head_forward, lib.q1env_head_backward

    def refused(rc, what):
        assert rc == -1 and what in lib.q1env_last_error(), (rc, lib.q1env_last_error())
    ok = head(rows=rows, width=width, classes=classes, **at)
    for p in (at["hidden_dev"], at["weight_dev"] + 4, at["bias_dev"], at["target_dev"] + 8, at["state_dev"] + 64, at["ws_dev"] + 16):
        refused(f(0, None, C.byref(ok), 0, p, None, None), b"overlaps")
        if p != at["target_dev"] + 8:
            refused(b(0, None, C.byref(ok), free, None, None, p, width, None, width, None), b"overlap")
    refused(f(0, None, C.byref(ok), 0, free, free + 4, None), b"overlap")
    refused(b(0, None, C.byref(ok), free, None, None, free, width, None, width, None), b"upstream")
    refused(b(0, None, C.byref(ok), free, None, None, free + 4096, width, free + 4096 + 4, width, None), b"two results")
    refused(f(0, None, C.byref(ok), 0, free + 2, None, None), b"aligned")
    refused(f(0, None, C.byref(head(rows=rows, width=width, classes=classes, **{**at, "ws_dev": at["ws_dev"] + 8})), 0, free, None, None), b"aligned")
    refused(f(0, None, C.byref(head(rows=rows, width=width, classes=classes, **{**at, "state_dev": at["ws_dev"] + 256})), 0, free, None, None), b"overlaps the workspace")
    refused(b(0, None, C.byref(ok), free + 1, None, None, free + 4096, width, None, width, None), b"aligned")
    pitched = head(rows=rows, width=width, classes=classes, **{**at, "hidden_stride": 2 * width})
    rc = b(99, None, C.byref(pitched), free, None, None, at["hidden_dev"] + 4 * width, 2 * width, None, width, None)
    assert rc != 0 and b"overlap" not in lib.q1env_last_error()                # (no such device)
    refused(b(0, None, C.byref(pitched), free, None, None, at["hidden_dev"] + 4 * width - 4, 2 * width, None, width, None), b"overlap")


# ---- masked classes under an entropy gradient, rows far from zero

@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(20, 64, 700), (60, 64, 700), (300, 72, 31), (400, 64, 700), (3000, 256, 700)])
@pytest.mark.parametrize("bonus", [2.0 ** -15, 0.5, 4.0])
def test_entropy_gradients_of_masked_classes(n, d, v, dtype, bonus):
    """A class at -inf, or at the type's lowest value, has probability zero and no gradient whatever the upstream of the entropy is (its log-probability times that
    upstream must not run past float32): every kernel of every type, from an entropy bonus of a mean over many rows to upstream values above 1."""
    h, w, b, t = make(n, d, v, dtype, seed=n + v)
    off = torch.zeros(v, dtype=torch.bool, device="cuda")
    off[3:v // 2] = True
    off[v - 1] = True
    t = torch.where((t != IGN) & off[t.clamp(min=0)], 1, t)
    T = Truth(h, w, torch.where(off, -float("inf"), b.float()).to(dtype), t)
    A, E = torch.linspace(-1, 1, n, device="cuda") * bonus, torch.linspace(0.5, 1, n, device="cuda") * bonus
    ref = T.grads(A, E)
    for low in (-float("inf"), torch.finfo(dtype).min):
        bias = torch.where(off, torch.full_like(b, low), b)
        leaves = [x.clone().requires_grad_() for x in (h, w, bias)]
        logp, ent = categorical.linear_categorical(leaves[0], leaves[1], t, leaves[2])
        near(logp, T.logp, T.elogp, "logp")
        near(ent, T.entropy, T.eent, "entropy")
        got = torch.autograd.grad((logp, ent), leaves, (A, E))
        for name, x, (r, tol) in zip(("dh", "dw", "db"), got, ref):
            near(x, r, tol, f"{name}, masked by {low}")
        assert not bool(got[1][off].any()) and not bool(got[2][off].any())


def _far_biases(dtype, v):
    """biases that put a row far from zero: (name, bias); logits are the biases themselves where the hidden row is zero"""
    info = torch.finfo(dtype)
    g = torch.Generator(device="cuda").manual_seed(v)
    r = torch.randn(v, device="cuda", generator=g)
    low = torch.full((v,), info.min, device="cuda", dtype=dtype)
    out = [("all at the lowest value", low)]
    some = low.clone()
    some[::3] = r[::3].to(dtype)
    out.append(("two thirds at the lowest value", some))
    top = r.to(dtype, copy=True)
    top[v // 2] = info.max
    out.append(("one at the largest value", top))
    if dtype == torch.float16:
        out.append(("around -6e4", (-60000.0 + 32.0 * torch.round(r)).to(dtype)))
    else:
        out.append(("all at -1e9", torch.full((v,), -1e9, device="cuda", dtype=dtype)))
        out.append(("around -1e9", (-1e9 + 64.0 * torch.round(r)).to(dtype)))
        out.append(("between 1e38 and 3e38", (torch.linspace(1e38, 3e38, v, device="cuda")).to(dtype)))
        out.append(("between -3e38 and -1e38", (torch.linspace(-1e38, -3e38, v, device="cuda")).to(dtype)))
        out.append(("from -3e38 to 3e38", (3e38 * torch.linspace(-1, 1, v, device="cuda")).to(dtype)))
    out.append(("around 1000", (1000.0 + r).to(dtype)))
    return out


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v", [(1, 700), (20, 700), (300, 31), (40, 700), (100, 300), (300, 700), (2500, 600)])
def test_rows_far_from_zero(n, v, dtype):
    """Rows whose logits are all very small, or of any size: the distribution depends on the differences alone.  With zero hidden rows the logits are the biases, exactly, so that only the
    sums, the exponentials and the final roundings are off; no term of the log-sum-exp's own magnitude is allowed.  (Differences past float32's range are held to its largest value.)"""
    d = 64
    h, w, _, t = make(n, d, v, dtype, seed=n)
    h = torch.zeros_like(h)
    for name, b in _far_biases(dtype, v):
        bd = b.double()
        T = Truth(h, w, bd - bd.max(), t)                                      # only differences count: the shift is exact enough in float64, and keeps log V
        T.logp = T.logp.clamp(min=-float(torch.finfo(torch.float32).max))
        T.el = torch.zeros_like(T.el)
        T.elogp = (256 + v / 2048 + 16) * 2 * U + 8 * U * (T.lse.abs() + T.logp.abs() + 1)
        few = (256 + v / 2048 + 16) * 2 * U + 8 * U * (T.lse.abs() + 30)       # of a probability that is not zero: its logarithm is above -105
        T.e = 2 * few
        T.eent = T.e * (T.p * (T.lp.abs() + 1)).sum(1) + few
        leaves = [x.clone().requires_grad_() for x in (h, w, b)]
        logp, ent = categorical.linear_categorical(leaves[0], leaves[1], t, leaves[2])
        near(logp, T.logp, T.elogp, f"logp, {name}")
        near(ent, T.entropy, T.eent, f"entropy, {name}")
        A, E = torch.linspace(-1, 1, n, device="cuda"), torch.linspace(0.5, 0.1, n, device="cuda")
        for what, x, (r, tol) in zip(("dh", "dw", "db"), torch.autograd.grad((logp, ent), leaves, (A, E)), T.grads(A, E)):
            near(x, r, tol, f"{what}, {name}")
    loss, dh, dw, db = categorical.linear_cross_entropy_grad(h, w, t, torch.full((v,), torch.finfo(dtype).min, device="cuda", dtype=dtype), reduction="sum")
    live = int((t != IGN).sum())
    assert abs(float(loss) - live * math.log(v)) <= live * math.log(v) * 2.0 ** -12 and all(bool(torch.isfinite(x).all()) for x in (dh, dw, db))


def test_refuses_forward_mode_tangents():
    """a dual tensor does not require grad: without a check it would go past the autograd function and come back without its tangent"""
    import torch.autograd.forward_ad as fwad
    h, w, b, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(5), torch.zeros(4, dtype=torch.int64)
    calls = (categorical.linear_categorical, categorical.linear_cross_entropy, categorical.linear_cross_entropy_grad)
    with fwad.dual_level():
        for f in calls:
            for k in (0, 1, 3):
                args = [h, w, t, b]
                args[k] = fwad.make_dual(args[k], torch.ones_like(args[k]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*args)
            with pytest.raises(_lib.Q1EnvError):                               # (no tangent: on to the next check)
                f(h, w, t, b)
    for f in calls[:2]:
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda x: f(x, w, t, b), (h,), (torch.ones_like(h),))


def _room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip(f"needs {gib} GiB of device memory")


@gpu
def test_more_tiles_than_one_launch_holds():
    """2^22 rows against 131073 classes: more than 2^32 threads in any tile, so that the classes go in pieces although the weights are taken as they lie"""
    _room(40)
    n, d, v = 2 ** 22, 8, 131073
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(n, d, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randn(v, d, device="cuda", generator=g).to(torch.bfloat16)
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    t[5], t[6], t[n - 1] = IGN, v - 1, v - 1
    logp, ent = categorical.linear_categorical(h, w, t)
    i = torch.cat([torch.arange(0, n, n // 100, device="cuda"), torch.arange(8, device="cuda"), torch.arange(n - 8, n, device="cuda")])
    T = Truth(h[i], w, None, t[i])
    near(logp[i], T.logp, T.elogp, "logp")
    near(ent[i], T.entropy, T.eent, "entropy")
    assert bool(torch.isfinite(logp).all() & torch.isfinite(ent).all()) and int((logp == 0).sum()) == 1
    del logp, ent
    torch.cuda.empty_cache()


@gpu
def test_more_values_than_one_launch_lays_out():
    """2^22 rows of 8191 halves, which have to be laid out: 2^32 threads"""
    _room(150)
    n, d, v = 2 ** 22, 8191, 3
    h = torch.zeros(n, d, device="cuda", dtype=torch.float16)
    w = torch.randn(v, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).mul_(0.01).to(torch.float16)
    i = torch.tensor([0, 1, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, n - 2, n - 1], device="cuda")
    h[i] = torch.randn(len(i), d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.float16)
    t = torch.arange(n, device="cuda") % v
    logp, ent = categorical.linear_categorical(h, w, t)
    T = Truth(h[i], w, None, t[i])
    near(logp[i], T.logp, T.elogp, "logp")
    near(ent[i], T.entropy, T.eent, "entropy")
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[i] = False
    assert bool(((logp[rest] + math.log(v)).abs() < 1e-6).all())              # zero rows are uniform
    del h, logp, ent
    torch.cuda.empty_cache()


@gpu
def test_more_parts_than_one_launch_adds_up():
    """the gradient of 2^22 rows of 4096 values over two pieces of the classes: 2^34 float32 sums, four to a thread"""
    _room(150)
    n, d, v = 2 ** 22, 4096, 300
    h = torch.zeros(n, d, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(v, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).mul_(0.03).to(torch.bfloat16)
    i = torch.tensor([0, 1, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, n - 2, n - 1], device="cuda")
    h[i] = torch.randn(len(i), d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.bfloat16)
    t = torch.full((n,), IGN, device="cuda")
    t[i] = torch.tensor([0, 299, 255, 256, 257, 1, 298], device="cuda")
    loss, dh, dw, _ = categorical.linear_cross_entropy_grad(h, w, t, reduction="sum")
    T = Truth(h[i], w, None, t[i])
    near(loss, -T.logp.sum(), T.elogp.sum() + 4 * U * T.logp.abs().sum(), "loss")
    ref = T.grads(torch.full((len(i),), -1.0, device="cuda"), torch.zeros(len(i), device="cuda"))
    near(dh[i], *ref[0], "dh")
    near(dw, *ref[1], "dw")
    dh[i] = 0
    assert not any(bool(x.any()) for x in dh.split(2 ** 18))
    del h, dh
    torch.cuda.empty_cache()


def test_the_library_refuses_a_workspace_or_state_over_an_operand():
    lib = _lib.load()
    rows, width, classes, base = 64, 8, 5, 1 << 24
    at = dict(hidden_dev=base, weight_dev=base + (1 << 16), bias_dev=base + (2 << 16), target_dev=base + (3 << 16), state_dev=base + (4 << 16), ws_dev=base + (1 << 20))
    free = base + (8 << 16)
    f, b = lib.q1env_head_forward, lib.q1env_head_backward
    for name in ("hidden_dev", "weight_dev", "bias_dev", "target_dev"):
        for what in ("ws_dev", "state_dev"):
            hd = head(rows=rows, width=width, classes=classes, **{**at, what: at[name]})
            assert f(0, None, C.byref(hd), 0, free, None, None) == -1 and b"overlaps an operand" in lib.q1env_last_error(), (name, what)
            if what == "ws_dev" and name != "target_dev":
                assert b(0, None, C.byref(hd), free, None, None, free + 4096, width, None, width, None) == -1 and b"overlaps an operand" in lib.q1env_last_error(), name
    ok = head(rows=rows, width=width, classes=classes, **at)
    assert b(0, None, C.byref(ok), at["ws_dev"] + 64, None, None, free + 4096, width, None, width, None) == -1 and b"workspace overlaps an upstream" in lib.q1env_last_error()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(20, 61, 300), (20, 64, 300), (60, 72, 500), (300, 64, 31), (300, 200, 700), (1500, 136, 2100)])
@pytest.mark.parametrize("gap", [0, 3, 8])
def test_results_at_a_pitch_and_every_choice_of_them(n, d, v, dtype, gap):
    """the C call writes rows of `width` values at any pitch and leaves what lies between them, and each of the three gradients is the same whichever others are asked for"""
    lib = _lib.load()
    h, w, b, t = make(n, d, v, dtype, seed=n + d)
    want = categorical.linear_cross_entropy_grad(h, w, t, b)[1:]
    dev, stream = h.device.index, torch.cuda.current_stream().cuda_stream
    dt = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]

    def struct(ws):
        return _lib.Q1Head(dt, 64, n, d, v, IGN, h.data_ptr(), d, w.data_ptr(), d, b.data_ptr(), t.data_ptr(), state.data_ptr(), ws.data_ptr(), ws.numel())
    state = torch.empty(lib.q1env_head_state_bytes(n), dtype=torch.uint8, device="cuda")
    logp, loss, one = torch.empty(n, device="cuda"), torch.empty((), device="cuda"), torch.ones((), device="cuda")
    ws = torch.empty(lib.q1env_head_workspace_bytes(dt, n, d, v, 0), dtype=torch.uint8, device="cuda")
    _lib.check(lib.q1env_head_forward(dev, stream, C.byref(struct(ws)), 0, logp.data_ptr(), None, loss.data_ptr()))
    ws = torch.empty(lib.q1env_head_workspace_bytes(dt, n, d, v, 1), dtype=torch.uint8, device="cuda")
    for asked in range(1, 8):
        dh, dw, db = (torch.full(s, 7.0, dtype=dtype, device="cuda") for s in ((n, d + gap), (v, d + gap), (v + 5,)))
        p = [x.data_ptr() if asked >> k & 1 else None for k, x in enumerate((dh, dw, db))]
        _lib.check(lib.q1env_head_backward(dev, stream, C.byref(struct(ws)), None, None, one.data_ptr(), p[0], d + gap, p[1], d + gap, p[2]))
        for k, (x, ref) in enumerate(zip((dh[:, :d], dw[:, :d], db[:v]), want)):
            if not asked >> k & 1:
                assert bool((x == 7).all())
            elif (asked == 7 and gap in (0, 8)) or k == 2:
                assert torch.equal(x, ref)                                    # the Python call, whole
            else:                                                             # (sums may be split elsewhere, and stored by other instructions: the same value to a rounding of the type and of the sums)
                far = (x.double() - ref.double()).abs() - 2.1 * HALF[dtype] * ref.double().abs() - (n + v + 16) * 2 * U * float(ref.abs().max())
                assert float(far.max()) <= (2.0 ** -24 if dtype == torch.float16 else 0.0)
        assert bool((dh[:, d:] == 7).all()) and bool((dw[:, d:] == 7).all()) and bool((db[v:] == 7).all())


@gpu
def test_no_rows_and_a_pitch():
    lib = _lib.load()
    w, dw, db = torch.randn(50, 24, device="cuda"), torch.full((50, 31), 7.0, device="cuda"), torch.full((53,), 7.0, device="cuda")
    hd = _lib.Q1Head(0, 64, 0, 24, 50, IGN, None, 24, w.data_ptr(), 24, None, None, None, None, 0)
    one = torch.ones((), device="cuda")
    _lib.check(lib.q1env_head_backward(0, torch.cuda.current_stream().cuda_stream, C.byref(hd), None, None, one.data_ptr(), None, 24, dw.data_ptr(), 31, db.data_ptr()))
    assert not bool(dw[:, :24].any()) and bool((dw[:, 24:] == 7).all()) and not bool(db[:50].any()) and bool((db[50:] == 7).all())


@gpu
def test_functional_transforms_are_refused_not_answered_wrongly():
    h, w, b, t = make(12, 16, 20, torch.float32, ignored=0.0)
    for f in (lambda: torch.func.grad(lambda x: categorical.linear_cross_entropy(x, w, t, b))(h), lambda: torch.func.jvp(lambda x: categorical.linear_cross_entropy(x, w, t, b), (h,), (h,)),
              lambda: torch.vmap(lambda x, y: categorical.linear_cross_entropy(x, w, y, b))(h.view(3, 4, 16), t.view(3, 4)),
              lambda: torch.func.jacrev(lambda x: categorical.linear_categorical(x, w, t, b)[0])(h)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(5, 8, 2 ** 22), (70, 8, 2 ** 22), (2 ** 22, 4, 3), (2 ** 22, 8, 40), (3, 2 ** 16, 5), (40, 2 ** 16, 70), (300, 2 ** 16, 33)])
def test_sizes_at_their_limits(n, d, v, dtype):
    _room(40)
    h, w, b, t = make(n, d, v, dtype, seed=d, ignored=0.2)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    logp, ent = categorical.linear_categorical(h, w, t, b)
    T = Truth(h, w, b, t)
    near(logp, T.logp, T.elogp, "logp")
    near(ent, T.entropy, T.eent, "entropy")
    A, E = torch.linspace(-1, 1, n, device="cuda"), torch.linspace(0.5, -0.5, n, device="cuda")
    got = torch.autograd.grad((logp, ent), leaves, (A, E))
    for name, x, (r, tol) in zip(("dh", "dw", "db"), got, T.grads(A, E)):
        near(x, r, tol, name)
    del T, got, leaves, logp, ent
    torch.cuda.empty_cache()
    for rows, width, classes in ((n + 1, d, v), (n, d + 1, v), (n, d, v + 1)):
        if rows > 2 ** 22 or width > 2 ** 16 or classes > 2 ** 22:
            with pytest.raises(ValueError, match="out of range"):
                categorical.linear_categorical(torch.empty(rows, width, dtype=dtype, device="cuda"), torch.empty(classes, width, dtype=dtype, device="cuda"),
                                               torch.zeros(rows, dtype=torch.int64, device="cuda"))
