"""The wide categorical head and gradient clipping as the learner uses them: Q1Policy.evaluate_actions, PPOLearner(logits_free=True), PPOLearner(grad_clip=...)."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from q1physrl_amd import _lib, clip, policy as P, ppo

gpu = pytest.mark.gpu
U = 2.0 ** -24


def make(steps, batch, device="cuda", seed=0):
    torch.manual_seed(seed)
    pol = P.Q1Policy(discrete_yaw_steps=steps).to(device)
    with torch.no_grad():
        pol.pi[-1].weight.mul_(100.0)                   # logits that differ: the constructor makes them nearly equal
    g = torch.Generator(device=device).manual_seed(seed)
    obs = torch.randn(batch, 6, device=device, generator=g)
    keys = torch.randint(0, 2, (batch, 4), device=device, generator=g)
    mouse = torch.randint(0, 2 * steps + 1, (batch, 1), device=device, generator=g).float()
    return pol, obs, keys, mouse


def trajectory(pol, steps, t, n, seed=0):
    """what the sampler leaves, with the policy's own log-probabilities"""
    pol2, obs, keys, mouse = make(steps, (t + 1) * n, seed=seed)
    with torch.no_grad():
        logits, value = pol(obs)
        logp = P.Q1PhysActionDist(logits, 10.0, discrete_yaw_steps=steps).logp(keys, mouse)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    k = t * n
    traj = {"obs": obs.view(t + 1, n, 6), "keys": P.pack_keys(keys)[:k].view(t, n), "mouse": mouse[:k].view(t, n), "logp": logp[:k].view(t, n), "value": value.view(t + 1, n),
            "reward": torch.zeros(t, n, device="cuda"), "done": torch.zeros(t, n, dtype=torch.uint8, device="cuda")}
    return traj, torch.randn(t, n, device="cuda", generator=g), torch.randn(t, n, device="cuda", generator=g)


@gpu
@pytest.mark.parametrize("steps,batch", [(5, 1), (5, 300), (360, 257), (2048, 100)])
def test_evaluate_actions_against_the_distribution(steps, batch):
    """the same policy in float64 through its logits.  The hidden layer's and the key logits' own float32 error is part of both sides' inputs: hidden values are below 1 and off by
    at most (256 + 6 + 16) 2u x 256^(1/2)-ish sums; the logits' weights sum to S <= sum |w| per class, so a logit is off by that times S; log-probabilities by twice it"""
    pol, obs, keys, mouse = make(steps, batch)
    logp, ent, value = pol.evaluate_actions(obs, keys, mouse)
    ref = P.Q1Policy(discrete_yaw_steps=steps).cuda().double()
    ref.load_state_dict({k: v.double() for k, v in pol.state_dict().items()})
    logits, v = ref(obs.double())
    d = P.Q1PhysActionDist(logits, 10.0, discrete_yaw_steps=steps)
    lp, en = d.logp(keys, mouse.double()), d.entropy()
    layer = [m.weight.detach().abs().sum(1).max().item() for m in (pol.pi[0], pol.pi[2], pol.pi[4])]
    e1 = (6 + 8) * 2 * U * layer[0] * float(obs.abs().max())
    e2 = e1 * layer[1] + (256 + 8) * 2 * U * layer[1]
    e3 = e2 * layer[2] + (256 + 8) * 2 * U * layer[2]
    tol = 2 * 5 * (e3 + 300 * 2 * U) + 1e-6
    assert float((logp - lp).abs().max()) <= tol and float((ent - en).abs().max()) <= tol * (1 + float(lp.abs().max()))
    w = torch.randn(batch, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    ga = torch.autograd.grad((w * logp).sum() + 0.1 * ent.sum(), list(pol.pi.parameters()))
    gb = torch.autograd.grad((w.double() * lp).sum() + 0.1 * en.sum(), list(ref.pi.parameters()))
    for a, b in zip(ga, gb):
        # relative to the whole gradient: a probability is off by tol relative, and sums of up to `batch` such terms keep that
        assert float((a.double() - b).norm()) <= 4 * tol * (float(b.norm()) + 1.0)


@gpu
def test_logits_free_update_is_the_loss_it_says():
    """one step of PPOLearner(logits_free=True) against autograd of the same loss through stored logits in float64: the parameters after one plain gradient step"""
    steps, t, n = 40, 8, 32
    pol, *_ = make(steps, 1)
    traj, adv, vtarg = trajectory(pol, steps, t, n)
    ref = P.Q1Policy(discrete_yaw_steps=steps).cuda().double()
    ref.load_state_dict({k: v.double() for k, v in pol.state_dict().items()})
    lrn = ppo.PPOLearner(pol, 10.0, lr=1e-3, num_sgd_iter=1, minibatch_size=t * n, discrete_yaw_steps=steps, logits_free=True, grad_clip=0.7, kl_coeff=0.2)
    seen = {}
    lrn.opt.step = lambda: seen.update({k: p.grad.clone() for k, p in pol.named_parameters()})
    out = lrn.update(traj, adv, vtarg)
    a = adv.double().reshape(-1)
    a = (a - a.mean()) / torch.sqrt(torch.clamp((a * a).mean() - a.mean() ** 2, min=1e-8))
    logits, value = ref(traj["obs"][:t].reshape(t * n, 6).double())
    keys = (traj["keys"].reshape(-1, 1).long() >> torch.arange(4, device="cuda")) & 1
    d = P.Q1PhysActionDist(logits, 10.0, discrete_yaw_steps=steps)
    lr = d.logp(keys, traj["mouse"].reshape(-1, 1).double()) - traj["logp"].reshape(-1).double()
    r = lr.exp()
    surr = torch.minimum(a * r, a * r.clamp(0.7, 1.3))
    v0, vt = traj["value"][:t].reshape(-1).double(), vtarg.reshape(-1).double()
    vf = torch.maximum((value - vt) ** 2, (v0 + (value - v0).clamp(-100, 100) - vt) ** 2)
    loss = (-surr + 0.2 * (r - 1 - lr) + vf - 0.01 * d.entropy()).mean()
    loss.backward()
    norm = torch.sqrt(sum((p.grad ** 2).sum() for p in ref.parameters()))
    assert float(norm) > 0.7 and abs(float(lrn.grad_norm) - float(norm)) <= 1e-4 * float(norm)
    total = 0.0
    for k, p in ref.named_parameters():
        g = p.grad * (0.7 / norm)
        assert float((seen[k].double() - g).norm()) <= 1e-4 * (float(g.norm()) + 1e-2), k
        total += float((seen[k].double() ** 2).sum())
    assert abs(total ** 0.5 - 0.7) <= 1e-5
    assert abs(out["total_loss"] - float(loss)) <= 1e-4 * (1 + abs(float(loss)))


@gpu
def test_a_run_of_both_together():
    """several updates with a mouse of 4 097 steps, clipped, with a reduced-precision hidden layer as well: every parameter moves and stays finite, the statistics are there"""
    for autocast in (None, torch.bfloat16):
        steps = 2048
        pol, *_ = make(steps, 1, seed=5)
        lrn = ppo.PPOLearner(pol, 10.0, lr=1e-4, num_sgd_iter=2, minibatch_size=64, discrete_yaw_steps=steps, logits_free=True, grad_clip=0.5, autocast_dtype=autocast)
        before = [p.detach().clone() for p in pol.parameters()]
        for it in range(3):
            traj, adv, vtarg = trajectory(pol, steps, 4, 40, seed=it)
            out = lrn.update(traj, adv, vtarg)
            assert out["sgd_steps"] == 4 and all(np.isfinite(v) for v in out.values())
            assert torch.isfinite(lrn.grad_norm) and float(clip.grad_norm([p.grad for p in pol.parameters()])) <= 0.5 * (1 + 1e-5)
        assert all(bool(torch.isfinite(p).all()) and not torch.equal(p, q) for p, q in zip(pol.parameters(), before))


@gpu
@pytest.mark.parametrize("use_graph", [False, True])
def test_grad_clip_of_the_torch_learner_eager_and_captured(use_graph):
    """the continuous mouse: the clipped step equals torch's gradients scaled by hand; a captured step replays to the same weights as the eager one"""
    def run(graph, grad_clip):
        torch.manual_seed(0)
        pol = P.Q1Policy().cuda()
        t, n = 4, 64
        g = torch.Generator(device="cuda").manual_seed(1)
        obs = torch.randn(t + 1, n, 6, device="cuda", generator=g)
        traj = {"obs": obs, "keys": torch.randint(0, 16, (t, n), device="cuda", generator=g).to(torch.uint8), "mouse": torch.rand(t, n, device="cuda", generator=g) * 10 - 5,
                "logp": torch.full((t, n), -5.0, device="cuda"), "value": torch.zeros(t + 1, n, device="cuda"), "reward": torch.zeros(t, n, device="cuda"),
                "done": torch.zeros(t, n, dtype=torch.uint8, device="cuda")}
        adv, vt = torch.randn(t, n, device="cuda", generator=g), torch.randn(t, n, device="cuda", generator=g)
        lrn = ppo.PPOLearner(pol, 10.0, lr=1e-3, num_sgd_iter=2, minibatch_size=64, use_graph=graph, grad_clip=grad_clip)
        for _ in range(2):
            lrn.update(traj, adv, vt)
        return pol, lrn
    pol, lrn = run(use_graph, 0.05)
    other, _ = run(not use_graph, 0.05)
    assert torch.isfinite(lrn.grad_norm) and float(lrn.grad_norm) > 0.05
    # the same kernels in the same order; capturable Adam divides in another order than the eager one, a few roundings per step of size lr
    for a, b in zip(pol.parameters(), other.parameters()):
        assert float((a - b).abs().max()) <= 1e-3 * 8 * 1e-2
    free, _ = run(use_graph, None)
    assert any(not torch.equal(a, b) for a, b in zip(pol.parameters(), free.parameters()))


@gpu
def test_grad_clip_with_the_native_step():
    """native gradients, clipped, then torch's Adam: gradients of the last step have the bound's norm"""
    from q1physrl_amd.env import Config
    from q1physrl_amd.sampler import GpuSampler
    from q1physrl_amd.tensor_env import TensorVectorEnv
    torch.manual_seed(0)
    env = TensorVectorEnv(Config(**{**Config.get_default().__dict__, "num_envs": 256}), device=0, seed=1)
    pol = P.Q1Policy().cuda()
    smp = GpuSampler(env, pol, horizon=16)
    traj = smp.collect()
    lrn = ppo.PPOLearner(pol, 10.08, lr=1e-4, num_sgd_iter=1, minibatch_size=2048, native=True, native_splits=8, env=env, grad_clip=1e-3)
    assert lrn.native_adam is False
    adv, vt = smp.advantages(traj, 0.99, 0.95)
    before = [p.detach().clone() for p in pol.parameters()]
    out = lrn.update(traj, adv, vt)
    assert out["sgd_steps"] == 2 and float(lrn.grad_norm) > 1e-3
    assert abs(float(clip.grad_norm([p.grad for p in pol.parameters()])) - 1e-3) <= 1e-8
    assert all(not torch.equal(p, q) for p, q in zip(pol.parameters(), before))
    with pytest.raises(ValueError, match="grad_clip"):
        ppo.PPOLearner(pol, 10.08, minibatch_size=128, native=True, env=env, grad_clip=1.0, persistent=True).update(traj, adv, vt)
    env.close()


# ---- CPU

def test_refused_combinations():
    pol = P.Q1Policy(discrete_yaw_steps=5)
    for kw in (dict(native=True, env=object()), dict(fused_loss=True, env=object()), dict(use_graph=True)):
        with pytest.raises(ValueError, match="logits_free"):
            ppo.PPOLearner(pol, 10.0, discrete_yaw_steps=5, logits_free=True, **kw)
    with pytest.raises(ValueError, match="discrete"):
        ppo.PPOLearner(P.Q1Policy(), 10.0, logits_free=True)
    with pytest.raises(ValueError, match="discrete"):
        P.Q1Policy().evaluate_actions(torch.zeros(1, 6), torch.zeros(1, 4), torch.zeros(1))
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            ppo.PPOLearner(pol, 10.0, grad_clip=bad)
    with pytest.raises(_lib.Q1EnvError):
        pol.evaluate_actions(torch.zeros(2, 6), torch.zeros(2, 4, dtype=torch.int64), torch.zeros(2))


def grads_of(seed, scale):
    torch.manual_seed(seed)
    pol = P.Q1Policy()
    g = torch.Generator().manual_seed(100 + seed)
    for p in pol.parameters():
        p.grad = torch.randn(p.shape, generator=g) * scale
    return list(pol.parameters())


def test_clip_on_the_cpu_is_the_formula():
    params = grads_of(0, 1.0)
    norm = float(torch.sqrt(sum((p.grad.double() ** 2).sum() for p in params)))
    kept = [p.grad.clone() for p in params]
    got = ppo.clip_grads_(params, 2.0)
    assert abs(float(got) - norm) <= 1e-6 * norm
    for p, k in zip(params, kept):
        assert torch.allclose(p.grad, k * (2.0 / norm), rtol=4e-7, atol=0)
    again = [p.grad.clone() for p in params]
    ppo.clip_grads_(params, 1e9)
    assert all(torch.equal(p.grad, a) for p, a in zip(params, again))


def _worker(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    params = grads_of(rank, 0.5)
    norm = ppo.allreduce_grads_(params, 2, grad_clip=0.25)
    torch.save(([p.grad for p in params], norm), f"{out}.{rank}")
    dist.destroy_process_group()


def test_two_ranks_clip_the_average(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(port, str(tmp_path / "g")), nprocs=2)
    a, b = (torch.load(f"{tmp_path / 'g'}.{r}", weights_only=True) for r in (0, 1))
    mean = [(x.grad + y.grad) / 2 for x, y in zip(grads_of(0, 0.5), grads_of(1, 0.5))]
    norm = float(torch.sqrt(sum((m.double() ** 2).sum() for m in mean)))
    for x, y, m in zip(a[0], b[0], mean):
        assert torch.equal(x, y) and torch.allclose(x, m * (0.25 / norm), rtol=1e-6, atol=1e-12)
    assert abs(float(a[1]) - norm) <= 1e-6 * norm


@gpu
def test_averaged_and_clipped_gradients_of_mixed_types_and_layouts(monkeypatch):
    """allreduce_grads_(grad_clip=...) where the bucket's views do not have the gradients' types or layouts: the same values as averaging and then clipping."""
    monkeypatch.setattr(ppo.dist, "all_reduce", lambda t, op=None: t.mul_(2))          # two ranks with the same gradients
    torch.manual_seed(0)
    for mixed in (False, True):
        params = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for n in (300, 40)] + [torch.nn.Parameter(torch.zeros(30, 20, device="cuda"))]
        if mixed:
            params[1] = torch.nn.Parameter(torch.zeros(40, device="cuda", dtype=torch.bfloat16))
        for p in params:
            p.grad = torch.randn(p.shape, device="cuda").to(p.dtype)
        params[2].grad = torch.randn(20, 30, device="cuda").t()
        want = [p.grad.clone() for p in params]
        norm = torch.sqrt(sum((g.double() ** 2).sum() for g in want))
        got = ppo.allreduce_grads_(params, 2, 0.5)
        assert abs(float(got) - float(norm)) <= 1e-6 * float(norm)                     # a double sum rounded once: half a step of float32
        for p, w in zip(params, want):
            ref = w.double() * (0.5 / norm)
            assert bool(((p.grad.double() - ref).abs() <= ref.abs() * (2 ** -8 + 2 ** -22 if p.dtype == torch.bfloat16 else 2 ** -22)).all())


@gpu
@pytest.mark.parametrize("use_graph", [False, True])
def test_from_the_sampler_to_the_logits_free_step(use_graph):
    """GpuSampler with a mouse of 4 097 steps into PPOLearner(logits_free=True): with and without kept logits the same trajectory and the same step; the sampler's
    log-probabilities, taken from its logits, are those the head gives for its actions; the statistics of the first step are the stored-logits loss's."""
    from q1physrl_amd.env import Config
    from q1physrl_amd.sampler import GpuSampler
    from q1physrl_amd.tensor_env import TensorVectorEnv
    steps, n, t = 2048, 64, 6
    cfg = Config(**{**Config.get_default().__dict__, "num_envs": n, "discrete_yaw_steps": steps})

    def run(keep, logits_free):
        torch.manual_seed(0)
        env = TensorVectorEnv(cfg, device=0, seed=1)
        pol, *_ = make(steps, 1, seed=3)
        smp = GpuSampler(env, pol, horizon=t, use_graph=use_graph, keep_logits=keep)
        assert smp.logits.shape == ((t if keep else 1), n, 8 + 2 * steps + 1)
        smp.collect()
        traj = smp.collect()
        assert ("logits" in traj) == keep
        with torch.no_grad():
            logp, ent, _ = pol.evaluate_actions(traj["obs"][:t].reshape(-1, 6), (traj["keys"].reshape(-1, 1).long() >> torch.arange(4, device="cuda")) & 1, traj["mouse"].reshape(-1))
        # both float32 sums over 256 terms of weights around 0.06 and logits of a few units
        assert float((logp - traj["logp"].reshape(-1)).abs().max()) <= 1e-4
        adv, vt = smp.advantages(traj, 0.99, 0.95)
        lrn = ppo.PPOLearner(pol, float(cfg.action_range), lr=1e-4, num_sgd_iter=1, minibatch_size=t * n, discrete_yaw_steps=steps, logits_free=logits_free)
        kept = {k: v.clone() for k, v in traj.items()}
        out = lrn.update(traj, adv, vt)
        grads = [p.grad.clone() for p in pol.parameters()]
        env.close()
        return kept, out, grads, float(ent.mean())
    a, oa, ga, ea = run(True, True)
    b, ob, gb, _ = run(False, True)
    assert all(torch.equal(a[k], b[k]) for k in b) and oa == ob and all(map(torch.equal, ga, gb))
    assert int(a["mouse"].max()) > steps and int(a["mouse"].min()) >= 0
    _, oc, gc, _ = run(True, False)
    assert abs(oa["entropy"] - ea) <= 1e-4 * ea
    for k in ("policy_loss", "vf_loss", "entropy"):
        assert abs(oa[k] - oc[k]) <= 1e-4 * (1 + abs(oc[k])), k
    assert abs(oa["kl"]) <= 1e-4 and abs(oc["kl"]) <= 1e-4
    for x, y in zip(ga, gc):                                     # at the old policy the estimated KL has no gradient, nor has the exact one
        assert float((x - y).norm()) <= 1e-3 * (float(y.norm()) + 1e-3)


def test_a_resident_sampler_keeps_its_logits():
    from q1physrl_amd.sampler import GpuSampler

    class Fused:
        _mlp = None
    with pytest.raises(ValueError, match="keeps its logits"):
        GpuSampler(None, Fused(), 4, resident=True, keep_logits=False)


@gpu
@pytest.mark.parametrize("steps,batch", [(5, 1), (5, 300), (360, 257), (2048, 100)])
def test_evaluate_actions_term_by_term(steps, batch):
    """The head's own error, without the layers before it: in float64 from the very hidden rows the call computed (test_categorical.Truth bounds the mouse's part, derived there; a key's
    logits are off by el, its log-probability and entropy by 2 el and a few roundings).  Log-probability and entropy are differentiated apart, and every part of the gradient is held to its
    own bound, so that none can be missing."""
    from tests.test_categorical import Truth, near
    pol, obs, keys, mouse = make(steps, batch)
    seen = []
    pol.pi[-2].register_forward_hook(lambda m, i, o: seen.append(o) or o.retain_grad())
    logp, ent, value = pol.evaluate_actions(obs, keys, mouse)
    assert torch.equal(value, pol.vf(obs).squeeze(-1))
    h = seen[0].detach()
    w, b = pol.pi[-1].weight.detach(), pol.pi[-1].bias.detach()
    T = Truth(h, w[8:], b[8:], mouse[:, 0].long())
    leaves = [x.double().requires_grad_() for x in (h, w[:8], b[:8])]
    z = torch.nn.functional.log_softmax((leaves[0] @ leaves[1].T + leaves[2]).view(batch, 4, 2), 2)
    klp, kent = z.gather(2, keys[:, :, None])[:, :, 0].sum(1), -(z.exp() * z).sum((1, 2))
    S = (h.double().abs() @ w[:8].double().abs().T + b[:8].double().abs()).amax(1)
    el = (256 + 8) * 2 * U * S
    ek = 4 * (2 * el + 16 * U * (z.detach().abs().amax((1, 2)) + 1)) + 8 * U * (T.logp.abs() + T.entropy)
    near(logp, T.logp + klp.detach(), T.elogp + ek, "logp")
    near(ent, T.entropy + kent.detach(), T.eent + 3 * ek, "entropy")
    g = torch.Generator(device="cuda").manual_seed(3)
    A, E, zero = torch.randn(batch, device="cuda", generator=g), torch.randn(batch, device="cuda", generator=g), torch.zeros(batch, device="cuda")
    for out, ref, A_, E_ in ((logp, klp, A, zero), (ent, kent, zero, E)):
        pol.zero_grad()
        seen[0].grad = None
        out.backward(A_ + E_, retain_graph=True)
        (dh, th), (dw, tw), (db, tb) = T.grads(A_, E_)
        kh, kw, kb = torch.autograd.grad(ref, leaves, (A_ + E_).double(), retain_graph=True)
        # a key's gradient of a logit is off by 3 ek of the upstream at most, and sums of those by that of the absolute products
        off = 3 * ek * (A_ + E_).double().abs()
        size = (A_ + E_).double().abs() * 2
        rounding = (batch + 264) * 2 * U
        near(seen[0].grad, dh + kh, th + (off + rounding * size)[:, None] * w[:8].double().abs().sum(0) + 8 * U * (dh.abs() + kh.abs()), "dhidden")
        near(pol.pi[-1].weight.grad[8:], dw, tw * 1.01, "dweight, mouse")
        near(pol.pi[-1].bias.grad[8:], db, tb * 1.01, "dbias, mouse")
        near(pol.pi[-1].weight.grad[:8], kw, ((off + rounding * size) @ h.double().abs()).expand(8, -1) + 8 * U * kw.abs(), "dweight, keys")
        near(pol.pi[-1].bias.grad[:8], kb, (off + rounding * size).sum().expand(8) + 8 * U * kb.abs(), "dbias, keys")
        assert all(p.grad is not None and bool(p.grad.any()) for p in pol.pi.parameters())
        # a part that were missing would be over its bound somewhere: it is larger than the bound as a whole
        assert float(th.norm()) < float(dh.norm()) and float(tw.norm()) < float(dw.norm())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_an_infinite_bound_measures_and_leaves_the_gradients(device):
    """grad_clip=inf is how a learner asks for the norm alone: inf / inf is no factor"""
    params = [torch.nn.Parameter(p.detach().to(device)) for p in grads_of(0, 1.0)]
    for p, q in zip(params, grads_of(0, 1.0)):
        p.grad = q.grad.to(device)
    kept = [p.grad.clone() for p in params]
    norm = float(ppo.clip_grads_(params, float("inf")))
    assert abs(norm - float(torch.sqrt(sum((k.double() ** 2).sum() for k in kept)))) <= 1e-6 * norm
    assert all(torch.equal(p.grad, k) for p, k in zip(params, kept))
    params[0].grad[0, 0] = float("inf")
    assert ppo.clip_grads_(params, 1.0) == float("inf") and bool((params[1].grad == 0).all()) and bool(torch.isnan(params[0].grad[0, 0]))
