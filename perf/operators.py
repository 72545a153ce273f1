"""What the training operators are measured on: the wide categorical head (log-probability and entropy of given actions, or the softmax cross
entropy of given classes, from hidden rows and the head's weights, without the logits ever being kept, and the gradients) and the clipping of
many gradients by their global norm.

`own = False`: elementary torch operations in 32 bits; `own = True`: q1physrl_amd.categorical and q1physrl_amd.clip."""
import math
import random

import torch

own = False

IGNORE = -100
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LARGEST = 8192 * 2048 * 131072          # rows x width x classes of the largest listed training step


def listed():
    return [
        # one environment asks for the log-probability of its action: the smallest call, the policy's own width, a mouse of half-degree steps
        dict(name="act_1", op="score", rows=1, width=256, classes=721, dtype="f32", bias=True, ignored=0.0),
        # the reference's 400 environments, a mouse of 2 x 2048 + 1 steps, half precision for the forward
        dict(name="act_400_f16", op="score", rows=400, width=256, classes=4097, dtype="f16", bias=True, ignored=0.0),
        # scoring a few long rows against a very wide head: the weights are read once and that is all the time there is
        dict(name="score_64_wide_bf16", op="score", rows=64, width=4096, classes=131073, dtype="bf16", bias=False, ignored=0.0),
        # the reference's minibatch of 128 samples, policy gradient with an entropy bonus, the learner's float32
        dict(name="policy_128", op="policy", rows=128, width=256, classes=361, dtype="f32", bias=True, ignored=0.0),
        # a large minibatch of 32 768 samples of the same network, a mouse of 2 x 720 + 1 steps
        dict(name="policy_32768", op="policy", rows=32768, width=256, classes=1441, dtype="f32", bias=True, ignored=0.05),
        # a train batch of 50 000 samples, padded rows among them, with reduced-precision operands
        dict(name="policy_50000_bf16", op="policy", rows=50000, width=256, classes=4097, dtype="bf16", bias=True, ignored=0.1),
        # cross entropy of recorded classes, nothing a multiple of anything, half precision
        dict(name="train_odd_f16", op="train", rows=1003, width=1000, classes=50001, dtype="f16", bias=True, ignored=0.1),
        # cross entropy of a middle-sized head with bfloat16 weights
        dict(name="train_4096_bf16", op="train", rows=4096, width=1024, classes=32768, dtype="bf16", bias=False, ignored=0.02),
        # the largest step: 8 192 rows against 131 072 classes
        dict(name="train_8192_bf16", op="train", rows=8192, width=2048, classes=131072, dtype="bf16", bias=False, ignored=0.0),
        # the gradients of the policy and value networks of the reference run: 12 tensors, 137 995 values, where latency counts
        dict(name="clip_policy", op="clip", layout="policy", tensors=12, values=137995, dtype="f32", max_norm=0.5),
        # hundreds of tensors of ragged sizes, down to single values
        dict(name="clip_ragged_bf16", op="clip", layout="ragged", tensors=500, values=25000003, dtype="bf16", max_norm=1.0),
        # a model's worth of gradients: the memory's rate counts
        dict(name="clip_large_f32", op="clip", layout="ragged", tensors=60, values=536870913, dtype="f32", max_norm=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("score", "policy", "train", "clip"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "clip":
        values = _log_int(rng, 100, 5e8)
        tensors = min(_log_int(rng, 1, 600), values)
        return dict(op=op, layout="ragged", tensors=tensors, values=values, dtype=dtype, max_norm=rng.choice((0.5, 1.0, 40.0, 1e6)))
    while True:
        rows, width, classes = _log_int(rng, 1, 50000), _log_int(rng, 16, 4096), _log_int(rng, 2, 131073)
        if rng.random() < 0.5:                       # widths are multiples of 64 more often than not
            width = max(64, width // 64 * 64)
        if rows * width * classes <= LARGEST // (16 if dtype == "f32" else 4):
            return dict(op=op, rows=rows, width=width, classes=classes, dtype=dtype, bias=rng.random() < 0.5,
                        ignored=rng.choice((0.0, 0.1, 0.5)) if op != "score" else 0.0)


# ---- inputs

POLICY_SIZES = [s for out in (10, 1) for s in (1536, 256, 65536, 256, 256 * out, out)]      # weights and biases of the two networks


def _sizes(case):
    """The gradients' sizes: the same for every seed, single values among them."""
    if case["layout"] == "policy":
        return list(POLICY_SIZES)
    rng = random.Random(case["values"] * 1009 + case["tensors"])
    n, total = case["tensors"], case["values"]
    w = [rng.random() ** 4 + 1e-9 for _ in range(n)]
    sizes = [1 + int((total - n) * x / sum(w)) for x in w]
    sizes[-1] += total - sum(sizes)
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    if case["op"] == "clip":
        sizes = _sizes(case)
        flat = torch.randn(sum(sizes), device="cuda", generator=gen)
        at = [0]
        for s in sizes:
            at.append(at[-1] + s)
        amp = torch.exp(torch.randn(len(sizes), device="cuda", generator=gen)).tolist()
        grads = [(flat[a:b] * m).to(dt) for a, b, m in zip(at, at[1:], amp)]
        bucket = torch.empty(sum(sizes), dtype=dt, device="cuda")
        return dict(case=case, grads=grads, bucket=bucket, out=[bucket[a:b] for a, b in zip(at, at[1:])])
    n, d, v = case["rows"], case["width"], case["classes"]
    s = dict(case=case)
    s["hidden"] = torch.tanh(torch.randn(n, d, device="cuda", generator=gen)).to(dt)            # a tanh layer's outputs
    s["weight"] = (torch.randn(v, d, device="cuda", generator=gen) * (2.5 / math.sqrt(d))).to(dt)
    s["bias"] = torch.randn(v, device="cuda", generator=gen).to(dt) if case["bias"] else None
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    padded = torch.rand(n, device="cuda", generator=gen) < case["ignored"]
    s["target"] = torch.where(padded, torch.full_like(target, IGNORE), target)
    if case["op"] == "policy":                       # what the loss above the head sends down: minus advantage x ratio, and the entropy bonus
        s["dlogp"] = torch.randn(n, device="cuda", generator=gen) / n
        s["dentropy"] = torch.full((n,), -0.01 / n, device="cuda")
    if case["op"] != "score":
        s["leaves"] = [s["hidden"].requires_grad_(), s["weight"].requires_grad_()] + ([s["bias"].requires_grad_()] if case["bias"] else [])
    return s


# ---- the plain forms

def _plain_rows(s):
    """logits' log-softmax (rows, classes), its probabilities, the kept rows, their classes (0 for the ignored)"""
    h, w = s["hidden"].detach().float(), s["weight"].detach().float()
    z = h @ w.T
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    z = z - z.amax(1, keepdim=True)
    logp = z - z.exp().sum(1, keepdim=True).log()
    keep = s["target"] != IGNORE
    return logp, logp.exp(), keep, torch.where(keep, s["target"], 0)


def _plain_grads(s, g):
    """The three products of the logits' gradient g (rows, classes)."""
    dt = s["hidden"].dtype
    dh, dw = g @ s["weight"].detach().float(), g.T @ s["hidden"].detach().float()
    return [dh.to(dt), dw.to(dt)] + ([g.sum(0).to(dt)] if s["bias"] is not None else [])


def _plain_score(s):
    logp, p, keep, t = _plain_rows(s)
    ent = -(p * logp).sum(1)
    return [logp.gather(1, t[:, None])[:, 0] * keep, ent * keep]


def _plain_policy(s):
    logp, p, keep, t = _plain_rows(s)
    ent = -(p * logp).sum(1)
    out = [logp.gather(1, t[:, None])[:, 0] * keep, ent * keep]
    a, b = s["dlogp"] * keep, s["dentropy"] * keep
    g = -p * (a[:, None] + b[:, None] * (logp + ent[:, None]))
    g.scatter_add_(1, t[:, None], a[:, None])
    return out + _plain_grads(s, g)


def _plain_train(s):
    logp, p, keep, t = _plain_rows(s)
    count = keep.sum().clamp(min=1)
    loss = -(logp.gather(1, t[:, None])[:, 0] * keep).sum() / count
    each = keep / count
    g = p * each[:, None]
    g.scatter_add_(1, t[:, None], -each[:, None])
    return [loss] + _plain_grads(s, g)


def _plain_clip(s):
    flat = torch.cat([g.reshape(-1).float() for g in s["grads"]])
    norm = flat.square().sum(dtype=torch.float64).sqrt().float()
    top = s["case"]["max_norm"]
    return [norm, (flat * (top / norm.clamp(min=top))).to(s["bucket"].dtype)]


# ---- the framework's calls

def _own_score(s):
    from q1physrl_amd import categorical
    with torch.no_grad():
        return list(categorical.linear_categorical(s["hidden"], s["weight"], s["target"], s["bias"], ignore_index=IGNORE))


def _own_policy(s):
    from q1physrl_amd import categorical
    logp, ent = categorical.linear_categorical(s["hidden"], s["weight"], s["target"], s["bias"], ignore_index=IGNORE)
    return [logp.detach(), ent.detach()] + list(torch.autograd.grad((logp, ent), s["leaves"], (s["dlogp"], s["dentropy"])))


def _own_train(s):
    from q1physrl_amd import categorical
    loss = categorical.linear_cross_entropy(s["hidden"], s["weight"], s["target"], s["bias"], ignore_index=IGNORE)
    return [loss.detach()] + list(torch.autograd.grad(loss, s["leaves"]))


def _own_clip(s):
    from q1physrl_amd import clip
    norm = clip.clip_grad_norm_(s["grads"], s["case"]["max_norm"], out=s["out"])
    return [norm, s["bucket"]]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"score": _own_score, "policy": _own_policy, "train": _own_train, "clip": _own_clip}[op](state)
    return {"score": _plain_score, "policy": _plain_policy, "train": _plain_train, "clip": _plain_clip}[op](state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "clip":
        return {"bytes": 2.0 * size * case["values"], "flops": 3.0 * case["values"]}
    n, d, v = case["rows"], case["width"], case["classes"]
    inputs = size * (n * d + v * d + (v if case["bias"] else 0)) + 8 * n
    if case["op"] == "score":
        return {"bytes": inputs + 8.0 * n, "flops": 2.0 * n * d * v}
    extra = 16.0 * n if case["op"] == "policy" else 4.0
    return {"bytes": inputs + extra + size * (n * d + v * d + (v if case["bias"] else 0)), "flops": 6.0 * n * d * v}


# ---- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        squares = [float(torch.dot(x, x)) for x in (g.double() for g in s["grads"])]
        norm = math.sqrt(math.fsum(squares))
        factor = min(1.0, case["max_norm"] / norm) if norm > 0.0 else 1.0
        return [torch.tensor(norm, dtype=torch.float64), torch.cat([g.double() for g in s["grads"]]) * factor]
    h, w, t = s["hidden"].detach().double(), s["weight"].detach().double(), s["target"]
    b = None if s["bias"] is None else s["bias"].detach().double()
    n, v = case["rows"], case["classes"]
    live = (t != IGNORE).double()
    a, e = None, None
    if case["op"] == "train":
        a = -live / max(1.0, float(live.sum()))      # d loss / d log-probability of the row's class
        e = torch.zeros_like(live)
    elif case["op"] == "policy":
        a, e = s["dlogp"].double() * live, s["dentropy"].double() * live
    logp, ent = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    dh = torch.zeros_like(h)
    dw, db = (torch.zeros_like(w), torch.zeros(v, dtype=torch.float64, device="cuda")) if a is not None else (None, None)
    step = max(1, (1 << 28) // v)                    # row by row, in pieces of the rows
    for i in range(0, n, step):
        z = h[i:i + step] @ w.T
        if b is not None:
            z += b
        lse = torch.logsumexp(z, 1)
        z -= lse[:, None]
        p = torch.exp(z)
        hrow = -(p * z).sum(1)
        k = t[i:i + step].clamp(min=0)
        rows = torch.arange(z.shape[0], device="cuda")
        logp[i:i + step] = z[rows, k] * live[i:i + step]
        ent[i:i + step] = hrow * live[i:i + step]
        if a is None:
            continue
        ai, ei = a[i:i + step], e[i:i + step]
        z += hrow[:, None]
        z *= p
        z *= -ei[:, None]
        z -= ai[:, None] * p
        z[rows, k] += ai
        dh[i:i + step] = z @ w
        dw += z.T @ h[i:i + step]
        db += z.sum(0)
    grads = [] if a is None else [dh, dw] + ([db] if b is not None else [])
    if case["op"] == "train":
        return [-(logp * live).sum() / max(1.0, float(live.sum()))] + grads
    return [logp, ent] + grads
