"""What is measured of the learning operators that stand next to the batched environments: the fused linear layer of a policy network, the draw of
actions from its logits, the advantages of a rollout and the clipped policy loss, each in a plain form (elementary torch operations) and, where `own`
is true, through minigrid_amd's public functions."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
OBS_SIZES = (147, 75, 243, 363, 192, 507, 1083)       # bytes of an observation: 7x7x3, 5x5x3, 9x9x3, 11x11x3, 8x8x3, 13x13x3, 19x19x3
ACTS = (None, "relu", "tanh", "gelu", "silu")
LARGEST_LINEAR = 32768 * 2048 * 4096                  # products of the largest listed linear case
LARGEST_LOSS = 16384 * 40961
LARGEST_ADVANTAGES = 128 * 65536
LARGEST_SAMPLE = 1 << 26


def listed():
    return [
        # one environment, one step: the first layer of a small policy on a byte observation, where only latency counts
        dict(name="linear_one_env", op="linear", rows=1, k=147, n=64, dtype="f32", obs=True, act="tanh", bias=True, residual=False, train=False),
        # the first layer of an update on 65 536 observations of 7x7x3 bytes: odd row length, no gradient of the input
        dict(name="linear_observations", op="linear", rows=65536, k=147, n=256, dtype="bf16", obs=True, act="relu", bias=True, residual=False, train=True),
        # a residual hidden layer of the same update, forward and backward
        dict(name="linear_hidden", op="linear", rows=65536, k=512, n=512, dtype="bf16", obs=False, act="gelu", bias=True, residual=True, train=True),
        # sizes that divide by nothing, in half precision, forward and backward
        dict(name="linear_ragged", op="linear", rows=5003, k=333, n=1001, dtype="f16", obs=False, act="silu", bias=True, residual=False, train=True),
        # the widening layer of a large network over 1024 environments x 32 steps, forward and backward
        dict(name="linear_wide", op="linear", rows=32768, k=2048, n=4096, dtype="bf16", obs=False, act="gelu", bias=True, residual=False, train=True),
        # a minibatch of 256 transitions with the seven actions
        dict(name="loss_minibatch", op="policy_loss", rows=256, vocab=7, dtype="f32", row_gap=0, padded=0.05, ref=False, closed=0.0),
        # a whole update of 262 144 transitions: the logits are seven of the eight columns of one head, the eighth is the value
        dict(name="loss_actions", op="policy_loss", rows=262144, vocab=7, dtype="f32", row_gap=1, padded=0.03, ref=True, closed=0.0),
        # answers as text: 16 384 tokens over an odd vocabulary, a quarter of them padding
        dict(name="loss_text", op="policy_loss", rows=16384, vocab=40961, dtype="bf16", row_gap=0, padded=0.25, ref=True, closed=0.0),
        # 128 steps of 65 536 environments
        dict(name="advantages_rollout", op="advantages", steps=128, envs=65536, done=0.004, next_step=True),
        # 2 048 steps of 16 environments: a long recurrence and few rows
        dict(name="advantages_long", op="advantages", steps=2048, envs=16, done=0.02, next_step=True),
        # the actions of one step of 65 536 environments
        dict(name="sample_actions", op="sample", rows=65536, vocab=7, dtype="bf16", greedy=False, closed=0.0),
        # the next token of 64 answers
        dict(name="sample_tokens", op="sample", rows=64, vocab=40961, dtype="f32", greedy=False, closed=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "policy_loss", "policy_loss", "advantages", "sample"])
    if op == "linear":
        obs = rng.random() < 0.3
        k = rng.choice(OBS_SIZES) if obs else _log(rng, 8, 4096)
        n = _log(rng, 1, 8192)
        rows = _log(rng, 1, max(1, min(131072, LARGEST_LINEAR // (k * n))))
        return dict(op=op, rows=rows, k=k, n=n, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), obs=obs, act=rng.choice(ACTS),
                    bias=rng.random() < 0.8, residual=rng.random() < 0.4, train=rng.random() < 0.7)
    if op == "policy_loss":
        vocab = rng.choice([2, 3, 5, 7, 7, _log(rng, 2, 131072), _log(rng, 2, 131072)])
        rows = _log(rng, 1, max(1, min(262144, LARGEST_LOSS // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "f16"]), row_gap=rng.choice([0, 1, 5]),
                    padded=rng.choice([0.0, 0.03, 0.3]), ref=rng.random() < 0.5, closed=rng.choice([0.0, 0.0, 0.2]))
    if op == "advantages":
        envs = _log(rng, 1, 262144)
        steps = _log(rng, 1, max(1, min(2048, LARGEST_ADVANTAGES // envs)))
        return dict(op=op, steps=steps, envs=envs, done=rng.choice([0.0, 0.004, 0.1]), next_step=rng.random() < 0.7)
    vocab = rng.choice([2, 5, 7, 7, _log(rng, 2, 131072)])
    rows = _log(rng, 1, max(1, min(262144, LARGEST_SAMPLE // vocab)))
    return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "f16"]), greedy=rng.random() < 0.25, closed=rng.choice([0.0, 0.3]))


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------

CLIP, KL, ENTROPY, GAMMA, LAM = 0.2, 0.05, 0.01, 0.99, 0.95


def _normal(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    flat = x.view(-1)
    for i in range(0, flat.numel(), 1 << 27):           # in pieces: the values pass through 32 bits
        part = flat[i:i + (1 << 27)]
        part.copy_(torch.randn(part.shape, generator=g, device=DEV).mul_(scale))
    return x


def _logits(case, g):
    """Logits as a head leaves them; with row_gap they are the first columns of a wider head, and `closed` is the share of columns that a mask has
    set to -inf (the lowest-numbered column always stays open)."""
    rows, vocab = case["rows"], case["vocab"]
    wide = _normal(g, (rows, vocab + case.get("row_gap", 0)), TYPES[case["dtype"]], 2.0)
    x = wide[:, :vocab]
    if case["closed"]:
        shut = torch.rand((vocab,), generator=g, device=DEV) < case["closed"]
        shut[0] = False
        x[:, shut] = float("-inf")
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    if op == "linear":
        rows, k, n, dt = case["rows"], case["k"], case["n"], TYPES[case["dtype"]]
        if case["obs"]:                                  # object types 0..10, colours 0..5 and states 0..2 in turn, as an observation holds them
            x = torch.randint(0, 1 << 30, (rows, k), generator=g, device=DEV)
            top = torch.tensor([11, 6, 3], device=DEV)[torch.arange(k, device=DEV) % 3]
            x = (x % top).to(torch.uint8)
        else:
            x = _normal(g, (rows, k), dt)
        s = dict(case=case, x=x, w=_normal(g, (n, k), dt, (0.2 if case["obs"] else 1.0) / math.sqrt(k)),
                 b=_normal(g, (n,), dt, 0.1) if case["bias"] else None, r=_normal(g, (rows, n), dt) if case["residual"] else None)
        if case["train"]:
            s["dy"] = _normal(g, (rows, n), dt)
            for key in ("x", "w", "b", "r"):
                if s[key] is not None and s[key].is_floating_point():
                    s[key].requires_grad_(True)
        return s
    if op == "policy_loss":
        rows, vocab = case["rows"], case["vocab"]
        x = _logits(case, g)
        a = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        if case["closed"]:
            a = torch.where(torch.isinf(x.gather(1, a[:, None])[:, 0]), torch.zeros_like(a), a)
        lp = torch.empty(rows, device=DEV)
        step = max(1, (1 << 26) // vocab)
        for i in range(0, rows, step):
            part = x[i:i + step].float()
            lp[i:i + step] = part.gather(1, a[i:i + step, None])[:, 0] - part.logsumexp(1)
        noise = lambda scale: torch.randn((rows,), generator=g, device=DEV) * scale
        mask = torch.rand((rows,), generator=g, device=DEV) >= case["padded"]
        # half-precision gradients of a mean over many rows would be subnormal: training scales the loss, by about the number of rows here
        scale = 2.0 ** int(math.log2(rows)) if case["dtype"] == "f16" else 1.0
        return dict(case=case, x=x.requires_grad_(True), a=a, old=lp + noise(0.15), adv=noise(1.0), mask=mask,
                    ref=lp + noise(0.3) if case["ref"] else None, scale=torch.tensor(scale, device=DEV))
    if op == "advantages":
        t, n = case["steps"], case["envs"]
        # reward and flags as the environments hand them out: fields of one 16-byte record per environment and step
        rec = torch.zeros((t, n, 16), dtype=torch.uint8, device=DEV)
        ends = torch.rand((t, n), generator=g, device=DEV) < case["done"]
        if case["next_step"]:                            # the step behind an end only resets
            for i in range(1, t):
                ends[i] &= ~ends[i - 1]
        cut = torch.rand((t, n), generator=g, device=DEV) < 0.5
        reward = rec.view(torch.float64)[:, :, 0]
        reward.copy_(torch.where(ends & ~cut, 1 - 0.9 * torch.rand((t, n), generator=g, device=DEV), torch.zeros((), device=DEV)))
        rec[:, :, 8] = (ends & ~cut).to(torch.uint8)
        rec[:, :, 9] = (ends & cut).to(torch.uint8)
        return dict(case=case, reward=reward, term=rec[:, :, 8], trunc=rec[:, :, 9], value=torch.randn((t, n), generator=g, device=DEV) * 0.3,
                    last=torch.randn((n,), generator=g, device=DEV) * 0.3)
    x = _logits(case, g)
    return dict(case=case, x=x, u=None if case["greedy"] else torch.rand((case["rows"],), generator=g, device=DEV))


# ---- one pass -------------------------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "policy_loss": _own_loss, "advantages": _own_advantages, "sample": _own_sample}[op](state)
    with torch.no_grad():
        return {"linear": _plain_linear, "policy_loss": _plain_loss, "advantages": _plain_advantages, "sample": _plain_sample}[op](state)


def _own_linear(s):
    import minigrid_amd as mg
    y = mg.linear(s["x"], s["w"], s["b"], activation=s["case"]["act"], residual=s["r"])
    if not s["case"]["train"]:
        return {"y": y}
    names = [k for k in ("x", "w", "b", "r") if s[k] is not None and s[k].requires_grad]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def _own_loss(s):
    import minigrid_amd as mg
    loss, stats = mg.policy_loss(s["x"], s["a"], s["old"], s["adv"], mask=s["mask"], ref_log_prob=s["ref"], clip=CLIP,
                                 kl_coef=0.0 if s["ref"] is None else KL, entropy_coef=ENTROPY)
    grad, = torch.autograd.grad(loss, [s["x"]], s["scale"])
    return {"loss": loss.detach(), "stats": stats, "dlogits": grad}


def _own_advantages(s):
    import minigrid_amd as mg
    adv, ret, valid = mg.advantages(s["reward"], s["value"], s["last"], s["term"], s["trunc"], gamma=GAMMA, lam=LAM,
                                    autoreset_mode="next_step" if s["case"]["next_step"] else "same_step")
    return {"advantage": adv, "return": ret, "valid": valid}


def _own_sample(s):
    import minigrid_amd as mg
    action, lp = mg.sample_actions(s["x"], s["u"])
    return {"action": action, "log_prob": lp}


def _plain_linear(s):
    act, dt = s["case"]["act"], s["w"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    if act is None:
        y = z
    elif act == "relu":
        y = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "tanh":
        y = torch.tanh(z)
    elif act == "silu":
        y = z / (1 + torch.exp(-z))
    else:
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y = z * phi
    if s["r"] is not None:
        y = y + s["r"].float()
    if not s["case"]["train"]:
        return {"y": y.to(dt)}
    dy = s["dy"].float()
    if act is None:
        dz = dy
    elif act == "relu":
        dz = torch.where(z > 0, dy, torch.zeros_like(dy))
    elif act == "tanh":
        t = torch.tanh(z)
        dz = dy * (1 - t * t)
    elif act == "silu":
        p = 1 / (1 + torch.exp(-z))
        dz = dy * p * (1 + z * (1 - p))
    else:
        dz = dy * (phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    out = {"y": y.to(dt)}
    if s["x"].is_floating_point():
        out["dx"] = (dz @ w).to(dt)
    out["dw"] = (dz.t() @ x).to(dt)
    if s["b"] is not None:
        out["db"] = dz.sum(0).to(dt)
    if s["r"] is not None:
        out["dr"] = s["dy"].clone()
    return out


def _plain_loss(s):
    x, a, mask = s["x"], s["a"], s["mask"]
    rows, vocab = x.shape
    # the clipping is a border: the row's statistics are held in 64 bits
    xs = x.double() if vocab <= 1024 else x.float()
    top = xs.max(1, keepdim=True).values
    e = torch.exp(xs - top)
    total = e.sum(1, dtype=torch.float64)
    lse = top[:, 0].double() + torch.log(total)
    lp = x.gather(1, a[:, None])[:, 0].double() - lse
    p = (e / total[:, None].to(e.dtype)).float()
    del e
    logp = (xs - lse[:, None].to(xs.dtype)).float()
    logp = torch.where(p > 0, logp, torch.zeros_like(logp))
    del xs
    entropy = -(p * logp).sum(1, dtype=torch.float64)
    adv, old = s["adv"].double(), s["old"].double()
    ratio = torch.exp(lp - old)
    clipped = torch.where(adv >= 0, ratio > 1 + CLIP, ratio < 1 - CLIP)
    bound = torch.where(adv >= 0, torch.full_like(adv, 1 + CLIP), torch.full_like(adv, 1 - CLIP))
    policy = -torch.where(clipped, bound, ratio) * adv
    dlp = torch.where(clipped, torch.zeros_like(adv), -ratio * adv)
    kl = torch.zeros_like(adv)
    if s["ref"] is not None:
        gap = s["ref"].double() - lp
        kl = torch.exp(gap) - gap - 1
        dlp = dlp + KL * (1 - torch.exp(gap))
    count = mask.sum()
    share = mask.double() / count.clamp(min=1)
    zero = torch.zeros_like(adv)
    mean = lambda v: (torch.where(mask, v, zero) * share).sum()
    loss = mean(policy + KL * kl - ENTROPY * entropy)
    stats = torch.stack([mean(policy), mean(kl), mean(entropy), mean(clipped.double()), count.double()])
    share = share * s["scale"]
    dlp = (dlp * share).float()
    share = share.float()
    grad = logp + entropy[:, None].float()
    grad = p * (ENTROPY * share[:, None] * grad - dlp[:, None])
    grad.scatter_add_(1, a[:, None], dlp[:, None])
    grad = torch.where(mask[:, None], grad, torch.zeros((), device=grad.device))
    return {"loss": loss.float(), "stats": stats.float(), "dlogits": grad.to(x.dtype)}


def _plain_advantages(s):
    reward, value = s["reward"], s["value"].double()
    term, trunc = s["term"] != 0, s["trunc"] != 0
    t, n = value.shape
    ends = term | trunc
    resets = torch.zeros_like(ends)
    if s["case"]["next_step"]:
        resets[1:] = ends[:-1]
    adv = torch.zeros((t, n), dtype=torch.float64, device=DEV)
    after = torch.cat([value[1:], s["last"].double()[None]])
    # a terminated step is worth its reward; a truncated one is bootstrapped from the observation it ended on where the next step shows it
    worth = torch.where(term if s["case"]["next_step"] else ends, torch.zeros_like(after), after)
    delta = reward + GAMMA * worth - value
    carry = torch.zeros((n,), dtype=torch.float64, device=DEV)
    for i in range(t - 1, -1, -1):
        carry = torch.where(ends[i], delta[i], delta[i] + GAMMA * LAM * carry)
        carry = torch.where(resets[i], torch.zeros_like(carry), carry)
        adv[i] = carry
    return {"advantage": adv.float(), "return": (adv + value).float(), "valid": ~resets}


def _plain_sample(s):
    x = s["x"].double()                                  # a drawn number next to a border of the distribution decides: 64 bits
    top, best = x.max(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    vocab = x.shape[1]
    index = torch.arange(vocab, device=DEV)
    if s["u"] is None:
        action = torch.where(x == top, index, vocab).min(1).values
    else:
        run_sum = torch.cumsum(e, 1)
        action = torch.where(run_sum > s["u"].double()[:, None] * total, index, vocab).min(1).values
        last = torch.where(e > 0, index, -1).max(1).values
        action = torch.minimum(action, last)
    lp = x.gather(1, action[:, None])[:, 0] - top[:, 0] - torch.log(total[:, 0])
    return {"action": action.to(torch.uint8 if vocab <= 256 else torch.int32), "log_prob": lp.float()}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "linear":
        m, k, n, b = case["rows"], case["k"], case["n"], 4 if case["dtype"] == "f32" else 2
        xb = 1 if case["obs"] else b
        one = m * k * xb + n * k * b + m * n * b + (n * b if case["bias"] else 0) + (m * n * b if case["residual"] else 0)
        flops = 2 * m * n * k
        if not case["train"]:
            return {"bytes": one, "flops": flops}
        more = m * n * b + n * k * b + (0 if case["obs"] else m * k * b) + (n * b if case["bias"] else 0) + (m * n * b if case["residual"] else 0)
        return {"bytes": one + more, "flops": flops * (2 if case["obs"] else 3)}
    if op == "policy_loss":
        m, v, b = case["rows"], case["vocab"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * m * v * b + m * (8 + 4 + 4 + 1 + (4 if case["ref"] else 0)) + 24, "flops": 8 * m * v}
    if op == "advantages":
        m = case["steps"] * case["envs"]
        return {"bytes": m * (8 + 1 + 1 + 4 + 4 + 4 + 1) + 4 * case["envs"], "flops": 8 * m}
    m, v, b = case["rows"], case["vocab"], 4 if case["dtype"] == "f32" else 2
    return {"bytes": m * v * b + m * (4 + (0 if case["greedy"] else 4) + (1 if v <= 256 else 4)), "flops": 4 * m * v}


# ---- the definitions in 64 bits, apart from the plain forms ------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "policy_loss": _exact_loss, "advantages": _exact_advantages, "sample": _exact_sample}[case["op"]](s)


def _exact_linear(s):
    act, train = s["case"]["act"], s["case"]["train"]
    leaf = {}
    for key in ("x", "w", "b", "r"):
        if s[key] is not None:
            leaf[key] = s[key].detach().double()
            if train and s[key].is_floating_point():
                leaf[key].requires_grad_(True)
    with torch.set_grad_enabled(train):
        z = torch.nn.functional.linear(leaf["x"], leaf["w"], leaf.get("b"))
        fn = {None: lambda v: v, "relu": torch.relu, "tanh": torch.tanh, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[act]
        y = fn(z) + leaf["r"] if "r" in leaf else fn(z)
    if not train:
        return {"y": y}
    names = [k for k in ("x", "w", "b", "r") if k in leaf and leaf[k].requires_grad]
    grads = torch.autograd.grad(y, [leaf[k] for k in names], s["dy"].double())
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def _exact_loss(s):
    rows, vocab = s["x"].shape
    count = int(s["mask"].sum())
    ref = s["ref"]
    sums = torch.zeros(4, dtype=torch.float64, device=DEV)
    grad = torch.zeros((rows, vocab), dtype=torch.float64, device=DEV)
    kept = s["mask"].nonzero()[:, 0]
    step = max(1, (1 << 25) // vocab)
    for i in range(0, count, step):
        at = kept[i:i + step]
        x = s["x"].detach()[at].double().requires_grad_(True)
        lp = torch.log_softmax(x, 1)
        mine = lp.gather(1, s["a"][at, None])[:, 0]
        p = lp.exp()
        entropy = -(p * lp.masked_fill(torch.isinf(lp), 0.0)).sum(1)
        ratio = (mine - s["old"][at].double()).exp()
        adv = s["adv"][at].double()
        policy = torch.maximum(-ratio * adv, -ratio.clamp(1 - CLIP, 1 + CLIP) * adv)
        kl = torch.zeros_like(policy)
        if ref is not None:
            d = ref[at].double() - mine
            kl = d.exp() - 1 - d
        total = ((policy + KL * kl - ENTROPY * entropy) / count).sum()
        grad[at] = torch.nan_to_num(torch.autograd.grad(total, x, s["scale"].double())[0])
        clipped = ((ratio > 1 + CLIP) & (adv >= 0)) | ((ratio < 1 - CLIP) & (adv < 0))
        sums += torch.stack([v.detach().double().sum() for v in (policy, kl, entropy, clipped)]) / count
    loss = sums[0] + KL * sums[1] - ENTROPY * sums[2]
    return {"loss": loss, "stats": torch.cat([sums, torch.tensor([float(count)], dtype=torch.float64, device=DEV)]), "dlogits": grad}


def _exact_advantages(s):
    import numpy as np
    r, v, last = (s[k].cpu().numpy().astype(np.float64) for k in ("reward", "value", "last"))
    term, trunc = (s[k].cpu().numpy() != 0 for k in ("term", "trunc"))
    steps, envs = v.shape
    valid = np.ones((steps, envs), bool)
    adv = np.zeros((steps, envs))
    held, seen = np.zeros(envs), last
    if s["case"]["next_step"]:
        valid[1:] = ~(term | trunc)[:-1]
    for i in reversed(range(steps)):
        gone = term[i] if s["case"]["next_step"] else term[i] | trunc[i]
        now = r[i] - v[i] + GAMMA * np.where(gone, 0.0, seen) + GAMMA * LAM * np.where(term[i] | trunc[i], 0.0, held)
        held = np.where(valid[i], now, 0.0)
        seen = v[i]
        adv[i] = held
    back = lambda z: torch.from_numpy(np.ascontiguousarray(z)).to(DEV)
    return {"advantage": back(adv), "return": back(adv + v), "valid": back(valid)}


def _exact_sample(s):
    x = s["x"].double()
    rows, vocab = x.shape
    p = torch.softmax(x, 1)
    if s["u"] is None:
        action = ((x == x.max(1, keepdim=True).values).cumsum(1) == 0).sum(1)
    else:
        action = (p.cumsum(1) <= s["u"].double()[:, None] * p.sum(1, keepdim=True)).sum(1)
        action = torch.minimum(action, vocab - 1 - (p.flip(1) > 0).to(torch.uint8).argmax(1))
    lp = torch.log_softmax(x, 1).gather(1, action[:, None])[:, 0]
    return {"action": action.to(torch.uint8 if vocab <= 256 else torch.int32), "log_prob": lp}
