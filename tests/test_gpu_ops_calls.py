"""Calls of the learning operators that their own sizes, masks and types do not reach: two captures, lazily negated tensors, saved-tensor hooks, ratios next to the
clipping border, rollouts one after the other."""
import math
import pickle

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_ops import DT, EL, U, advantages64, check_loss, gen, half, linear_inputs, loss_inputs, mg, run_linear, tiny, within


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_policy_loss_backward_in_a_graph_of_its_own(dt):
    """the loss in one graph, its backward pass in another that is replayed several times behind one replay of the first: every replay gives the gradient of the
    factor that it finds, whatever the one before left and the caller did to it"""
    x, a, old, adv, ref, mask = loss_inputs(37, 700, DT[dt], 4)
    x = x.detach().clone().requires_grad_(True)
    scale = torch.ones((), device="cuda")
    make = lambda: mg().policy_loss(x, a, old, adv, mask=mask, ref_log_prob=ref, kl_coef=0.1, entropy_coef=0.01)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(make(), [x], scale)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward):
        loss = make()
    with torch.cuda.graph(backward, pool=forward.pool()):
        d, = torch.autograd.grad(loss, [x], scale, retain_graph=True)
    want = {f: torch.autograd.grad(make(), [x], torch.full((), f, device="cuda"))[0] for f in (1.0, 2.0)}
    for i in range(2):
        forward.replay()
        for f, spoil in ((1.0, False), (2.0, False), (1.0, False), (1.0, True), (2.0, True), (1.0, False)):
            scale.fill_(f)
            if spoil:
                d.fill_(7.0)
            backward.replay()
            torch.cuda.synchronize()
            assert torch.equal(d, want[f]), (i, f, spoil)


def test_a_tangent_of_the_incoming_gradient_is_refused():
    """(forward over reverse: the gradient's own tangent would be lost)"""
    import torch.autograd.forward_ad as fw
    x, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    x = x.contiguous().requires_grad_(True)
    w = torch.randn((5, 7), generator=gen(1), device="cuda", requires_grad=True)
    for y in (mg().linear(x, w, activation="tanh"), mg().policy_loss(x, a, old, adv)[0]):
        with fw.dual_level():
            g = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises((RuntimeError, ValueError), match="forward-mode"):
                torch.autograd.grad(y, [x], g, retain_graph=True)
        torch.autograd.grad(y, [x], torch.ones_like(y))


def test_a_fake_tensor_beside_real_ones_is_refused():
    """(its address is 0: an optional argument would be taken for one that was not given)"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w, b, r, dy = linear_inputs(50, 24, 40, torch.float32, False, True, True, False, 5)
    l, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    with FakeTensorMode():
        fake = lambda t: torch.empty(t.shape, dtype=t.dtype, device="cuda")
        fb, fr, fref, fmask, fu = fake(b), fake(r), fake(ref), fake(mask), fake(ref)
    for call in (lambda: mg().linear(x, w, fb), lambda: mg().linear(x, w, residual=fr), lambda: mg().policy_loss(l, a, old, adv, mask=fmask),
                 lambda: mg().policy_loss(l, a, old, adv, ref_log_prob=fref), lambda: mg().sample_actions(l, fu)):
        with pytest.raises(ValueError, match="has no memory"):
            call()


# rows of every way that the loss is computed: a lane, a workgroup that holds the row, a workgroup that walks it
@pytest.mark.parametrize("dt,vocab", [("f32", 7), ("f32", 65), ("f32", 100), ("f32", 1000), ("f32", 4099), ("f32", 20487), ("f32", 40961), ("bf16", 64), ("bf16", 100), ("bf16", 1023),
                                      ("bf16", 40961), ("bf16", 90001), ("f16", 300)])
@pytest.mark.parametrize("upper", [True, False])
def test_policy_loss_next_to_the_border(dt, vocab, upper):
    """ratios as close to 1.3 (or 0.8) as f32 log-probabilities allow, on either side: which rows are clipped is what 64 bits say.  (The action's probability is
    about 0.88, so old_log_prob lies below 0.5, where f32 has steps of 3e-8 and less.)"""
    rows = 512
    g = gen(vocab)
    x = (torch.randn((rows, vocab), generator=g, device="cuda") * 2).to(DT[dt])
    a = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    x.scatter_(1, a[:, None], (x.double().logsumexp(1, keepdim=True) + 2).to(DT[dt]))
    lp = torch.log_softmax(x.double(), 1).gather(1, a[:, None])[:, 0]
    border = 1.0 + 0.3 if upper else 1.0 - 0.2
    old = (lp - math.log(border)).float()
    away = lp - old.double() - math.log(border)
    clipped = away > 0 if upper else away < 0
    sure = away.abs() > 1e-13                                        # (64-bit sums of a row's exponentials agree to a few 1e-16)
    assert float(away.abs().max()) < 1e-7 and 0.2 < float(clipped.double().mean()) < 0.8
    adv = torch.full((rows,), 1.0 if upper else -1.0, device="cuda")
    X = x.clone().requires_grad_(True)
    loss, stats = mg().policy_loss(X, a, old, adv, clip=(0.2, 0.3))
    d, = torch.autograd.grad(loss, X)
    got = ~(d != 0).any(1)
    assert torch.equal(got[sure], clipped[sure])
    assert abs(float(stats[3]) * rows - int(got.sum())) < 0.01
    with torch.no_grad():
        again, s2 = mg().policy_loss(x, a, old, adv, clip=(0.2, 0.3))
    assert torch.equal(again, loss) and torch.equal(s2, stats)


def toy_policy(obs):
    """equal logits; the value is a whole number of the observation, so that it does not depend on how it is summed"""
    image = obs["image"]
    n = image.shape[0]
    return torch.zeros((n, 7), device=image.device), image.reshape(n, -1).sum(1).float() + obs["direction"].float()


def toy_envs(n=64, env_id="MiniGrid-Empty-5x5-v0", **kw):
    return mg().make_vec(env_id, n, output="torch", **kw)


def test_rollouts_one_after_the_other_draw_other_numbers():
    """the draws of a seed go on from rollout to rollout, begin again with reset(seed=...), and are others for other environments and other seeds"""
    envs = toy_envs()
    envs.reset(seed=1)
    a, b, c = (envs.rollout(20, policy=toy_policy).action for _ in range(3))
    assert not torch.equal(a, b) and not torch.equal(b, c) and not torch.equal(a, c)
    for e in range(0, 64, 7):                                        # no environment is given the same number at the same step again and again
        assert not torch.equal(a[:, e], b[:, e])
    envs.reset(seed=1)
    again = [envs.rollout(20, policy=toy_policy).action for _ in range(2)]
    assert torch.equal(a, again[0]) and torch.equal(b, again[1])
    envs.reset()                                                     # (goes on)
    assert not torch.equal(envs.rollout(20, policy=toy_policy).action, a)
    envs.reset(seed=1, options={"reset_mask": [1] + [0] * 63})       # (one environment's map, not the draws of all)
    assert not torch.equal(envs.rollout(20, policy=toy_policy).action, a)
    envs.reset(seed=1)
    assert not torch.equal(envs.rollout(20, action_seed=1, policy=toy_policy).action, a)
    other = toy_envs(env_index_base=64)
    other.reset(seed=1)
    assert not torch.equal(other.rollout(20, policy=toy_policy).action, a)
    share = torch.bincount(torch.cat([a, b, c]).flatten().long(), minlength=7).double() / (60 * 64)
    within(share, torch.full((7,), 1 / 7, dtype=torch.float64, device="cuda"), 5 * math.sqrt(6 / 49 / (60 * 64)), "share")
    envs.close()
    other.close()


def test_a_pickled_env_goes_on_drawing():
    envs = toy_envs()
    envs.reset(seed=1)
    a = envs.rollout(20, policy=toy_policy).action
    twin, fresh = pickle.loads(pickle.dumps(envs)), toy_envs()
    fresh.load_state(envs.save_state())
    want = envs.rollout(20, policy=toy_policy).action
    assert not torch.equal(want, a)
    assert torch.equal(twin.rollout(20, policy=toy_policy).action, want) and torch.equal(fresh.rollout(20, policy=toy_policy).action, want)
    for e in (envs, twin, fresh):
        e.close()


@pytest.mark.parametrize("env_id", ["MiniGrid-DoorKey-5x5-v0", "BabyAI-GoToRedBall-v0", "MiniGrid-Dynamic-Obstacles-5x5-v0"])
def test_truncated_steps_are_worth_the_observation_they_ended_on(env_id):
    """same_step with final_obs=True and final_value=True: the policy's value of every terminal observation comes with the trajectory, and its advantages use it"""
    n, steps = 96, 60
    envs, twin = (toy_envs(n, env_id, autoreset_mode="same_step", final_obs=True, max_steps=9) for _ in range(2))
    envs.reset(seed=5)
    obs, _ = twin.reset(seed=5)
    traj = envs.rollout(steps, action_seed=3, policy=toy_policy, final_value=True)
    final = torch.zeros((steps, n), device="cuda")
    for i in range(steps):                                           # the same environments stepped by hand with the drawn actions
        assert torch.equal(traj.image[i], obs["image"]) and torch.equal(traj.direction[i], obs["direction"]) and torch.equal(traj.mission_id[i], obs["mission_id"])
        assert torch.equal(traj.value[i], toy_policy(obs)[1])
        obs, rew, term, trunc, info = twin.step(traj.action[i])
        assert torch.equal(traj.reward[i], rew) and torch.equal(traj.terminated[i].bool(), term) and torch.equal(traj.truncated[i].bool(), trunc)
        if info:
            final[i, info["final_obs_indices"]] = toy_policy(info["final_obs"])[1]
    assert torch.equal(traj.last_value, toy_policy(obs)[1])
    cut = traj.truncated.bool()
    assert int(cut.sum()) > n and torch.equal(traj.final_value[cut], final[cut]) and bool((final[cut] > 0).all())
    adv, ret, valid = traj.advantages(0.97, 0.9)
    args = (traj.reward, traj.value, traj.last_value, traj.terminated, traj.truncated, 0.97, 0.9, "same_step")
    wa, wr, wv = advantages64(*args, None, final)
    assert torch.equal(valid, wv) and bool(valid.all())
    within(adv, wa, 1.01 * U * wa.abs() + 1e-12, "advantage")
    within(ret, wr, 1.01 * U * wr.abs() + 1e-12, "return")
    assert float((wa - advantages64(*args, None, None)[0]).abs().max()) > 1.0                 # (worth 0 otherwise: that is far off here)
    # a second rollout goes on where the first ended
    more = envs.rollout(3, action_seed=4, policy=toy_policy, final_value=True)
    assert torch.equal(more.image[0], obs["image"])
    envs.close()
    twin.close()


def test_final_values_where_there_are_none_are_refused():
    for kw in (dict(), dict(autoreset_mode="same_step")):
        envs = toy_envs(8, **kw)
        envs.reset(seed=0)
        with pytest.raises(ValueError, match="final_obs=True"):
            envs.rollout(4, policy=toy_policy, final_value=True)
        envs.close()
    envs = toy_envs(8, autoreset_mode="same_step", final_obs=True)
    with pytest.raises(ValueError, match="final_value=True"):
        envs.rollout(4, policy=toy_policy)
    with pytest.raises(ValueError, match="policy"):
        envs.rollout(4, final_value=True)
    envs.close()


def test_a_rollout_that_leaves_truncated_steps_worth_nothing_says_so():
    envs = toy_envs(8, autoreset_mode="same_step")
    envs.reset(seed=0)
    with pytest.warns(UserWarning, match="final_value=True"):
        traj = envs.rollout(4, policy=toy_policy)
    assert traj.final_value is None
    envs.close()


def step_until_some_end(envs):
    for _ in range(2000):
        obs, _, term, trunc, _ = envs.step(torch.full((envs.num_envs,), 2, dtype=torch.uint8, device="cuda"))
        if bool((term | trunc).any()):
            return obs, (term | trunc).clone()
    raise AssertionError("no episode ended")


@pytest.mark.parametrize("env_id", ["MiniGrid-DoorKey-5x5-v0", "BabyAI-GoToRedBall-v0", "BabyAI-GoToSeqS5R2-v0"])
def test_rollout_begins_where_the_env_is(env_id):
    """behind a restored checkpoint and behind a masked reset the first observation is the live one, and a step that only resets is known as one"""
    n = 48
    envs = toy_envs(n, env_id, max_steps=6)
    envs.reset(seed=3)
    obs, ended = step_until_some_end(envs)
    image = obs["image"].clone()
    twin = toy_envs(n, env_id, max_steps=6)
    twin.reset(seed=9)
    twin.load_state(envs.save_state())
    pickled = pickle.loads(pickle.dumps(envs))
    want = envs.rollout(9, policy=toy_policy)
    assert torch.equal(want.done, ended) and torch.equal(want.image[0], image)
    for e in (twin, pickled):
        got = e.rollout(9, policy=toy_policy)
        for name in ("image", "direction", "mission_id", "action", "value", "reward", "terminated", "truncated", "done", "last_value"):
            assert torch.equal(getattr(got, name), getattr(want, name)), name
        e.close()
    # a masked reset: the others are still due for theirs
    envs.reset(seed=3)
    obs, ended = step_until_some_end(envs)
    some = [i % 3 == 0 for i in range(n)]
    envs.reset(options={"reset_mask": some})
    done = ended & ~torch.tensor(some, device="cuda")
    traj = envs.rollout(3, policy=toy_policy)
    assert torch.equal(traj.done, done) and torch.equal(traj.advantages()[2][0], ~done)
    envs.close()


def test_rollout_of_restored_obstacles():
    """DynamicObstacles draws its resets when it is observed: a restored env whose reset is due is refused, any other goes on as it would have"""
    n = 48
    envs, twin = (toy_envs(n, "MiniGrid-Dynamic-Obstacles-5x5-v0", max_steps=6) for _ in range(2))
    envs.reset(seed=3)
    step = lambda: envs.step(torch.zeros(n, dtype=torch.uint8, device="cuda"))
    while True:
        _, _, term, trunc, _ = step()
        if not bool((term | trunc).any()):
            break
    twin.reset(seed=9)
    twin.load_state(envs.save_state())
    want, got = envs.rollout(9, policy=toy_policy), twin.rollout(9, policy=toy_policy)
    for name in ("image", "direction", "mission_id", "action", "value", "reward", "terminated", "truncated", "done", "last_value"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    while True:
        _, _, term, trunc, _ = step()
        if bool((term | trunc).any()):
            break
    twin.load_state(envs.save_state())
    with pytest.raises(ValueError, match="reset is due"):
        twin.rollout(9, policy=toy_policy)
    twin.step(torch.zeros(n, dtype=torch.uint8, device="cuda"))
    twin.rollout(2, policy=toy_policy)
    envs.close()
    twin.close()


def test_rollout_behind_fused_steps():
    """(a block of fused steps need not leave its last step in slot 0)"""
    envs = toy_envs(48, "MiniGrid-Empty-5x5-v0", max_steps=20, traj_slots=16)
    envs.reset(seed=3)
    envs.rollout_block(4, 0, slot0=11)
    image, done = envs.torch_outputs(8)["image"].clone(), (envs.torch_outputs(8)["terminated"] | envs.torch_outputs(8)["truncated"]).bool()
    traj = envs.rollout(3, policy=toy_policy)
    assert torch.equal(traj.image[0], image) and torch.equal(traj.done, done)
    envs.close()


def kept_calls():
    """operators whose backward pass reads every kind of tensor that they keep"""
    x, w, b, r, dy = linear_inputs(50, 24, 40, torch.bfloat16, False, True, True, False, 5)
    l, a, old, adv, ref, mask = loss_inputs(41, 7, torch.bfloat16, 3)
    l2, a2, old2, adv2, ref2, mask2 = loss_inputs(41, 130, torch.float32, 3)
    leaf = lambda t: t.detach().clone().requires_grad_(True)
    x, w, b, l, l2 = leaf(x), leaf(w), leaf(b), leaf(l), leaf(l2)
    two = torch.full((), 2.0, device="cuda")
    return {"silu": (lambda: mg().linear(x, w, b, activation="silu"), [x, w, b], dy), "relu": (lambda: mg().linear(x, w, b, activation="relu"), [x, w, b], dy),
            "leading": (lambda: mg().linear(x.view(5, 10, 24), w, b, activation="tanh"), [x, w, b], dy.view(5, 10, 40)),
            "loss": (lambda: mg().policy_loss(l, a, old, adv, mask=mask, ref_log_prob=ref, kl_coef=0.1)[0], [l], two),
            "long loss": (lambda: mg().policy_loss(l2, a2.int(), old2, adv2, mask=mask2, entropy_coef=0.1)[0], [l2], two)}


@pytest.mark.parametrize("name", ["silu", "relu", "leading", "loss", "long loss"])
def test_saved_tensor_hooks_that_give_back_other_strides(name):
    """the same numbers at other addresses: columns first, or every second element of a row"""
    f, leaves, dy = kept_calls()[name]
    want = torch.autograd.grad(f(), leaves, dy)
    for other in (lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() else t.clone(), lambda t: torch.stack([t, t], -1)[..., 0]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            y = f()
        for p, q in zip(torch.autograd.grad(y, leaves, dy), want):
            assert torch.equal(p, q)


@pytest.mark.parametrize("name", ["silu", "relu", "leading", "loss", "long loss"])
def test_saved_tensor_hooks_that_give_back_something_else_are_refused(name):
    """another type, shape or device, one kept tensor at a time"""
    f, leaves, dy = kept_calls()[name]
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t), lambda i: None):
        f()
    assert len(kept) >= 3
    for at in range(len(kept)):
        for other in (lambda t: t.to(torch.float16 if t.dtype != torch.float16 else torch.bfloat16), lambda t: t[:-1], lambda t: t.cpu()):
            count = iter(range(len(kept)))
            with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(count), t), lambda p: other(p[1]) if p[0] == at else p[1]):
                y = f()
            with pytest.raises(RuntimeError, match="saved-tensor hook"):
                torch.autograd.grad(y, leaves, dy)


def test_lazily_negated_tensors():
    """a real tensor whose minus sign is still to be applied (the imaginary part of a conjugated tensor is one): the same numbers as from its values"""
    neg, val = torch._neg_view, lambda t: torch._neg_view(t).resolve_neg()
    c = torch.complex(*(torch.randn((20, 8), generator=gen(i), device="cuda") for i in range(2)))
    assert c.conj().imag.is_neg() and neg(c.real).is_neg()
    x, w, b, r, dy = linear_inputs(50, 24, 40, torch.float32, False, True, True, False, 5)
    leaves = lambda f: [f(t).detach().requires_grad_(True) for t in (x, w, b, r)]
    run = lambda l, g: torch.autograd.grad(mg().linear(l[0], l[1], l[2], activation="silu", residual=l[3]), l, g)
    lazy, plain = leaves(neg), leaves(val)
    assert lazy[0].is_neg() and not plain[0].is_neg()
    assert torch.equal(mg().linear(*lazy[:3], residual=lazy[3]), mg().linear(*plain[:3], residual=plain[3]))
    for p, q in zip(run(lazy, neg(dy)), run(plain, val(dy))):
        assert torch.equal(p, q)
    for vocab in (7, 100):
        l, a, old, adv, ref, mask = loss_inputs(40, vocab, torch.float32, 3)
        out = []
        for f in (neg, val):
            X = f(l).detach().requires_grad_(True)
            loss, stats = mg().policy_loss(X, a, f(old), f(adv), mask=mask, ref_log_prob=f(ref), kl_coef=0.1)
            d, = torch.autograd.grad(loss, X, f(torch.full((), 0.5, device="cuda")))
            act, lp = mg().sample_actions(f(l), f(-torch.rand(40, generator=gen(1), device="cuda")))
            out.append((loss, stats, d, act, lp))
        assert all(torch.equal(p, q) for p, q in zip(*out)), vocab
    t = torch.zeros((20, 8), dtype=torch.bool, device="cuda")
    reward, value = c.conj().imag, neg(c.real)
    last = neg(torch.randn(8, generator=gen(3), device="cuda"))
    for p, q in zip(mg().advantages(reward, value, last, t, t), mg().advantages(reward.resolve_neg(), value.resolve_neg(), last.resolve_neg(), t, t)):
        assert torch.equal(p, q)
    cut = t.clone()
    cut[5] = True
    for p, q in zip(mg().advantages(reward, value, last, t, cut, autoreset_mode="same_step", final_value=value),
                    mg().advantages(reward.resolve_neg(), value.resolve_neg(), last.resolve_neg(), t, cut, autoreset_mode="same_step", final_value=value.resolve_neg())):
        assert torch.equal(p, q)


# few rows, guarded tiles, whole ones, the split and joined, the largest at aligned rows and at odd ones
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,n,res", [(1, 147, 64, False), (8, 30, 33, True), (9, 30, 8, False), (40, 4096, 130, True), (200, 75, 96, False), (300, 513, 257, True), (2049, 300, 136, False),
                                          (4104, 1032, 2056, True), (4103, 1031, 2055, False)])
def test_linear_slope_of_tanh(dt, rows, k, n, res):
    """tanh's slope at a rounded z would be off by 2 |z| half steps of it: what is kept for it is not rounded, so that bias's gradient, which is summed before anything is
    rounded, is off by its own rounding, by that of 32-bit sums, and by EL for the slope"""
    x, w, b, r, dy = linear_inputs(rows, k, n, DT[dt], False, True, res, False, 3)
    w = (w.float() * 2).to(DT[dt])                                   # z as large as 2 and more
    _, _, _, db = run_linear(x, w, b, r, dy, "tanh")
    z, S = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t() + b.double().abs()
    dz = dy.double() * (1 - torch.tanh(z) ** 2)
    es = dy.double().abs() * 0.8 * (k + 4) * U * S + EL * dz.abs()   # (no second derivative is above 0.8)
    want = dz.sum(0)
    within(db, want, es.sum(0) * 1.01 + (rows + 4) * U * (dz.abs() + es).sum(0) + half(DT[dt]) * (1.01 * want.abs() + es.sum(0)) + tiny(DT[dt]), "db")


# rows of every class that a workgroup's registers hold, at its first and last sizes: 16, 32, 80 and 160 KB
@pytest.mark.parametrize("dt,vocab", [(t, n) for t, sizes in (("f32", (4096, 4097, 4099, 4100, 8192, 8193, 8196, 20480, 20483, 20484, 20485, 40959, 40960)),
                                                              ("bf16", (8192, 8193, 8199, 8200, 16384, 16391, 16392, 40960, 40967, 40968, 40969, 81919, 81920)),
                                                              ("f16", (8193, 16385, 40969, 81920))) for n in sizes])
def test_policy_loss_held_rows(dt, vocab):
    for gap, padded in ((0, 0.3), (1, 0.0), (3, 0.3)):
        check_loss(*loss_inputs(11, vocab, DT[dt], vocab + gap, gap=gap, padded=padded, ref=gap != 1), scale=8.0 if dt == "f16" else 1.0)


@pytest.mark.parametrize("dt,vocab", [("f32", 70), ("f32", 5001), ("f32", 20487), ("bf16", 131), ("bf16", 9001), ("bf16", 41003)])
def test_policy_loss_held_rows_several_to_a_workgroup(dt, vocab):
    check_loss(*loss_inputs(8195, vocab, DT[dt], 3, gap=1, padded=0.3))


def recurrence64(r, v, last, term, trunc, gamma, lam, mode, done=None, final=None):
    """(advantages64 with the environments side by side)"""
    T, N = v.shape
    r, v, last = r.double(), v.double(), last.double()
    term, trunc = term != 0, trunc != 0
    ends, zero = term | trunc, torch.zeros(N, dtype=torch.float64, device="cuda")
    resets = torch.zeros_like(ends)
    if mode == "next_step":
        resets[1:] = ends[:-1]
        resets[0] = done != 0 if done is not None else False
    adv, run = torch.zeros_like(v), zero
    for t in reversed(range(T)):
        worth = v[t + 1] if t + 1 < T else last
        if mode == "same_step":
            worth = torch.where(trunc[t], final[t].double() if final is not None else zero, worth)
        worth = torch.where(term[t], zero, worth)
        run = r[t] + gamma * worth - v[t] + torch.where(ends[t], zero, gamma * lam * run)
        run = torch.where(resets[t], zero, run)
        adv[t] = run
    return adv, adv + v, ~resets


@pytest.mark.parametrize("envs", [32768, 32805, 40000])
@pytest.mark.parametrize("steps", [16, 17, 33, 128, 129, 300])
@pytest.mark.parametrize("mode", ["next_step", "same_step"])
def test_advantages_of_many_environments(envs, steps, mode):
    """64 environments a workgroup, one stretch and several, one block of stretches and several"""
    g = gen(steps + envs)
    apart = steps % 2 == 0
    rec = torch.zeros((steps, envs, 16), dtype=torch.uint8, device="cuda")
    r = rec.view(torch.float64)[:, :, 0]
    r.copy_(torch.randn((steps, envs), generator=g, device="cuda"))
    ends = torch.rand((steps, envs), generator=g, device="cuda")
    rec[:, :, 8], rec[:, :, 9] = ends < 0.02, (ends > 0.015) & (ends < 0.04)
    term, trunc = rec[:, :, 8], rec[:, :, 9]
    if apart:
        r, term, trunc = r.float(), term.bool(), trunc.bool()
    vt = [torch.float32, torch.bfloat16, torch.float16][(steps + envs) % 3]
    f = lambda *s: torch.randn(s, generator=g, device="cuda").to(vt)
    v, last = f(steps, envs), f(envs)
    done = torch.rand(envs, generator=g, device="cuda") < 0.3 if mode == "next_step" else None
    final = f(steps, envs) if mode == "same_step" and steps % 3 else None
    args = (r, v, last, term, trunc)
    wa, wr, wv = recurrence64(*args, 0.97, 0.9, mode, done, final)
    adv, ret, valid = mg().advantages(*args, gamma=0.97, lam=0.9, autoreset_mode=mode, done=done, final_value=final)
    assert torch.equal(valid, wv)
    within(adv, wa, 1.01 * U * wa.abs() + 1e-12, "advantage")
    within(ret, wr, 1.01 * U * wr.abs() + 1e-12, "return")


@pytest.mark.parametrize("op", ["linear", "policy_loss"])
def test_capture_of_what_was_made_from_leaves_of_an_eager_graph_is_refused(op):
    """(the backward pass would end the process.)  The leaves may be any number of operations away, and what the capture goes on from may itself be eager"""
    x, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    w = torch.randn((5, 7), generator=gen(1), device="cuda", requires_grad=True)
    x = x.contiguous().requires_grad_(True)
    call = {"linear": lambda x: mg().linear(x, (w * 1.0).detach(), activation="tanh").sum(), "policy_loss": lambda x: mg().policy_loss(x, a, old, adv)[0]}[op]
    step = lambda: call((x * 2.0).tanh())
    alive = x * 3.0                                                  # an eager graph of the leaf
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="outside of this capture"):
        with torch.cuda.graph(g):
            step()
    del alive, g
    before = x * 2.0                                                 # the capture goes on from an eager result
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="outside of this capture"):
        with torch.cuda.graph(g):
            call(before)
    del before, g
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d, = torch.autograd.grad(step(), [x])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(d, torch.autograd.grad(step(), [x])[0])


def test_capture_over_two_streams():
    """a stream that has joined the capture is part of it: what was recorded there is no eager graph"""
    x = torch.randn((40, 7), generator=gen(1), device="cuda", requires_grad=True)
    w, v = (torch.randn((7, 7), generator=gen(i), device="cuda", requires_grad=True) for i in (2, 3))
    want = mg().linear(mg().linear(x, w, activation="tanh"), v).detach().clone()
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            h = mg().linear(x, w, activation="tanh")
        torch.cuda.current_stream().wait_stream(side)
        y = mg().linear(h, v)
    for _ in range(3):
        y.detach().zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("act", ["gelu", "silu", "tanh", "relu"])
@pytest.mark.parametrize("rows", [3, 40, 300])
def test_linear_slope_beyond_the_largest_half(act, rows):
    """values in front of the activation that do not fit 16 bits: far on the negative side the result is 0 and so is the slope, on the positive side the slope is 1 (tanh: 0)"""
    k, n = 64, 72
    x = torch.full((rows, k), 100.0, dtype=torch.float16, device="cuda")
    w = torch.full((n, k), -100.0, dtype=torch.float16, device="cuda")
    w[1::2] = 100.0                                                  # z = -640 000 and 640 000
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    b = torch.zeros(n, dtype=torch.float16, device="cuda", requires_grad=True)
    r = torch.zeros((rows, n), dtype=torch.float16, device="cuda")
    for res in (None, r):
        y = mg().linear(x, w, b, activation=act, residual=res)
        dy = torch.full_like(y, 2.0 ** -10)
        dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
        slope = 0.0 if act == "tanh" else 1.0
        if act != "tanh":
            assert not bool(y[:, ::2].any()) and bool(y[:, 1::2].isinf().all())
        assert not bool(db[::2].any()) and not bool(dw[::2].any())
        # (powers of two and small whole numbers of them: exact up to 2 048 of the smallest)
        assert torch.equal(db[1::2].double(), torch.full((n // 2,), rows * slope * 2.0 ** -10, dtype=torch.float64, device="cuda"))
        want = dw[1::2].double() - rows * slope * 100 * 2.0 ** -10
        assert float(want.abs().max()) <= half(torch.float16) * rows * 100 * 2.0 ** -10
        assert torch.equal(dx.double(), torch.full((rows, k), 36 * slope * 100 * 2.0 ** -10, dtype=torch.float64, device="cuda").half().double())


def test_rollout_behind_a_changed_observation():
    """an observation wrapper changes what the env shows: the first observation of a rollout is the new one"""
    envs, twin = (toy_envs(48, "MiniGrid-DoorKey-5x5-v0", max_steps=20) for _ in range(2))
    twin = mg().FullyObsWrapper(twin)
    envs.reset(seed=3)
    obs, _ = twin.reset(seed=3)
    image = obs["image"].clone()
    envs = mg().FullyObsWrapper(envs)
    got, want = envs.rollout(6, policy=toy_policy), twin.rollout(6, policy=toy_policy)
    assert torch.equal(got.image[0], image)
    for name in ("image", "direction", "mission_id", "action", "value", "reward", "done"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    envs.close()
    twin.close()


@pytest.mark.parametrize("act,kept", [(2, torch.bfloat16), (18, torch.float32)])
@pytest.mark.parametrize("rows,k,n", [(3, 30, 33), (40, 30, 33), (40, 4096, 130), (300, 513, 257), (4104, 1032, 2056)])
def test_c_entry_keeps_z_as_the_header_says(act, kept, rows, k, n):
    """tanh's z in the operands' type, or in 32 bits for MG_ACTIVATION_TANH_Z32: no byte behind (rows, n) of it is written, and the slope is told from it"""
    import ctypes as C

    from minigrid_amd import ops
    L = ops._lib()
    x, w, b, _, dy = linear_inputs(rows, k, n, torch.bfloat16, False, True, False, False, 3)
    z = torch.full((rows * n + 4096,), -7.0, dtype=kept, device="cuda")
    y, dz = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda"), torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    need = C.c_int64()
    assert L.mg_op_linear_workspace(rows, k, n, 1, C.byref(need), None, None) == 0
    ws = torch.empty(need.value + 256, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()
    assert L.mg_op_linear(0, st, 1, 1, act, rows, k, n, p(x), k, p(w), k, p(b), None, 0, p(y), n, p(z), p(ws), need.value) == 0, L.mg_ops_last_error()
    assert L.mg_op_linear_dz(0, st, 1, act, rows, n, p(dy), n, p(z), p(dz), None, None, 0) == 0, L.mg_ops_last_error()
    torch.cuda.synchronize()
    assert bool((z[rows * n:] == -7.0).all())
    Z = x.double() @ w.double().t() + b.double()
    ez = (k + 4) * U * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    within(z[:rows * n].view(rows, n), Z, 1.01 * ez + half(kept) * Z.abs() * 1.01 + 1e-30, "z")
    kz = z[:rows * n].view(rows, n).double()
    want = dy.double() * (1 - torch.tanh(kz) ** 2)
    within(dz, want, 4 * EL * want.abs() + half(torch.bfloat16) * 1.01 * want.abs() + 1e-30, "dz")
    assert L.mg_op_linear(0, st, 1, 1, 17, rows, k, n, p(x), k, p(w), k, p(b), None, 0, p(y), n, p(z), p(ws), need.value) != 0
