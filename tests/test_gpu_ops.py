"""The learning operators (minigrid_amd/ops.py) against their formulas in 64 bits on the same inputs.

Tolerances come from arithmetic, element by element.  A sum of d products in 32 bits, whatever its order, is off by at most (d + 2) 2^-24 of the sum of
the products' magnitudes; rounding a result to its type by half a step, H = finfo.eps / 2 of its value (plus half of the smallest f16 step); the
elementary functions used are good to EL = 2^-20 of their value (a handful of 2^-24 each).  What enters a later sum enters with its own bound."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24
EL = 2.0 ** -20
ACTS = [None, "relu", "tanh", "gelu", "silu"]


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else 1e-37


def mg():
    import minigrid_amd
    return minigrid_amd


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        at = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {float(got[tuple(at)])} for {float(want[tuple(at)])}, "
                             f"tolerance {float(torch.as_tensor(tol).expand_as(got)[tuple(at)])}")


# ---- linear -----------------------------------------------------------------------------------------------------------------------------

def act64(name, z):
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    phi = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def linear_inputs(rows, k, n, dt, obs, bias, res, exact, seed):
    g = gen(seed)
    if exact:       # small integers over 4: every sum is exact, so that relu's border is where it is
        r = lambda *s: (torch.randint(-3, 4, s, generator=g, device="cuda").double() / 4).to(dt)
    else:
        r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
    x = torch.randint(0, 11, (rows, k), generator=g, device="cuda", dtype=torch.uint8) if obs else r(rows, k)
    w = r(n, k)
    if not exact:
        w = (w.float() / math.sqrt(k) / (3 if obs else 1)).to(dt)
    return x, w, r(n) if bias else None, r(rows, n) if res else None, r(rows, n)


def check_linear(x, w, b, r, dy, act, got):
    """got: y, dx, dw, db (None where not wanted)"""
    y, dx, dw, db = got
    dt, H, tn = w.dtype, half(w.dtype), tiny(w.dtype)
    (rows, k), n = x.shape, w.shape[0]
    X, W, DY = x.double(), w.double(), None if dy is None else dy.double()
    z, S = X @ W.t(), X.abs() @ W.abs().t()
    if b is not None:
        z, S = z + b.double(), S + b.double().abs()
    ez = (k + 4) * U * S
    a, d = act64(act, z)
    want = a if r is None else a + r.double()
    within(y, want, 1.13 * ez + EL * a.abs() + (H + U) * (want.abs() + (0 if r is None else r.double().abs() * U)) + tn, "y")
    if dy is None:
        return
    dz = DY * d
    # the kept z is rounded; no second derivative here is above 0.8; relu's slope does not change with it
    slope = torch.zeros_like(z) if act in (None, "relu") else 0.8 * (H * z.abs() + (1 + H) * ez + tn)
    es = DY.abs() * (slope + (0 if act in (None, "relu") else EL))
    ed = es + H * (dz.abs() + es) + tn if act is not None else torch.zeros_like(dz)
    if dx is not None:
        want = dz @ W
        within(dx, want, (ed @ W.abs()) * 1.01 + (n + 4) * U * ((dz.abs() + ed) @ W.abs()) + H * 1.01 * want.abs() + H * (ed @ W.abs()) + tn, "dx")
    if dw is not None:
        want = dz.t() @ X
        within(dw, want, (ed.t() @ X.abs()) * 1.01 + (rows + 4) * U * ((dz.abs() + ed).t() @ X.abs()) + H * 1.01 * want.abs() + H * (ed.t() @ X.abs()) + tn, "dw")
    if db is not None:
        want = dz.sum(0)
        within(db, want, es.sum(0) * 1.01 + (rows + 4) * U * (dz.abs() + es).sum(0) + H * 1.01 * want.abs() + H * es.sum(0) + tn, "db")


def run_linear(x, w, b, r, dy, act):
    leaves = {"x": x, "w": w, "b": b, "r": r}
    leaves = {q: t.detach().requires_grad_(t.is_floating_point()) if t is not None else None for q, t in leaves.items()}
    y = mg().linear(leaves["x"], leaves["w"], leaves["b"], activation=act, residual=leaves["r"])
    names = [q for q, t in leaves.items() if t is not None and t.requires_grad]
    grads = dict(zip(names, torch.autograd.grad(y, [leaves[q] for q in names], dy)))
    if r is not None:
        assert torch.equal(grads["r"], dy)
    return y.detach(), grads.get("x"), grads.get("w"), grads.get("b")


SIZES = [(1, 1, 1), (1, 147, 64), (3, 5, 7), (17, 147, 8), (33, 64, 33), (64, 8, 8), (100, 147, 256), (129, 130, 131), (257, 333, 65), (1000, 72, 1), (31, 1000, 300),
         (2049, 40, 136), (300, 513, 257), (5, 4096, 130), (512, 512, 512)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_linear_sizes(size, dt):
    rows, k, n = size
    act = ACTS[(rows + k + n) % 5]
    obs = (rows + n) % 3 == 0
    x, w, b, r, dy = linear_inputs(rows, k, n, DT[dt], obs, rows % 2 == 1, n % 2 == 1, act == "relu", rows + k)
    check_linear(x, w, b, r, dy, act, run_linear(x, w, b, r, dy, act))


# products large enough for the largest tiles: whole rows of 16 bytes and odd ones, edges that stick out of a tile, and a rest behind the last whole piece of
# the summed axis, in the forward product and both of the backward pass's (4104, 1032 and 2056 are 8 more than a multiple of 64)
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("size,act,obs", [((4104, 1032, 2056), "gelu", False), ((4096, 1024, 2048), None, False), ((4103, 1031, 2055), "silu", False), ((4104, 1083, 2056), "relu", True)])
def test_linear_large_tiles(size, act, obs, dt):
    rows, k, n = size
    x, w, b, r, dy = linear_inputs(rows, k, n, DT[dt], obs, True, act == "gelu", act == "relu", 11)
    check_linear(x, w, b, r, dy, act, run_linear(x, w, b, r, dy, act))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_linear_large_tiles_whatever_the_alignment(dt):
    """the same numbers from rows at 16-byte addresses and from copies at others"""
    rows, k, n = 4104, 1032, 2056
    x, w, b, r, dy = linear_inputs(rows, k, n, DT[dt], False, True, True, False, 12)
    shift = lambda t, by: torch.nn.functional.pad(t, (by, 16 - by))[:, by:by + t.shape[1]]
    want = run_linear(x, w, b, r, dy, "silu")
    for by in (8, 3):
        got = run_linear(shift(x, by), shift(w, by), b, shift(r, by), shift(dy, by), "silu")
        assert all(torch.equal(p, q) for p, q in zip(want, got)), by


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("obs", [False, True])
def test_linear_activations(dt, act, obs):
    x, w, b, r, dy = linear_inputs(200, 75, 96, DT[dt], obs, True, True, act == "relu", 7)
    check_linear(x, w, b, r, dy, act, run_linear(x, w, b, r, dy, act))
    with torch.no_grad():
        check_linear(x, w, b, r, None, act, (mg().linear(x, w, b, activation=act, residual=r), None, None, None))
        check_linear(x, w, None, None, None, act, (mg().linear(x, w, activation=act), None, None, None))


@pytest.mark.parametrize("dt", list(DT))
def test_linear_strides_and_offsets(dt):
    """rows with a gap, rows at odd addresses, a transposed weight, a sliced observation: the same numbers as from packed copies"""
    g = gen(3)
    wide = torch.randn((70, 200), generator=g, device="cuda").to(DT[dt])
    w = torch.randn((150, 48), generator=g, device="cuda").to(DT[dt])
    b = torch.randn((49,), generator=g, device="cuda").to(DT[dt])[1:]
    res = torch.randn((70, 99), generator=g, device="cuda").to(DT[dt])
    for x in (wide[:, 1:151], wide[:, 8:158], wide[::2, 50:], wide.t()[:150].t()):
        with torch.no_grad():
            r = res[:x.shape[0], 3:51]
            got = mg().linear(x, w.t(), b, activation="gelu", residual=r)
            assert torch.equal(got, mg().linear(x.contiguous(), w.t().contiguous(), b.clone(), activation="gelu", residual=r.contiguous()))
    obs = torch.randint(0, 11, (40, 7, 7, 3), generator=g, device="cuda", dtype=torch.uint8)
    w = torch.randn((32, 147), generator=g, device="cuda").to(DT[dt])
    with torch.no_grad():
        want = mg().linear(obs.reshape(40, 147), w)
        assert torch.equal(mg().linear(obs.reshape(5, 8, 147), w).reshape(40, 32), want)
        assert torch.equal(mg().linear(obs.view(-1)[147:].view(39, 147), w), want[1:])
    x = torch.randn((6, 33), generator=g, device="cuda").to(DT[dt]).requires_grad_(True)
    w = torch.randn((9, 33), generator=g, device="cuda").to(DT[dt]).requires_grad_(True)
    a = torch.autograd.grad(mg().linear(x, w, activation="tanh").sum(), [x, w])          # the gradient comes as one broadcast number
    b = torch.autograd.grad(mg().linear(x, w, activation="tanh"), [x, w], torch.ones((6, 9), device="cuda", dtype=DT[dt]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_linear_rows_far_apart():
    """rows of the residual 2^21 elements apart, of x 2^23: more than 32-bit offsets within a tile reach; the same numbers as from packed copies"""
    rows, k, n = 300, 136, 264
    x, w, b, r, dy = linear_inputs(rows, k, n, torch.bfloat16, False, True, True, False, 13)
    for shift in (21, 23):
        far = torch.empty((rows, 1 << shift), dtype=torch.bfloat16, device="cuda")
        far[:, :n] = r
        far[:, n:n + k] = x
        want = run_linear(x, w, b, r, dy, "gelu")
        for got in (run_linear(x, w, b, far[:, :n], dy, "gelu"), run_linear(far[:, n:n + k], w, b, r, dy, "gelu")):
            assert all(torch.equal(p, q) for p, q in zip(want, got)), shift


def test_linear_against_differences():
    g = gen(11)
    f = lambda *s: torch.randn(s, generator=g, device="cuda")
    x, w, b, r, dy = f(19, 21), f(13, 21) / 4, f(13), f(19, 13), f(19, 13)
    for act in ("tanh", "gelu", "silu"):
        _, dx, dw, db = run_linear(x, w, b, r, dy, act)
        value = lambda x, w, b: float((mg().linear(x, w, b, activation=act, residual=r).double() * dy.double()).sum())
        for name, grad, at in (("x", dx, 0), ("w", dw, 1), ("b", db, 2)):
            v = f(*grad.shape)
            v = v / v.norm()
            h, args = 2.0 ** -6, [x, w, b]
            lo, hi = list(args), list(args)
            hi[at], lo[at] = args[at] + h * v, args[at] - h * v
            fd = (value(*hi) - value(*lo)) / (2 * h)
            # the central difference is off by h^2 / 6 of the third derivative along v (none of these functions has one above 2; a step of x or w moves z by
            # at most its row's norm times |v|), and by the sums' rounding over 2 h
            move = {"x": w.double().norm(dim=1).max(), "w": x.double().norm(dim=1).max(), "b": torch.ones((), device="cuda").double()}[name]
            size = float((x.double().abs() @ w.double().abs().t() + b.double().abs() + r.double().abs()).mul(dy.double().abs()).sum())
            tol = h * h / 6 * 2 * float(move) ** 3 * float(dy.abs().max()) * math.sqrt(dy.numel()) + 30 * U * size / h
            assert abs(fd - float((grad.double() * v.double()).sum())) <= tol, (act, name, fd, tol)


def test_linear_nan_and_infinity_stay_in_their_rows():
    x, w, b, r, dy = linear_inputs(70, 40, 50, torch.bfloat16, False, True, False, False, 1)
    want = mg().linear(x, w, b, activation="gelu")
    x2 = x.clone()
    x2[3], x2[69] = float("nan"), float("inf")
    got = mg().linear(x2, w, b, activation="gelu")
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[3] = keep[69] = False
    assert torch.equal(got[keep], want[keep]) and bool(got[3].isnan().all())
    assert bool(mg().linear(x2[3:4], w, activation="relu").isnan().all()) and bool(mg().linear(x2[3:4], w, activation="tanh").isnan().all())


def test_linear_without_rows():
    w = torch.randn((4, 6), device="cuda", requires_grad=True)
    b = torch.randn(4, device="cuda", requires_grad=True)
    x = torch.empty((0, 6), device="cuda", requires_grad=True)
    y = mg().linear(x, w, b, activation="gelu")
    assert y.shape == (0, 4)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert dx.shape == (0, 6) and not bool(dw.any()) and not bool(db.any())


def test_linear_only_some_gradients():
    x, w, b, r, dy = linear_inputs(50, 24, 40, torch.bfloat16, False, True, True, False, 5)
    full = run_linear(x, w, b, r, dy, "silu")
    for name, want in (("x", full[1]), ("w", full[2]), ("b", full[3]), ("r", dy)):
        t = {"x": x, "w": w, "b": b, "r": r}
        t = {q: v.detach().clone() for q, v in t.items()}
        t[name].requires_grad_(True)
        got, = torch.autograd.grad(mg().linear(t["x"], t["w"], t["b"], activation="silu", residual=t["r"]), [t[name]], dy)
        assert torch.equal(got, want), name


def test_linear_same_tensor_twice():
    """a weight used by two layers, and one tensor as input and residual: the gradients add"""
    g = gen(2)
    w = torch.randn((32, 32), generator=g, device="cuda", requires_grad=True)
    x = torch.randn((20, 32), generator=g, device="cuda", requires_grad=True)
    y = mg().linear(mg().linear(x, w, activation="tanh", residual=x), w, residual=x)
    dx, dw = torch.autograd.grad(y.square().sum(), [x, w])
    X, W = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    Y = (torch.tanh(X @ W.t()) + X) @ W.t() + X
    DX, DW = torch.autograd.grad(Y.square().sum(), [X, W])
    # two layers of depth 32 and 20 rows: every sum below has fewer than 32 terms in each of at most 4 nested sums, bounded by the sums of magnitudes
    a = W.abs().detach()
    h = X.abs().detach() + 1
    top = 2 * (h @ a.t() + X.abs().detach())
    mag_x = top @ a @ a + top @ a + top
    mag_w = top.t() @ h + (top @ a).t() @ X.abs().detach()
    within(dx, DX, 200 * U * mag_x, "dx")
    within(dw, DW, 200 * U * mag_w, "dw")


# ---- policy loss ------------------------------------------------------------------------------------------------------------------------

def loss64(x, a, old, adv, ref, mask, lo, hi, kl, ent, scale=1.0):
    X = x.detach().double().requires_grad_(True)
    keep = torch.ones(x.shape[0], dtype=torch.bool, device="cuda") if mask is None else mask.bool()
    n = int(keep.sum())
    if n == 0:
        return torch.zeros(6, dtype=torch.float64, device="cuda"), torch.zeros_like(X), None
    L = torch.log_softmax(X[keep], 1)
    P = L.exp()
    lp = L.gather(1, a.long()[keep, None])[:, 0]
    ent_rows = -(P * torch.where(P > 0, L, torch.zeros_like(L))).sum(1)
    q, A = (lp - old[keep].double()).exp(), adv[keep].double()
    bound = torch.where(A >= 0, 1.0 + hi, 1.0 - lo)
    clipped = torch.where(A >= 0, q > bound, q < bound)
    pol = -torch.where(clipped, bound.expand_as(q), q) * A
    gap = None if ref is None else ref[keep].double() - lp
    klr = torch.zeros_like(pol) if ref is None else gap.exp() - gap - 1
    loss = (pol + kl * klr - ent * ent_rows).mean()
    grad, = torch.autograd.grad(loss, X, torch.tensor(float(scale), device="cuda", dtype=torch.float64))
    grad = torch.where(torch.isnan(grad) & torch.isinf(X), torch.zeros_like(grad), grad)
    out = torch.stack([loss, pol.mean(), klr.mean(), ent_rows.mean(), clipped.double().mean(), torch.tensor(float(n), device="cuda")]).detach()
    # bounds, per row: what lp is off by, and what that makes of the terms
    V = x.shape[1]
    e = (2 * math.log(V + 1) + 16) * U
    dlp = torch.where(clipped, torch.zeros_like(q), q * A).abs() + (0 if ref is None else kl * (1 - gap.exp()).abs())
    rough = (q * A).abs() + (0 if ref is None else kl * (gap.exp() + 1))
    H = ent_rows
    tol_loss = float(((rough + ent * (H + 3)) * 2 * e).mean().detach()) + 2 * U * float(loss.detach().abs()) + 1e-30
    d = torch.where(P > 0, L, torch.zeros_like(L)).abs()
    E = 2 * e + (d + 4) * 2 * U
    tol = torch.zeros_like(X)
    share = scale / n
    body = P * (dlp[:, None] + ent * (d + H[:, None] + 1)) * E + P * (ent * e * (H[:, None] + 3) + rough[:, None] * 2 * e)
    body = body.scatter_add(1, a.long()[keep, None], (rough * 2 * e + dlp * 4 * U)[:, None])
    tol[keep] = body.detach() * share
    return out, grad.detach(), (tol_loss, tol)


def loss_inputs(rows, vocab, dt, seed, gap=0, padded=0.2, closed=0.0, ref=True):
    g = gen(seed)
    x = (torch.randn((rows, vocab + gap), generator=g, device="cuda") * 2).to(dt)[:, :vocab]
    a = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if closed:
        shut = torch.rand((rows, vocab), generator=g, device="cuda") < closed
        shut.scatter_(1, a[:, None], False)
        x.masked_fill_(shut, float("-inf"))
    lp = torch.log_softmax(x.double(), 1).gather(1, a[:, None])[:, 0]
    f = lambda s: torch.randn((rows,), generator=g, device="cuda", dtype=torch.float64) * s
    mask = torch.rand((rows,), generator=g, device="cuda") >= padded
    return x, a, (lp + f(0.2)).float(), f(1.0).float(), (lp + f(0.3)).float() if ref else None, mask


def check_loss(x, a, old, adv, ref, mask, clip=(0.2, 0.3), kl=0.1, ent=0.01, scale=1.0):
    kl = kl if ref is not None else 0.0
    want, dwant, tols = loss64(x, a, old, adv, ref, mask, clip[0], clip[1], kl, ent, scale)
    X = x.detach().requires_grad_(True)
    loss, stats = mg().policy_loss(X, a, old, adv, mask=mask, ref_log_prob=ref, clip=clip, kl_coef=kl, entropy_coef=ent)
    d, = torch.autograd.grad(loss, X, torch.tensor(scale, device="cuda"))
    assert d.dtype == x.dtype and loss.dtype == torch.float32 and not stats.requires_grad
    if tols is None:
        assert float(loss) == 0 and not bool(stats.any()) and not bool(d.any())
        return loss, stats, d
    tl, td = tols
    within(loss.detach(), want[0], tl, "loss")
    within(stats[:3], want[1:4], tl / min(1.0, kl or 1.0, ent or 1.0) + 4 * U * want[1:4].abs(), "stats")
    within(stats[3:], want[4:], 2 * U * want[4:].abs(), "clipped share and count")
    within(d, dwant, td * 1.01 + half(x.dtype) * 1.01 * dwant.abs() + half(x.dtype) * td + tiny(x.dtype), "dlogits")
    if mask is not None:
        assert not bool(d[~mask.bool()].any())
    with torch.no_grad():
        again, s2 = mg().policy_loss(x.detach(), a, old, adv, mask=mask, ref_log_prob=ref, clip=clip, kl_coef=kl, entropy_coef=ent)
    assert torch.equal(again, loss) and torch.equal(s2, stats)
    return loss, stats, d


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 7), (2, 2), (256, 7), (257, 7), (1000, 3), (63, 31), (65, 32), (130, 64), (5, 65), (300, 100), (7, 1023), (64, 2048), (3, 2049),
                                        (2, 16385), (1, 40961), (5, 131071)])
def test_policy_loss_sizes(dt, rows, vocab):
    gap = (rows + vocab) % 3
    check_loss(*loss_inputs(rows, vocab, DT[dt], rows + vocab, gap=gap, padded=0.0 if rows == 1 else 0.2, ref=vocab % 2 == 1),
               scale=2.0 ** int(math.log2(rows)) if dt == "f16" else 1.0)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("vocab", [7, 200])
def test_policy_loss_closed_actions(dt, vocab):
    check_loss(*loss_inputs(100, vocab, DT[dt], 4, closed=0.5), scale=64.0)


@pytest.mark.parametrize("vocab", [7, 500])
@pytest.mark.parametrize("terms", [(0.0, 0.0), (0.3, 0.0), (0.0, 0.05)])
def test_policy_loss_terms_alone(vocab, terms):
    x, a, old, adv, ref, mask = loss_inputs(90, vocab, torch.float32, 9)
    check_loss(x, a, old, adv, ref, mask, kl=terms[0], ent=terms[1])
    check_loss(x, a, old, adv, ref, None, clip=(0.0, 0.0), kl=terms[0], ent=terms[1])


@pytest.mark.parametrize("vocab", [7, 300])
def test_policy_loss_rows_that_do_not_count_are_not_read(vocab):
    x, a, old, adv, ref, mask = loss_inputs(200, vocab, torch.bfloat16, 21, padded=0.3)
    want = check_loss(x, a, old, adv, ref, mask)
    off = ~mask
    x, old, adv, ref, a = x.clone(), old.clone(), adv.clone(), ref.clone(), a.clone()
    x[off] = float("nan")
    x[off.nonzero()[:5, 0]] = float("inf")
    x[off.nonzero()[5:9, 0]] = float("-inf")
    old[off], adv[off], ref[off], a[off] = float("nan"), float("inf"), float("-inf"), -100
    X = x.requires_grad_(True)
    loss, stats = mg().policy_loss(X, a, old, adv, mask=mask.to(torch.uint8), ref_log_prob=ref, clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.01)
    d, = torch.autograd.grad(loss, X)
    assert torch.equal(loss, want[0]) and torch.equal(stats, want[1]) and torch.equal(d, want[2])


@pytest.mark.parametrize("vocab", [7, 300])
def test_policy_loss_without_a_row_that_counts(vocab):
    x, a, old, adv, ref, mask = loss_inputs(40, vocab, torch.float32, 1)
    check_loss(x, a, old, adv, ref, torch.zeros_like(mask))
    x = torch.empty((0, vocab), device="cuda", requires_grad=True)
    e = torch.empty(0, device="cuda")
    loss, stats = mg().policy_loss(x, torch.empty(0, dtype=torch.int64, device="cuda"), e, e)
    d, = torch.autograd.grad(loss, x)
    assert float(loss) == 0 and not bool(stats.any()) and d.shape == (0, vocab)


@pytest.mark.parametrize("vocab", [7, 300])
@pytest.mark.parametrize("action", [-1, 100000])
def test_policy_loss_action_outside_is_loud(vocab, action):
    x, a, old, adv, ref, _ = loss_inputs(20, vocab, torch.float32, 1)
    a[3] = action
    X = x.clone().requires_grad_(True)
    loss, _ = mg().policy_loss(X, a, old, adv)
    d, = torch.autograd.grad(loss, X)
    assert bool(loss.isnan()) and bool(d[3].isnan().all()) and not bool(d[:3].isnan().any())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,vocab", [(9, 65), (4099, 130), (6, 40961)])
@pytest.mark.parametrize("masked", [False, True])
def test_policy_loss_gradient_whatever_the_factor(dt, rows, vocab, masked):
    """the gradient that is made along with the loss, the one for another factor, and the one of a second pass: factor times the same numbers.  A factor of
    two changes no rounding (f16: gradients of unmasked sums over a few rows are far above the subnormal numbers only for large factors, which is why they
    are compared with a tolerance of half its smallest step)"""
    x, a, old, adv, ref, mask = loss_inputs(rows, vocab, DT[dt], 21)
    x = x.detach().clone().requires_grad_(True)
    make = lambda: mg().policy_loss(x, a, old, adv, mask=mask if masked else None, ref_log_prob=ref, kl_coef=0.1, entropy_coef=0.01)[0]
    one, two = torch.ones((), device="cuda"), torch.full((), 2.0, device="cuda")
    loss = make()
    first, = torch.autograd.grad(loss, [x], one, retain_graph=True)
    kept = first.clone()
    first.zero_()                                                    # (what was handed out is the caller's)
    again, = torch.autograd.grad(loss, [x], one, retain_graph=True)
    twice, = torch.autograd.grad(loss, [x], two)
    assert torch.equal(again, kept)
    other, = torch.autograd.grad(make(), [x], two)
    assert torch.equal(other, twice)
    assert bool(((twice.double() - 2 * kept.double()).abs() <= (2.0 ** -24 * 1.5 if dt == "f16" else 0)).all())
    (2 * make()).backward()
    assert torch.equal(x.grad, twice)
    if masked:
        assert not bool(kept[~mask].any())


@pytest.mark.parametrize("t", [torch.uint8, torch.int32, torch.int64])
def test_policy_loss_action_types_and_shapes(t):
    x, a, old, adv, ref, mask = loss_inputs(60, 7, torch.float32, 13, gap=1)
    want, _ = mg().policy_loss(x, a, old, adv, mask=mask)
    got, _ = mg().policy_loss(x.reshape(5, 12, 7), a.to(t).reshape(5, 12), old.reshape(5, 12), adv.reshape(5, 12), mask=mask.reshape(5, 12))
    assert torch.equal(got, want)
    got, _ = mg().policy_loss(x.t().contiguous().t(), a.to(t), torch.stack([old, old], 1)[:, 1], adv, mask=mask)
    assert torch.equal(got, want)


@pytest.mark.parametrize("vocab", [7, 130])
def test_policy_loss_against_differences(vocab):
    x, a, old, adv, ref, mask = loss_inputs(24, vocab, torch.float32, 17)
    q = (torch.log_softmax(x.double(), 1).gather(1, a[:, None])[:, 0] - old.double()).exp()
    mask = mask & ((q - 0.8).abs() > 0.05) & ((q - 1.3).abs() > 0.05)          # (no row crosses the border within the step)
    run = lambda x: mg().policy_loss(x, a, old, adv, mask=mask, ref_log_prob=ref, clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.05)[0]
    X = x.clone().requires_grad_(True)
    d, = torch.autograd.grad(run(X), X)
    v = torch.randn(x.shape, generator=gen(5), device="cuda")
    v /= v.norm(dim=1, keepdim=True)
    h = 2.0 ** -7
    fd = (float(run(x + h * v)) - float(run(x - h * v))) / (2 * h)
    # each row's loss along a unit direction: exp(lp) and softmax terms with third derivatives below 8 (|q adv| + kl e^gap + ent (H + 1)); the difference also
    # carries two roundings of the loss
    gap = ref.double() - (q.log() + old.double())
    third = 8 * ((q * adv).abs() + 0.1 * gap.exp() + 0.05 * (math.log(vocab) + 1))
    tol = h * h / 6 * float(third[mask].mean()) + 40 * U * float((q * adv).abs()[mask].mean() + 1) / h
    assert abs(fd - float((d.double() * v.double()).sum())) <= tol, (fd, tol)


def test_policy_loss_offsets_beyond_32_bits():
    """the last rows of a logits matrix with more than 2^31 elements: the same gradients as on their own"""
    rows, vocab = 70000, 40960
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device="cuda")
    last, a, old, adv, ref, _ = loss_inputs(16, vocab, torch.bfloat16, 2)
    x[-16:] = last
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    mask[-16:] = True
    pad = lambda t: torch.cat([torch.zeros(rows - 16, dtype=t.dtype, device="cuda"), t])
    X = x.requires_grad_(True)
    loss, _ = mg().policy_loss(X, pad(a), pad(old), pad(adv), mask=mask, ref_log_prob=pad(ref), kl_coef=0.1)
    d, = torch.autograd.grad(loss, X)
    Y = last.clone().requires_grad_(True)
    want, _ = mg().policy_loss(Y, a, old, adv, ref_log_prob=ref, kl_coef=0.1)
    e, = torch.autograd.grad(want, Y)
    assert abs(float(loss) - float(want)) <= 4 * U * abs(float(want)) and torch.equal(d[-16:], e) and not bool(d[:rows - 16].any())


# ---- sampling ---------------------------------------------------------------------------------------------------------------------------

def sample64(x, u):
    X = x.double()
    top = X.max(1, keepdim=True).values
    e = (X - top).exp()
    S = e.sum(1)
    idx = torch.arange(x.shape[1], device="cuda")
    if u is None:
        act = torch.where(X == top, idx, x.shape[1]).min(1).values
    else:
        act = torch.where(e.cumsum(1) > u.double()[:, None] * S[:, None], idx, x.shape[1]).min(1).values
        act = torch.minimum(act, torch.where(e > 0, idx, -1).max(1).values)
    return act, X.gather(1, act[:, None])[:, 0] - top[:, 0] - S.log()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 7), (255, 7), (1000, 7), (64, 31), (65, 64), (9, 65), (33, 256), (33, 257), (10, 4096), (5, 8191), (3, 40961), (2, 131072)])
@pytest.mark.parametrize("greedy", [False, True])
def test_sample_actions(dt, rows, vocab, greedy):
    g = gen(rows * vocab)
    x = (torch.randn((rows, vocab + 1), generator=g, device="cuda") * 2).to(DT[dt])[:, :vocab]
    u = None if greedy else torch.rand((rows,), generator=g, device="cuda")
    act, lp = mg().sample_actions(x, u)
    want, wlp = sample64(x, u)
    assert act.dtype == (torch.uint8 if vocab <= 256 else torch.int32)
    assert torch.equal(act.long(), want)
    within(lp, wlp, 2 * U * wlp.abs() + 1e-9, "log_prob")


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,vocab", [(512, 197), (513, 1024), (600, 1025), (4097, 66), (4100, 1500), (2, 255), (70, 256), (70, 513), (1100, 2600)])
@pytest.mark.parametrize("greedy", [False, True])
def test_sample_actions_ways(dt, rows, vocab, greedy):
    """a wave per row, a workgroup per row, several workgroups per row; pieces that are empty, whole, or hold one element"""
    test_sample_actions(dt, rows, vocab, greedy)


@pytest.mark.parametrize("vocab", [7, 300, 20000])
def test_sample_actions_edges(vocab):
    g = gen(vocab)
    x = torch.randn((64, vocab), generator=g, device="cuda")
    shut = torch.rand((64, vocab), generator=g, device="cuda") < 0.7
    shut[torch.arange(64), torch.randint(0, vocab, (64,), generator=g, device="cuda").cpu()] = False
    x.masked_fill_(shut, float("-inf"))
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        t = torch.full((64,), u, device="cuda")
        act, lp = mg().sample_actions(x, t)
        assert torch.equal(act.long(), sample64(x, t)[0]) and bool(lp.isfinite().all())
        assert not bool(shut.gather(1, act.long()[:, None]).any())
    # equal logits: the border of action k is k / vocab exactly, ties of the greedy draw go to the lowest index
    x = torch.zeros((vocab, vocab if vocab < 1000 else 512), device="cuda")
    n = x.shape[1]
    u = torch.arange(vocab, device="cuda").float() / vocab
    assert torch.equal(mg().sample_actions(x, u)[0].long(), sample64(x, u)[0])
    assert not bool(mg().sample_actions(x)[0].any())
    y = torch.zeros((3, n), device="cuda")
    y[0, 2:], y[1, n - 1], y[2, 3] = 5.0, 9.0, float("nan")
    act, lp = mg().sample_actions(y)
    assert act.tolist() == [2, n - 1, 0] and bool(lp[2].isnan()) and bool(lp[:2].isfinite().all())
    y = torch.full((3, n), float("-inf"), device="cuda")
    y[1, 4], y[2, 1] = float("inf"), -3.0
    for uu in (None, torch.full((3,), 0.3, device="cuda")):
        act, lp = mg().sample_actions(y, uu)
        assert act.tolist() == [0, 0, 1] and lp[:2].isnan().all() and float(lp[2]) == 0.0
    assert mg().sample_actions(torch.zeros((0, n), device="cuda"))[0].shape == (0,)


def test_sample_actions_distribution():
    """shares of 2^20 draws from seven logits, each within five standard deviations"""
    x = torch.tensor([0.0, 1.0, -2.0, 0.5, float("-inf"), 3.0, -1.0], device="cuda").expand(1 << 20, 7)
    act, _ = mg().sample_actions(x, torch.rand(1 << 20, generator=gen(1), device="cuda"))
    p = torch.softmax(x[0].double(), 0)
    share = torch.bincount(act.long(), minlength=7).double() / (1 << 20)
    within(share, p, 5 * (p * (1 - p) / (1 << 20)).sqrt() + 1e-12, "share")


# ---- advantages -------------------------------------------------------------------------------------------------------------------------

def advantages64(r, v, last, term, trunc, gamma, lam, mode, done=None, final=None):
    import numpy as np
    f = lambda t: None if t is None else t.double().cpu().numpy()
    r, v, last, final = f(r), f(v), f(last), f(final)
    term, trunc = term.cpu().numpy() != 0, trunc.cpu().numpy() != 0
    T, N = v.shape
    adv, valid = np.zeros((T, N)), np.ones((T, N), bool)
    for e in range(N):
        run = 0.0
        for t in reversed(range(T)):
            nxt = v[t + 1, e] if t + 1 < T else last[e]
            end = term[t, e] or trunc[t, e]
            if mode == "next_step":
                reset = (term[t - 1, e] or trunc[t - 1, e]) if t else (done is not None and bool(done[e]))
                worth = 0.0 if term[t, e] else nxt
            else:
                reset = False
                worth = 0.0 if term[t, e] else ((final[t, e] if final is not None else 0.0) if trunc[t, e] else nxt)
            run = 0.0 if reset else r[t, e] + gamma * worth - v[t, e] + (0.0 if end else gamma * lam * run)
            adv[t, e], valid[t, e] = run, not reset
    c = lambda a: torch.from_numpy(a).cuda()
    return c(adv), c(adv + v), c(valid)


@pytest.mark.parametrize("steps,envs", [(1, 1), (2, 1), (1, 300), (5, 3), (32, 64), (33, 65), (128, 17), (1000, 2), (2049, 1), (257, 130)])
@pytest.mark.parametrize("mode", ["next_step", "same_step"])
def test_advantages(steps, envs, mode):
    g = gen(steps + envs)
    rec = torch.zeros((steps, envs, 16), dtype=torch.uint8, device="cuda")
    r = rec.view(torch.float64)[:, :, 0]
    r.copy_(torch.randn((steps, envs), generator=g, device="cuda"))
    ends = torch.rand((steps, envs), generator=g, device="cuda")
    term, trunc = rec[:, :, 8], rec[:, :, 9]
    term.copy_(ends < 0.05)
    trunc.copy_((ends > 0.03) & (ends < 0.1))                        # (some steps end both ways)
    vt = [torch.float32, torch.bfloat16, torch.float16][(steps + envs) % 3]
    f = lambda *s: torch.randn(s, generator=g, device="cuda").to(vt)
    v, last = f(envs, steps).t(), f(envs)
    done = torch.rand(envs, generator=g, device="cuda") < 0.3 if mode == "next_step" else None
    final = f(steps, envs) if mode == "same_step" and steps % 2 else None
    if steps % 2 == 0:
        r = r.float()
    args = (r, v, last, term, trunc)
    adv, ret, valid = mg().advantages(*args, gamma=0.97, lam=0.9, autoreset_mode=mode, done=done, final_value=final)
    wa, wr, wv = advantages64(*args, 0.97, 0.9, mode, done, final)
    assert torch.equal(valid, wv)
    within(adv, wa, 1.01 * U * wa.abs() + 1e-12, "advantage")
    within(ret, wr, 1.01 * U * wr.abs() + 1e-12, "return")
    a2, _, _ = mg().advantages(r.contiguous(), v.contiguous(), last, term.bool(), trunc.bool(), gamma=0.97, lam=0.9, autoreset_mode=mode, done=done, final_value=final)
    assert torch.equal(a2, adv)


def test_advantages_nan_stays_behind_an_end_and_in_rows_that_reset():
    T, N = 40, 5
    z = lambda: torch.zeros((T, N), device="cuda")
    r, v, term, trunc = z(), z(), z().byte(), z().byte()
    term[20, 1] = trunc[20, 2] = 1
    r[21] = float("nan")                                             # (a row that only resets for env 1 and 2, an ordinary one for the others)
    v[30, 4] = float("inf")
    adv, ret, valid = mg().advantages(r, v, torch.zeros(N, device="cuda"), term, trunc)
    assert bool(adv[:22, 0].isnan().all()) and bool(adv[22:, 0].eq(0).all())
    assert not bool(adv[:, 1:3].isnan().any()) and valid[21].tolist() == [True, False, False, True, True]
    assert bool(adv[:30, 4].isnan().any())


def test_advantages_empty():
    e = torch.empty((0, 4), device="cuda")
    adv, ret, valid = mg().advantages(e, e, torch.zeros(4, device="cuda"), e.bool(), e.bool())
    assert adv.shape == ret.shape == valid.shape == (0, 4)


# ---- streams, graphs, repetition ----------------------------------------------------------------------------------------------------------

def everything(seed=0, rows=300):
    x, w, b, r, dy = linear_inputs(rows, 147, 72, torch.bfloat16, True, True, True, False, seed)
    head = torch.randn((8, 72), generator=gen(seed + 1), device="cuda").to(torch.bfloat16)
    _, a, old, adv, ref, mask = loss_inputs(rows, 7, torch.bfloat16, seed)
    u = torch.rand(rows, generator=gen(seed), device="cuda")
    w, b, head = w.requires_grad_(True), b.requires_grad_(True), head.requires_grad_(True)

    def step():
        h = mg().linear(x, w, b, activation="gelu", residual=r)
        out = mg().linear(h, head)
        loss, stats = mg().policy_loss(out[:, :7], a, old, adv, mask=mask, ref_log_prob=ref, kl_coef=0.1, entropy_coef=0.01)
        grads = torch.autograd.grad(loss, [w, b, head])
        with torch.no_grad():
            act, lp = mg().sample_actions(out.detach()[:, :7], u)
            flags = mask.view(10, -1)
            gae = mg().advantages(adv.view(10, -1), old.view(10, -1), old[:rows // 10], flags & flags.roll(1, 0), ~flags)
        return (loss.detach(), stats, act, lp) + grads + gae
    return step, (x, r, adv)


def test_same_results_again_and_on_another_stream():
    step, _ = everything()
    first = step()
    for got in (step(), step()):
        assert all(torch.equal(p, q) for p, q in zip(first, got))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_captured_and_replayed():
    """the whole chain with its gradients in two graphs over the same inputs, replayed with new inputs, eager work and each other in between"""
    step, (x, r, adv) = everything()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(4):
        adv.copy_(torch.randn(adv.shape, generator=gen(50 + i), device="cuda"))
        r.copy_(torch.randn(r.shape, generator=gen(90 + i), device="cuda"))
        x.copy_(torch.randint(0, 11, x.shape, generator=gen(70 + i), device="cuda", dtype=torch.uint8))
        want = step()
        for g, out in graphs:
            g.replay()
        if i % 2:
            step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(want, out)), i


@pytest.mark.parametrize("op", ["linear", "policy_loss"])
def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(op):
    """(the backward pass would end the process)"""
    x, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    x = x.contiguous().requires_grad_(True)
    w = torch.randn((5, 7), generator=gen(1), device="cuda", requires_grad=True)
    step = (lambda: mg().linear(x, w, activation="tanh")) if op == "linear" else (lambda: mg().policy_loss(x, a, old, adv)[0])
    alive = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="outside of this capture"):
        with torch.cuda.graph(g):
            step()
    del alive, g
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
        d, = torch.autograd.grad(y.sum(), [x])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(d, torch.autograd.grad(step().sum(), [x])[0])


def test_second_derivatives_are_refused():
    x, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    x = x.contiguous().requires_grad_(True)
    w = torch.randn((5, 7), generator=gen(1), device="cuda", requires_grad=True)
    for y in (mg().linear(x, w, activation="tanh").square().sum(), mg().policy_loss(x, a, old, adv)[0]):
        d, = torch.autograd.grad(y, [x], create_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(d.sum(), [x])


def test_changes_in_place_between_the_passes_are_noticed():
    x, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    w = torch.randn((5, 7), generator=gen(1), device="cuda", requires_grad=True)
    x = x.contiguous()
    y = mg().linear(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), [w])
    L = x.clone().requires_grad_(True)
    loss, stats = mg().policy_loss(L, a, old, adv)
    want, = torch.autograd.grad(loss, [L], retain_graph=True)
    stats.zero_()                                                    # (what was returned is the caller's)
    got, = torch.autograd.grad(loss, [L], retain_graph=True)
    assert torch.equal(got, want)
    a.zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(loss, [L])
    loss = mg().policy_loss(L, a, old, adv)[0]
    torch.autograd.grad(loss, [L])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, [L])


def test_saved_tensor_hooks_and_checkpointing():
    """what the backward pass keeps goes through torch's hooks: recomputed, or moved to the host and back, the gradients are the same"""
    x, w, b, r, dy = linear_inputs(50, 24, 40, torch.bfloat16, False, True, True, False, 5)
    for t in (x, w, b, r):
        t.requires_grad_(True)
    f = lambda: mg().linear(x, w, b, activation="gelu", residual=r)
    want = torch.autograd.grad(f(), [x, w, b, r], dy)
    with torch.autograd.graph.save_on_cpu():
        y = f()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, [x, w, b, r], dy), want))
    from torch.utils.checkpoint import checkpoint
    y = checkpoint(lambda *t: mg().linear(t[0], t[1], t[2], activation="gelu", residual=t[3]), x, w, b, r, use_reentrant=False)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, [x, w, b, r], dy), want))


def test_relu_keeps_its_result():
    """without a residual the backward pass reads relu's result: through hooks and checkpoints the same gradients, and a change of it in place is noticed"""
    x, w, b, _, dy = linear_inputs(70, 24, 40, torch.bfloat16, False, True, False, True, 6)
    for t in (x, w, b):
        t.requires_grad_(True)
    f = lambda *t: mg().linear(*t, activation="relu")
    want = torch.autograd.grad(mg().linear(x, w, b, activation="relu", residual=torch.zeros_like(dy)), [x, w, b], dy)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(f(x, w, b), [x, w, b], dy), want))
    with torch.autograd.graph.save_on_cpu():
        y = f(x, w, b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, [x, w, b], dy), want))
    from torch.utils.checkpoint import checkpoint
    y = checkpoint(f, x, w, b, use_reentrant=False)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, [x, w, b], dy), want))
    y = f(x.view(7, 10, 24), w, b)
    assert torch.equal(torch.autograd.grad(y, [x], dy.view(7, 10, 40))[0], want[0])
    y = f(x, w, b)
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, [x], dy)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_long_rows_captured_and_replayed(dt):
    """the gradient that comes with the loss is made anew by every replay, whatever the caller did to the one before"""
    x, a, old, adv, ref, mask = loss_inputs(37, 700, DT[dt], 4)
    x = x.detach().clone().requires_grad_(True)
    scale = torch.ones((), device="cuda")

    def step():
        loss, stats = mg().policy_loss(x, a, old, adv, mask=mask, ref_log_prob=ref, kl_coef=0.1, entropy_coef=0.01)
        d, = torch.autograd.grad(loss, [x], scale)
        return loss.detach(), stats, d
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(5):
        scale.fill_(1.0 if i % 2 else 0.5 + i)
        adv.copy_(torch.randn(adv.shape, generator=gen(50 + i), device="cuda"))
        mask.copy_(torch.rand(mask.shape, generator=gen(60 + i), device="cuda") < 0.7)
        want = step()
        out[2].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out)), i


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------

def test_refusals():
    m, c = mg(), dict(device="cuda")
    x, w = torch.zeros((4, 8), **c), torch.zeros((6, 8), **c)
    bad = [lambda: m.linear(x, w, activation="swish"), lambda: m.linear(x.half(), w), lambda: m.linear(x.double(), w.double()), lambda: m.linear(x[:, :7], w),
           lambda: m.linear(x, w, torch.zeros(5, **c)), lambda: m.linear(x, w, torch.zeros(6, dtype=torch.bfloat16, **c)), lambda: m.linear(x, w, residual=torch.zeros(6, **c)),
           lambda: m.linear(x, w, residual=torch.zeros((1, 6), **c)), lambda: m.linear(x.cpu(), w), lambda: m.linear(x, w[0]), lambda: m.linear(x[:, :0], w[:, :0])]
    l, a, f = torch.zeros((5, 7), **c), torch.zeros(5, dtype=torch.int64, **c), torch.zeros(5, **c)
    bad += [lambda: m.policy_loss(l, a[:4], f, f), lambda: m.policy_loss(l, a.float(), f, f), lambda: m.policy_loss(l, a, f.double(), f), lambda: m.policy_loss(l, a, f, f, kl_coef=0.1),
            lambda: m.policy_loss(l, a, f, f, clip=1.5), lambda: m.policy_loss(l, a, f, f, clip=(0.1, -0.1)), lambda: m.policy_loss(l, a, f, f, clip=float("nan")),
            lambda: m.policy_loss(l, a, f, f, mask=f), lambda: m.policy_loss(l.double(), a, f, f), lambda: m.policy_loss(l, a, f, f.clone().requires_grad_(True)),
            lambda: m.policy_loss(l, a.cpu(), f, f)]
    bad += [lambda: m.sample_actions(l, f[:4]), lambda: m.sample_actions(l, f.double()), lambda: m.sample_actions(l.clone().requires_grad_(True)), lambda: m.sample_actions(l[:, :0])]
    v, t = torch.zeros((3, 5), **c), torch.zeros((3, 5), dtype=torch.bool, **c)
    bad += [lambda: m.advantages(v, v, f, t, t, autoreset_mode="disabled"), lambda: m.advantages(v[:2], v, f, t, t), lambda: m.advantages(v, v, f[:4], t, t),
            lambda: m.advantages(v, v, f, t.float(), t), lambda: m.advantages(v.half(), v, f, t, t), lambda: m.advantages(v, v, f, t, t, final_value=v),
            lambda: m.advantages(v, v, f, t, t, autoreset_mode="same_step", done=t[0]), lambda: m.advantages(v, v.clone().requires_grad_(True), f, t, t),
            lambda: m.advantages(v, v.double(), f.double(), t, t)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)


# ---- the chain as it is used: environments -> policy -> rollout -> advantages -> loss -> gradients ------------------------------------------

@pytest.mark.parametrize("env_id,mode", [("MiniGrid-Empty-5x5-v0", "next_step"), ("BabyAI-GoToRedBall-v0", "next_step"), ("MiniGrid-DoorKey-5x5-v0", "same_step")])
def test_rollout_of_a_policy(env_id, mode):
    from minigrid_amd.policy import ActorCritic
    n, steps = 96, 80
    envs = mg().make_vec(env_id, n, output="torch", autoreset_mode=mode, max_steps=25)
    twin = mg().make_vec(env_id, n, autoreset_mode=mode, max_steps=25)
    envs.reset(seed=5)
    obs, _ = twin.reset(seed=5)
    torch.manual_seed(0)
    policy = ActorCritic(envs.image_shape, hidden=64, dtype=torch.float32)
    traj = envs.rollout(steps, action_seed=3, policy=policy)
    assert traj.action.shape == (steps, n) and traj.image.shape == (steps, n) + envs.image_shape
    for i in range(steps):                                           # the same environments stepped by hand with the drawn actions
        assert (traj.image[i].cpu().numpy() == obs["image"]).all() and (traj.direction[i].cpu().numpy() == obs["direction"]).all()
        obs, rew, term, trunc, _ = twin.step(traj.action[i].cpu().numpy())
        assert (traj.reward[i].cpu().numpy() == rew).all() and (traj.terminated[i].cpu().numpy() == term).all() and (traj.truncated[i].cpu().numpy() == trunc).all()
    assert bool(traj.truncated.any())
    adv, ret, valid = traj.advantages(0.99, 0.95)
    wa, wr, wv = advantages64(traj.reward, traj.value, traj.last_value, traj.terminated, traj.truncated, 0.99, 0.95, mode, traj.done if mode == "next_step" else None)
    assert torch.equal(valid, wv) and (mode == "same_step" or not bool(valid.all()))
    within(adv, wa, 1.01 * U * wa.abs() + 1e-12, "advantage")
    logits, value = policy(traj.image)
    index = torch.randperm(steps * n, device="cuda")[:1000]
    loss, stats = traj.loss(logits, adv, valid, entropy_coef=0.01)
    part, pstats = traj.loss(logits.reshape(-1, 7)[index], adv, valid, index=index, entropy_coef=0.01)
    assert float(stats[4]) == int(valid.sum()) and float(pstats[4]) == int(valid.reshape(-1)[index].sum())
    # the policy has not moved: every ratio is 1 (up to the rounding of two evaluations), nothing is clipped, and the policy term is minus the mean advantage
    assert float(stats[3]) == 0.0
    assert abs(float(stats[0]) + float(adv.double()[valid].mean())) <= 100 * U * float(adv.abs()[valid].mean())
    total = loss + part + 0.5 * (value - ret).square().mean()
    grads = torch.autograd.grad(total, list(policy.parameters()))
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in grads)
    # a second rollout goes on where the first ended, and the same seed draws the same actions from the same state
    more = envs.rollout(5, action_seed=4, policy=policy)
    assert (more.image[0].cpu().numpy() == obs["image"]).all()
    envs.reset(seed=5)
    assert torch.equal(envs.rollout(10, action_seed=3, policy=policy).action[0], traj.action[0])
    envs.close()
    twin.close()


def test_rollout_of_a_policy_refusals():
    policy = lambda obs: (torch.zeros((8, 7), device="cuda"), torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError, match="output='torch'"):
        mg().make_vec("MiniGrid-Empty-5x5-v0", 8).rollout(4, policy=policy)
    envs = mg().make_vec("MiniGrid-Empty-5x5-v0", 8, output="torch")
    envs.reset(seed=0)
    with pytest.raises(ValueError, match="fused"):
        envs.rollout(4, fused=True, policy=policy)
    with pytest.raises(ValueError, match="steps"):
        envs.rollout(0, policy=policy)
    with pytest.raises(ValueError, match="logits"):
        envs.rollout(4, policy=lambda obs: (torch.zeros((8, 6), device="cuda"), torch.zeros(8, device="cuda")))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), pytest.raises(ValueError, match="stream"):
        envs.rollout(4, policy=policy)
    with pytest.raises(ValueError, match="autoreset"):
        mg().make_vec("MiniGrid-Empty-5x5-v0", 8, output="torch", autoreset_mode="disabled").rollout(4, policy=policy)
    with pytest.raises(ValueError, match="final_obs"):
        mg().make_vec("MiniGrid-Empty-5x5-v0", 8, output="torch", autoreset_mode="same_step", final_obs=True).rollout(4, policy=policy)
