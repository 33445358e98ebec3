"""GPU tests of the distillation operators where weights, masks and probabilities are extreme: what one user or one part of
a row holds must not reach the others.  Against the formula in float64 (torch, on the device)."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from recommender_amd import ops
    return ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def inputs(seed, n, M, f, k):
    g = gen(seed)
    X = torch.randn(n, f, generator=g, device="cuda") / f ** 0.25
    Y = torch.randn(M, f, generator=g, device="cuda") / f ** 0.25
    idx = torch.stack([torch.randperm(M, generator=g, device="cuda")[:k] for _ in range(n)]).to(torch.int32)
    val = torch.randn(n, k, generator=g, device="cuda")
    return X, Y, idx, val


# ----------------------------------------------------------------------------- users that ask for nothing
@pytest.mark.parametrize("n", [3, 8, 40])
@pytest.mark.parametrize("bad", [INF, -INF, NAN, 3e37])
def test_an_unknown_user_adds_nothing_whatever_its_weight(ops, n, bad):
    """Its list is like the others'; all products with it are left out, so the items' gradients are the same bits."""
    X, Y, idx, val = inputs(n, n, 70001, 24, 20)
    X *= 50.0                                            # 3e37 x 50 passes float32's range
    users = torch.arange(n, device="cuda")
    users[1] = 10 ** 9
    w = torch.rand(n, generator=gen(5), device="cuda") + 0.5
    w[1] = 0.0
    want = ops.distill_topk(X, Y, users, idx, val, temperature=40.0, weight=w)
    w[1] = bad
    got = ops.distill_topk(X, Y, users, idx, val, temperature=40.0, weight=w)
    assert torch.isfinite(want[2]).all() and torch.equal(got[2], want[2])
    keep = [u for u in range(n) if u != 1]
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])


# ----------------------------------------------------------------------------- the formula in float64
def formula(X, Y, idx, val, T, w):
    """(loss, dX, dY), and the sums of their terms' magnitudes over the users / items; lists hold an item once, -1 is padding.
    Also d: how far a score / T can be off, from operands of 22 bits and float32 sums (2^-20 of the terms' magnitudes)."""
    T = float(torch.tensor(T, dtype=torch.float32))
    X, Y, val, w = X.double(), Y.double(), val.double(), w.double()
    s = X @ Y.T.contiguous() / T
    d = 2.0 ** -20 * (X.abs() @ Y.abs().T.contiguous()).amax(1, keepdim=True) / T
    log_q = torch.log_softmax(s, 1)
    t = torch.softmax(torch.where(idx >= 0, val / T, float("-inf")), 1)
    none = ~torch.isfinite(t).all(1)
    t = torch.where(none[:, None] | (idx < 0), 0.0, t)
    at = idx.clamp(min=0).long()
    loss = torch.where(t > 0, t * (torch.log(t) - log_q.gather(1, at)), 0.0).sum(1)
    q = torch.where(none[:, None], 0.0, log_q.exp())
    slope = q.scatter_add(1, at, -t)
    slope[none] = 0.0
    mag = q.scatter_add(1, at, t)
    c = torch.where(none, 0.0, w / T)[:, None]
    slope, mag = slope * c, mag * c.abs()
    return loss, slope @ Y, slope.T.contiguous() @ X, mag, d


def rel_tolerance(d, terms):
    """Of a term c (q - t) x: both of its scores' errors (the numerator's and ln Z's), the exponential's argument (2^-19: a
    float32 of up to 64), the operands' 22 bits (2^-19 for both), and a float32 sum over `terms` in steps of 16."""
    return 2 * d + 2.0 ** -19 + 2.0 ** -19 + 3 * terms / 16 * 2.0 ** -24


def off_over_tolerance(got, want, tol):
    return float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("n, M, f", [(64, 250001, 16), (20, 1000003, 32), (40, 70001, 64), (33, 90001, 100), (12, 70001, 200)])
def test_items_that_nobody_lists_have_gradients_as_good_as_the_listed(ops, n, M, f):
    """q of 10^-6 and less beside t of up to 1: every element of dY is held to its own terms."""
    X, Y, idx, val = inputs(f, n, M, f, 50)
    X *= 2.0
    w = torch.rand(n, generator=gen(9), device="cuda") + 0.5
    _, dX, dY = ops.distill_topk(X, Y, None, idx, val, weight=w)
    _, _, want, mag, d = formula(X, Y, idx, val, 1.0, w)
    tol = (mag * rel_tolerance(d, n)).T.contiguous() @ X.double().abs()
    tol += 2.0 ** -33 * mag.amax(0)[:, None] * X.double().abs().sum(0)
    assert off_over_tolerance(dY, want, tol) <= 1.0


# ----------------------------------------------------------------------------- weights
def check_formula(ops, X, Y, idx, val, T, w):
    """Every element of dX and dY against the magnitudes of its own terms."""
    loss, dX, dY = ops.distill_topk(X, Y, None, idx, val, temperature=T, weight=w)
    wl, wx, wy, mag, d = formula(X, Y, idx, val, T, w)
    n, M = len(X), len(Y)
    ty = (mag * rel_tolerance(d, n)).T.contiguous() @ X.double().abs()
    # pieces of q - t, a user's row and its share's float32 (below 2^-126 of the largest): one part in 2^33 of an item's largest
    ty += 2.0 ** -33 * (mag * X.double().abs().amax(1, keepdim=True)).sum(0)[:, None]
    tx = rel_tolerance(d, M) * (mag @ Y.double().abs())
    # pieces of a user's weights (2^-34 of its largest, of a part of at most 2^15 items) and of Y (2^-38 of its largest)
    tx += (min(M, 1 << 15) * 2.0 ** -34 * mag.amax(1, keepdim=True) + 2.0 ** -38 * mag.sum(1, keepdim=True)) * Y.double().abs().max()
    assert off_over_tolerance(dY, wy, ty + 1e-300) <= 1.0 and off_over_tolerance(dX, wx, tx + 1e-300) <= 1.0
    assert off_over_tolerance(loss, wl, 1e-4 + 2e-5 * wl.abs()) <= 1.0
    return loss, dX, dY


@pytest.mark.parametrize("n", [3, 8, 40, 300])
@pytest.mark.parametrize("bad", [1e8, 1e12, 1e25, 3e38, -1e30, INF, NAN])
def test_the_weight_of_an_empty_list_reaches_nobody(ops, n, bad):
    """1 / (length + 1e-12) as a weight, say: the same bits as with weight 0."""
    X, Y, idx, val = inputs(n, n, 9000, 24, 20)
    X *= 20.0
    none = [1] if n == 3 else [1, 4, n - 1]
    idx[1] = -1
    if n > 3:
        val[4] = -INF
        idx[n - 1] = 7; val[n - 1, 0] = -INF             # one item, and its first entry asks for nothing
    w = torch.rand(n, generator=gen(6), device="cuda") + 0.5
    w[none] = 0.0
    want = ops.distill_topk(X, Y, None, idx, val, temperature=20.0, weight=w)
    w[none] = bad
    got = ops.distill_topk(X, Y, None, idx, val, temperature=20.0, weight=w)
    for g, v in zip(got, want):
        assert torch.equal(g, v)
    assert torch.isfinite(want[2]).all() and bool(want[2].any())


@pytest.mark.parametrize("n", [8, 40, 700])
@pytest.mark.parametrize("power", [-100, -70, -40, 1, 33, 57, 90])
def test_weights_times_a_power_of_two(ops, n, power):
    """Gradients times the same power of two, bit for bit: nothing about them is relative to 1."""
    X, Y, idx, val = inputs(n + 1, n, 5000, 24, 20)
    w = torch.rand(n, generator=gen(6), device="cuda") + 0.5
    loss, dX, dY = ops.distill_topk(X, Y, None, idx, val, weight=w)
    l2, x2, y2 = ops.distill_topk(X, Y, None, idx, val, weight=w * 2.0 ** power)
    assert torch.equal(loss, l2)
    assert torch.equal(x2.double(), dX.double() * 2.0 ** power) or power < -60      # below float32's normal range
    off = (y2.double() - dY.double() * 2.0 ** power).abs()
    assert bool((off <= 2.0 ** -149).all()) if power < -60 else not off.any()


@pytest.mark.parametrize("n", [8, 40, 300])
@pytest.mark.parametrize("spread", [1.0, 2.0 ** 30, 2.0 ** 60])
def test_users_of_very_different_weight(ops, n, spread):
    """Weights from 1 to `spread`, of either sign.  Half of the users' scores leave some items alone (30 to 80 temperatures below
    the top), so that there the light users' share is what counts."""
    X, Y, idx, val = inputs(n + 2, n, 6000, 16, 20)
    g = gen(7)
    w = spread ** torch.rand(n, generator=g, device="cuda") * torch.where(torch.rand(n, generator=g, device="cuda") < 0.3, -1.0, 1.0)
    w[0], w[1] = 1.0, spread
    Y[:, 0] = 0.0
    Y[1000:1010, 0] = 60.0                               # what the light half ranks first, and the heavy half last
    light = w.abs() < spread ** 0.5
    X[:, 0] = torch.where(light, 0.1, -1.0)
    check_formula(ops, X, Y, idx, val, 1.0, w)


def test_factors_far_from_one_with_weights_that_make_up_for_it(ops):
    for n in (8, 40):
        X, Y, idx, val = inputs(n + 3, n, 5000, 20, 20)
        w = torch.rand(n, generator=gen(6), device="cuda") + 0.5
        for a, b in ((2.0 ** -60, 2.0 ** 60), (2.0 ** 50, 2.0 ** -50), (2.0 ** 112, 2.0 ** -112)):
            want = ops.distill_topk(X, Y, None, idx, val, weight=w)
            loss, dX, dY = ops.distill_topk(X * a, Y * b, None, idx, val, weight=w)
            assert torch.equal(loss, want[0])
            assert torch.equal(dY, want[2] * a)
            if b < 2.0 ** -100:                          # some of dX lies below float32's normal range, in steps of 2^-149
                off = (dX.double() - want[1].double() * b).abs()
                assert bool((off <= 2.0 ** -22 * want[1].double().abs() * b + 2.0 ** -140).all())
                continue
            assert torch.equal(dX, want[1] * b)
            _, dX, dY = ops.distill_topk(X * a, Y * b, None, idx, val, weight=w * b)
            assert torch.equal(dY, want[2])


# ----------------------------------------------------------------------------- long sums
@pytest.mark.parametrize("n", [2, 12, 1 << 16])
def test_a_long_tail_far_below_the_top(ops, n):
    """One item far above a million others at 2^-32 to 2^-34 of it, and a column of Y that is 1: there dX is weight (1 - 1),
    whatever the q are.  A sum of 2^15 items, the part that the top is in, may lose its other terms beside that one, in float32 as
    in the pieces of q (2^-34 each); q and t sums take 2^-20 more."""
    M = (1 << 20) + 3
    Y = torch.zeros(M, 8, device="cuda")
    Y[:, 0] = 1.0
    Y[:, 1] = -math.log(2.0) * (32 + 2 * torch.rand(M, generator=gen(3), device="cuda"))
    Y[5, 1] = 0.0
    X = torch.zeros(16, 8, device="cuda")
    X[:, 1] = torch.linspace(0.98, 1.0, 16)
    users = torch.arange(n, device="cuda") % 16
    idx = torch.tensor([[5, 9]], dtype=torch.int32, device="cuda").repeat(n, 1)
    val = torch.zeros(n, 2, device="cuda")
    loss, dX, dY = ops.distill_topk(X, Y, users, idx, val)
    assert float(dX[:, 0].abs().max()) <= 2.0 ** 15 * (2.0 ** -32 + 2.0 ** -34) + 2.0 ** -20
    s = X.double() @ Y.double().T.contiguous()
    want = -math.log(2.0) - torch.log_softmax(s, 1)[:, [5, 9]].mean(1)
    assert float((loss.double() - want[users]).abs().max()) <= 2.0 ** -16          # of terms up to 24, scores within 2^-18


def test_ln_z_of_many_users(ops):
    """Of so many users that a lane sums half of the items: equal terms, whose roundings in float32 would all fall one way."""
    n, M = 1 << 17, 120001
    Y = torch.zeros(M, 8, device="cuda")
    Y[:, 0] = 1.0
    Y[0, 0] = 4.0
    X = torch.zeros(8, 8, device="cuda")
    X[:, 0] = torch.linspace(0.05, 0.6, 8)
    users = torch.arange(n, device="cuda") % 8
    idx = torch.tensor([[0, 9]], dtype=torch.int32, device="cuda").repeat(n, 1)
    val = torch.zeros(n, 2, device="cuda")
    loss, _, _ = ops.distill_topk(X, Y, users, idx, val)
    x = X[:, 0].double()
    want = -math.log(2.0) - 2.5 * x + torch.log(torch.exp(4 * x) + (M - 1) * torch.exp(x))
    # scores within 2^-20 of up to 2.4, both in ln Z and in the terms; logarithms and sums of float32 numbers up to 16
    assert float((loss.double() - want[users]).abs().max()) <= 2 * 2.4 * 2.0 ** -20 + 4 * 16 * 2.0 ** -24


@pytest.mark.parametrize("first", [(1 << 21) - 40, (1 << 21) + 45 - 80, 1_000_003])
def test_the_items_gradients_of_users_on_every_axis_of_a_launch(ops, first):
    """More users than one launch axis takes, of which 80 weigh anything: dY is theirs, to what 80 terms allow.  (All weighted
    alike, what the users behind the first axis add would be lost in the tolerance of a sum over two million.)"""
    n, M, f, k = (1 << 21) + 45, 40, 8, 3
    g = gen(52)
    X = torch.rand(n, f, generator=g, device="cuda") * 2 - 1
    Y = torch.rand(M, f, generator=g, device="cuda") * 2 - 1
    idx = (torch.randint(0, M - k, (n, 1), generator=g, device="cuda") + torch.arange(k, device="cuda")).to(torch.int32)
    val = torch.randn(n, k, generator=g, device="cuda")
    part = slice(first, first + 80)
    w = torch.zeros(n, device="cuda")
    w[part] = torch.rand(80, generator=g, device="cuda") + 0.5
    loss, dX, dY = ops.distill_topk(X, Y, None, idx, val, weight=w)
    wl, wx, wy, mag, d = formula(X[part], Y, idx[part], val[part], 1.0, w[part])
    tol = (mag * rel_tolerance(d, 80)).T.contiguous() @ X[part].double().abs() + 2.0 ** -33 * mag.sum(0)[:, None]
    assert off_over_tolerance(dY, wy, tol) <= 1.0
    assert off_over_tolerance(dX[part], wx, rel_tolerance(d, M) * (mag @ Y.double().abs())) <= 1.0
    assert not dX[: first].any() and not dX[first + 80:].any()
    assert off_over_tolerance(loss[part], wl, 1e-5 + 1e-5 * wl.abs()) <= 1.0
