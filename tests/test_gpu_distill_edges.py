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
