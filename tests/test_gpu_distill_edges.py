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
