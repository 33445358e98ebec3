"""GPU tests of the distillation loss from the factors (csrc/als_distill_factors.hip, ops.distill_topk) against its formula
in float64.  No reference counterpart: parity is with the formula, and the gradients also with differences of the loss.

Tolerances.  Operands are two fp16 pieces (2^-22 of the value, or of 2^-18 of the factor's largest), so a score is within
d = 2^-20 sum_k |x_k y_k| of itself, q within e = 2 d / T + 2^-19 (the exponential's argument is rounded at up to 64) of
itself relatively, and each product q y, t x loses another 2^-20.  Sums of N terms run in float32 over chains of 3 N / 16
additions (16 terms per matrix instruction, three products).  A gradient is thus within (e + 2^-20 + 3 N / 16 2^-24 + 2^-20)
of sum c (q + t) |y| - the sum of its terms' magnitudes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from recommender_amd import ops
    return ops


def definition(X, Y, idx, val, T, w):
    """float64: loss [n], dX, dY, and the tolerances of each."""
    X, Y, val = X.astype(np.float64), Y.astype(np.float64), val.astype(np.float64)
    n, M = len(X), len(Y)
    s = X @ Y.T / T
    top = s.max(1, keepdims=True)
    z = np.exp(s - top).sum(1, keepdims=True)
    q = np.exp(s - top) / z
    t = np.zeros((n, M)); loss = np.zeros(n)
    for u in range(n):
        seen, keep = set(), []
        for p, i in enumerate(idx[u]):
            if 0 <= i < M and i not in seen:
                seen.add(int(i)); keep.append(p)
        if not keep or val[u, keep].max() == -np.inf:
            q[u] = 0.0
            continue
        e = np.exp((val[u, keep] - val[u, keep].max()) / T)
        e /= e.sum()
        js = idx[u, keep].astype(np.int64)
        t[u, js] = e
        ok = e > 0
        loss[u] = (e[ok] * (np.log(e[ok]) - (s[u, js[ok]] - top[u] - np.log(z[u])))).sum()
    c = (w / T)[:, None]
    d = 2.0 ** -20 * (np.abs(X) @ np.abs(Y).T + 2.0 ** -2 * np.abs(X).max() * np.abs(Y).max()).max(1, keepdims=True) / T
    e = 2 * d + 2.0 ** -19
    mag = np.abs(c) * (q + t)
    tx = (e + 2.0 ** -19 + 3 * M / 16 * 2.0 ** -24) * (mag @ np.abs(Y))
    ty = (mag * e + mag * (2.0 ** -19 + 3 * n / 16 * 2.0 ** -24)).T @ np.abs(X)
    tl = (2 * d[:, 0] + 2.0 ** -19) * (1 + np.abs(s).max(1) * 2 + np.log(M + 1))
    return loss, (c * (q - t)) @ Y, (c * (q - t)).T @ X, tl, tx + 1e-30, ty + 2.0 ** -37 * np.abs(c).max() * np.abs(X).max() * n


def check(ops, X, Y, users, idx, val, T=1.0, w=None, M=None):
    loss, dX, dY = ops.distill_topk(X, Y, users, idx, val, temperature=T, weight=w, M=M)
    Xn = X.cpu().numpy() if users is None else X[users].cpu().numpy()
    Yn = Y.cpu().numpy()[: M or len(Y)]
    wn = np.ones(len(Xn)) if w is None else w.cpu().numpy().astype(np.float64)
    wl, wx, wy, tl, tx, ty = definition(Xn, Yn, idx.cpu().numpy(), val.cpu().numpy(), float(np.float32(T)), wn)
    assert loss.shape == (len(Xn),) and dX.shape == Xn.shape and dY.shape == Yn.shape
    for name, got, want, tol in (("loss", loss, wl, tl), ("dX", dX, wx, tx), ("dY", dY, wy, ty)):
        off = np.abs(got.double().cpu().numpy() - want)
        assert np.all(off <= tol), (name, float((off / tol).max()), np.unravel_index(np.argmax(off / tol), off.shape))
    return loss, dX, dY


def inputs(rng, n, M, f, k, users=True, scale=1.0):
    X = torch.from_numpy((scale * rng.normal(size=(2 * n if users else n, f)) / f ** 0.25).astype(np.float32)).cuda()
    Y = torch.from_numpy((scale * rng.normal(size=(M, f)) / f ** 0.25).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.permutation(2 * n)[:n]).cuda() if users else None
    idx = torch.from_numpy(np.stack([rng.choice(M, size=k, replace=False) for _ in range(n)]).astype(np.int32)).cuda()
    val = torch.from_numpy(np.ascontiguousarray(-np.sort(-rng.normal(size=(n, k)).astype(np.float32), axis=1))).cuda()
    return X, Y, u, idx, val


@pytest.mark.parametrize("f", [1, 2, 7, 20, 31, 32, 33, 50, 64, 65, 96, 100, 128, 129, 200, 255, 256])
def test_factor_counts(ops, f):
    rng = np.random.default_rng(f)
    for n, M, k in [(5, 300, 20), (70, 1031, 64)]:
        X, Y, u, idx, val = inputs(rng, n, M, f, k)
        w = torch.from_numpy(rng.uniform(-1, 2, n).astype(np.float32)).cuda()
        check(ops, X, Y, u, idx, val, 0.6, w)


@pytest.mark.parametrize("n,M,k", [(1, 1, 1), (1, 2, 2), (2, 31, 31), (3, 32, 5), (31, 33, 33), (32, 255, 1), (33, 257, 100), (64, 256, 40),
                                   (255, 500, 17), (257, 1000, 64), (300, 4099, 1024), (1025, 700, 50), (1, 20001, 200), (2100, 900, 30)])
def test_sizes(ops, n, M, k):
    rng = np.random.default_rng(n + M)
    X, Y, u, idx, val = inputs(rng, n, M, 24, k)
    check(ops, X, Y, u, idx, val, 0.8)
    X, Y, _, idx, val = inputs(rng, n, M, 72, k, users=False)
    check(ops, X, Y, None, idx, val, 1.7, M=max(1, M - 1))


def test_many_splits_and_long_lists_in_one_block(ops):
    """Enough tiles that both passes are split, and lists that lie within one block of items (many entries per stage)."""
    rng = np.random.default_rng(2)
    X, Y, u, idx, val = inputs(rng, 2500, 6000, 16, 100)
    idx = torch.from_numpy(np.stack([rng.choice(200, size=100, replace=False) + 256 * (r % 3) for r in range(2500)]).astype(np.int32)).cuda()
    check(ops, X, Y, u, idx, val, 0.5)
    X, Y, u, idx, val = inputs(rng, 500, 900, 160, 100)
    idx = torch.from_numpy(np.stack([rng.choice(120, size=100, replace=False) for _ in range(500)]).astype(np.int32)).cuda()
    check(ops, X, Y, u, idx, val, 0.5)


def test_padding_repeats_and_empty_lists(ops):
    rng = np.random.default_rng(3)
    X, Y, u, idx, val = inputs(rng, 40, 2000, 40, 60)
    idx[0, 20:] = -1
    idx[1] = -1
    idx[2, ::3] = -5
    idx[3, 5:] = idx[3, 0]
    idx[4, 1::2] = idx[4, 0::2]
    idx[5, 3] = 2000; idx[5, 9] = 2 ** 31 - 1; idx[5, 10] = -2 ** 31
    val[6, 10:] = float("-inf")
    val[7] = float("-inf")
    loss, dX, dY = check(ops, X, Y, u, idx, val, 0.7)
    for r in (1, 7):
        assert float(loss[r]) == 0.0 and not dX[r].any()
    idx[:] = -1
    loss, dX, dY = check(ops, X, Y, u, idx, val, 0.7)
    assert not loss.any() and not dX.any() and not dY.any()


def test_repeated_and_unknown_users(ops):
    rng = np.random.default_rng(4)
    X, Y, u, idx, val = inputs(rng, 50, 700, 32, 20)
    u = torch.from_numpy(rng.integers(0, 6, 50)).cuda()
    check(ops, X, Y, u, idx, val, 0.9)
    bad = u.clone()
    bad[[3, 17]] = torch.tensor([-1, 100], device="cuda")
    loss, dX, dY = ops.distill_topk(X, Y, bad, idx, val, temperature=0.9)
    assert torch.isnan(loss[[3, 17]]).all() and torch.isnan(dX[[3, 17]]).all()
    keep = torch.ones(50, dtype=torch.bool, device="cuda"); keep[[3, 17]] = False
    l2, x2, y2 = check(ops, X, Y, u[keep], idx[keep].contiguous(), val[keep].contiguous(), 0.9)
    assert torch.allclose(loss[keep], l2, rtol=1e-5) and torch.allclose(dY, y2, rtol=1e-4, atol=1e-6)


def test_strided_factors_and_lists(ops):
    rng = np.random.default_rng(5)
    big_x = torch.from_numpy(rng.normal(size=(60, 90)).astype(np.float32)).cuda()
    big_y = torch.from_numpy(rng.normal(size=(801, 77)).astype(np.float32)).cuda()
    _, _, _, idx, val = inputs(rng, 60, 801, 8, 64)
    for f, a, b in [(33, 1, 2), (64, 3, 5), (70, 0, 7)]:
        check(ops, big_x[:, a:a + f], big_y[:, b:b + f], None, idx[:, 4:40], val[:, 4:40], 2.0)


def test_wide_range_of_scores_and_magnitudes(ops):
    """Scores up to some hundred temperatures apart (one item takes nearly all of q), rows a thousand times smaller than
    others, zero rows and columns; and factors far from 1, where the power-of-two scales matter."""
    rng = np.random.default_rng(6)
    for scale, T in [(6.0, 0.5), (1e-4, 1e-6), (1e3, 1e6), (0.0, 1.0)]:
        X, Y, u, idx, val = inputs(rng, 70, 1500, 48, 30, scale=scale)
        X[::7] *= 1e-3
        X[5] = 0.0; Y[::9] = 0.0; Y[:, 3] = 0.0
        val *= T
        check(ops, X, Y, u, idx, val, T)


def test_gradients_are_the_loss_differences(ops):
    """Central differences of sum w loss (float32 losses, about 2^-20 of ~5 each over 6 rows): at h = 2^-5 the noise is
    about 6 2^-20 5 / 2^-5 = 9e-4 and the truncation h^2 / 6 times a third derivative of order 1."""
    rng = np.random.default_rng(7)
    X, Y, _, idx, val = inputs(rng, 6, 50, 5, 8, users=False)
    w = torch.from_numpy(rng.uniform(0.5, 1.0, 6).astype(np.float32)).cuda()
    total = lambda X, Y: float((ops.distill_topk(X, Y, None, idx, val, temperature=1.3, weight=w)[0].double() * w).sum())  # noqa: E731
    _, dX, dY = ops.distill_topk(X, Y, None, idx, val, temperature=1.3, weight=w)
    h = 2.0 ** -5
    for grad, leaf, other in ((dX, X, 0), (dY, Y, 1)):
        for _ in range(12):
            r, c = int(rng.integers(0, leaf.shape[0])), int(rng.integers(0, 5))
            up, down = leaf.clone(), leaf.clone()
            up[r, c] += h; down[r, c] -= h
            diff = (total(up, Y) - total(down, Y)) if other == 0 else (total(X, up) - total(X, down))
            assert abs(diff / (2 * h) - float(grad[r, c])) < 3e-3


def test_agrees_with_the_row_form(ops):
    """distill_topk = scores + distill_rows + two products, as a program would chain them."""
    rng = np.random.default_rng(8)
    X, Y, u, idx, val = inputs(rng, 130, 3001, 64, 40)
    S = ops.scores(X, Y, u)
    loss, slope = ops.distill_rows(S, idx, val, temperature=0.5)
    l2, dX, dY = ops.distill_topk(X, Y, u, idx, val, temperature=0.5)
    assert torch.allclose(loss, l2, rtol=2e-5, atol=1e-6)
    wx, wy = slope.double() @ Y.double(), slope.double().t().contiguous() @ X[u].double()
    assert float((dX - wx).norm() / wx.norm()) < 1e-5 and float((dY - wy).norm() / wy.norm()) < 1e-5


def test_same_bits_again_on_a_stream_and_in_a_graph(ops):
    rng = np.random.default_rng(9)
    for n, M, f in [(300, 5003, 64), (90, 9000, 20)]:
        X, Y, u, idx, val = inputs(rng, n, M, f, 50)
        want = ops.distill_topk(X, Y, u, idx, val, temperature=0.5)
        poison = torch.full((1 << 26,), float("nan"), device="cuda")     # what the workspace held before must not matter
        del poison
        again = ops.distill_topk(X, Y, u, idx, val, temperature=0.5)
        assert all(torch.equal(a, b) for a, b in zip(want, again))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = ops.distill_topk(X, Y, u, idx, val, temperature=0.5)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, there))
        Xg = X.clone()
        ops.distill_topk(Xg, Y, u, idx, val, temperature=0.5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.distill_topk(Xg, Y, u, idx, val, temperature=0.5)
        for step in range(4):
            Xg.copy_(X.roll(step, 0))
            graph.replay()
            eager = ops.distill_topk(Xg, Y, u, idx, val, temperature=0.5)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), step


def test_no_users_and_refusals(ops):
    rng = np.random.default_rng(10)
    X, Y, u, idx, val = inputs(rng, 4, 30, 8, 5)
    loss, dX, dY = ops.distill_topk(X, Y, u[:0], idx[:0], val[:0])
    assert loss.shape == (0,) and dX.shape == (0, 8) and dY.shape == (30, 8) and not dY.any()
    wide = torch.zeros(40, 257, device="cuda")
    for bad in [lambda: ops.distill_topk(X.cpu(), Y, u, idx, val), lambda: ops.distill_topk(X, Y.cpu(), u, idx, val),
                lambda: ops.distill_topk(X.half(), Y, u, idx, val), lambda: ops.distill_topk(X, Y[:, :7], u, idx, val),
                lambda: ops.distill_topk(X, Y, u.int(), idx, val), lambda: ops.distill_topk(X, Y, u[:3], idx, val),
                lambda: ops.distill_topk(X, Y, None, idx, val), lambda: ops.distill_topk(X, Y, u, idx.long(), val),
                lambda: ops.distill_topk(X, Y, u, idx, val, temperature=0.0), lambda: ops.distill_topk(X, Y, u, idx, val, temperature=1e7),
                lambda: ops.distill_topk(X, Y, u, idx, val, weight=torch.ones(3, device="cuda")),
                lambda: ops.distill_topk(X, Y, u, idx, val, M=31), lambda: ops.distill_topk(X, Y, u, idx, val, M=0),
                lambda: ops.distill_topk(X.t(), Y, u, idx, val), lambda: ops.distill_topk(wide, wide, u, idx, val)]:
        with pytest.raises(ValueError):
            bad()


def test_an_empty_list_weighted_by_infinity(ops):
    """1 / (length of the list) as a weight: an empty list asks for nothing, and the items' gradients stay finite."""
    rng = np.random.default_rng(51)
    X, Y, u, idx, val = inputs(rng, 70, 300, 20, 9)
    idx[3] = -1; idx[40] = 300; val[41] = -np.inf
    idx[42] = 5; val[42, 0] = -np.inf                    # an item listed again: its first entry stands, and has no weight
    w = torch.rand(70, device="cuda") + 0.5
    none = [3, 40, 41, 42]
    w[none] = 0.0
    want = ops.distill_topk(X, Y, u, idx, val, weight=w)
    for bad in (np.inf, -np.inf, np.nan):
        w[none] = bad
        got = ops.distill_topk(X, Y, u, idx, val, weight=w)
        for g, v in zip(got, want):
            assert torch.equal(g, v)
    w[none] = 1.0
    check(ops, X, Y, u, idx, val, w=w)


def test_more_users_than_one_axis_of_a_launch_takes(ops):
    rng = np.random.default_rng(52)
    n, M, f, k = (1 << 21) + 45, 40, 8, 3
    X = torch.from_numpy(rng.uniform(-0.99, 0.99, size=(n, f)).astype(np.float32)).cuda()
    X[-1, 0] = 1.0                                       # the largest value, which sets the operands' scale, in the part looked at
    Y = torch.from_numpy(rng.uniform(-1, 1, size=(M, f)).astype(np.float32)).cuda()
    idx = torch.from_numpy((rng.integers(0, M - k, (n, 1)) + np.arange(k)).astype(np.int32)).cuda()
    val = torch.from_numpy(rng.normal(size=(n, k)).astype(np.float32)).cuda()
    loss, dX, dY = ops.distill_topk(X, Y, None, idx, val)
    part = slice(n - 80, n)
    wl, wx, _, tl, tx, _ = definition(X[part].cpu().numpy(), Y.cpu().numpy(), idx[part].cpu().numpy(), val[part].cpu().numpy(), 1.0,
                                      np.ones(80))
    assert np.all(np.abs(loss[part].double().cpu().numpy() - wl) <= tl)
    assert np.all(np.abs(dX[part].double().cpu().numpy() - wx) <= tx)
    # every user's share of dY, in float64
    Xd, Yd = X.double(), Y.double()
    slope = torch.softmax(Xd @ Yd.T.contiguous(), 1)
    mag = slope.clone()
    t = torch.softmax(val.double(), 1)
    slope.scatter_add_(1, idx.long(), -t)
    mag.scatter_add_(1, idx.long(), t)
    want = slope.T.contiguous() @ Xd
    e = 2.0 ** -18 * f + 2.0 ** -19                      # scores: 2 d with |x|, |y| <= 1
    tol = (e + 2.0 ** -19 + 3 * n / 16 * 2.0 ** -24) * (mag.T.contiguous() @ Xd.abs())
    assert ((dY.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("M, f", [(700, 20), (9000, 33), (70001, 64), (66000, 100), (70000, 256)])
def test_few_users(ops, n, M, f):
    """Up to four users, eight of a large catalogue: lists that share items, repeat them, or are empty; a user listed twice and
    an unknown one; lists of more than 64 items; both alignments of the factors' rows."""
    rng = np.random.default_rng(100 * n + f)
    X, Y, u, idx, val = inputs(rng, n, M, f, 150)
    idx[:, :40] = idx[0, :40].clone()                    # shared by all
    idx[:, 50] = idx[:, 3]                               # repeated
    if n > 2:
        idx[1] = -1
        u[2] = u[0]
    w = torch.from_numpy(rng.uniform(0.2, 2, n).astype(np.float32)).cuda()
    check(ops, X, Y, u, idx, val, T=0.7, w=w)
    if n > 3:
        loss, dX, dY = ops.distill_topk(X, Y, u, idx, val, weight=w)
        lost = u.clone(); lost[3] = 10 ** 9              # the others' rows and the items as if it were not there
        l2, a2, d2 = ops.distill_topk(X, Y, lost, idx, val, weight=w)
        keep = [i for i in range(n) if i != 3]
        assert torch.isnan(l2[3]) and torch.isnan(a2[3]).all() and torch.isfinite(d2).all()
        assert torch.equal(l2[keep], loss[keep]) and torch.equal(a2[keep], dX[keep])
        _, _, d3 = ops.distill_topk(X, Y, u[keep].contiguous(), idx[keep].contiguous(), val[keep].contiguous(), weight=w[keep].contiguous())
        assert torch.allclose(d2, d3, rtol=1e-5, atol=1e-6)
    bad = w.clone()
    if n > 2:
        bad[1] = np.inf                                  # its list is empty
        want = ops.distill_topk(X, Y, u, idx, val, weight=w)
        got = ops.distill_topk(X, Y, u, idx, val, weight=bad)
        assert all(torch.equal(g, v) for g, v in zip(got, want))


def test_few_users_in_a_graph(ops):
    rng = np.random.default_rng(61)
    X, Y, u, idx, val = inputs(rng, 3, 30001, 48, 70)
    want = ops.distill_topk(X, Y, u, idx, val)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.distill_topk(X, Y, u, idx, val)
    for _ in range(4):
        g.replay()
        (torch.randn(500, 500, device="cuda") * 2).sum()
        torch.cuda.synchronize()
        assert all(torch.equal(o, v) for o, v in zip(out, want))
        for o in out:
            o.zero_()
