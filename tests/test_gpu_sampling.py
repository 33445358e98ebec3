"""GPU tests of the random draws from score rows (csrc/als_sampling.hip, ops.sample_rows) against the definition in
float64 numpy.  No reference counterpart (the reference always shows the ranked list): parity is with the definition.

Columns have to be equal.  The kernel's weights are integers of 2^-Q of the row's largest (Q >= 39 here), so a draw can
differ from the definition's only where u W lies within the summed roundings of a border: at most M 2^-Q / 2 of W >= 1
in all, below 1e-6 a row at these sizes.  ln q is float32, from a weight whose own rounding is 2^-(Q+1) / w: the test
allows half a float32 step of |ln q| plus that."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from recommender_amd import ops
    return ops


def definition(s, u, T, k, p, mp):
    """One row in float64: (columns, ln q, weights)."""
    s = np.where(np.isnan(s), -np.inf, s.astype(np.float64))
    top = s.max() if s.size else -np.inf
    if top == -np.inf:
        return np.full(u.shape, -1), np.full(u.shape, -np.inf), np.ones(u.shape)
    if not T > 0:
        return np.full(u.shape, int(np.argmax(s))), np.zeros(u.shape), np.ones(u.shape)
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(s == top, 0.0, (s - top) / float(T))
    w = np.exp(x)
    w[~(w >= mp)] = 0.0
    w[s == -np.inf] = 0.0
    order = np.lexsort((np.arange(len(s)), -s))
    w = w[order]
    if 0 < k < len(w):
        w[k:] = 0.0
    if p < 1:
        cum = np.cumsum(w)
        w[(cum - w >= max(p, 0.0) * cum[-1]) & (np.arange(len(w)) > 0)] = 0.0        # the first always stays
    cum = np.cumsum(w)
    u = np.clip(np.nan_to_num(u.astype(np.float64)), 0.0, 1.0)
    last = np.nonzero(w)[0][-1]
    at = np.minimum(np.searchsorted(cum, u * cum[-1], side="right"), last)
    return order[at], np.log(w[at] / cum[-1]), w[at]


def check(ops, S, u, T=1.0, k=0, p=1.0, mp=0.0, **kw):
    S0 = S.float().cpu().numpy()
    idx, logp = ops.sample_rows(S, u, temperature=T, top_k=k, top_p=p, min_p=mp, **kw)
    assert idx.dtype == torch.int32 and logp.dtype == torch.float32 and idx.shape == u.shape == logp.shape
    idx, logp, un = idx.cpu().numpy(), logp.cpu().numpy().astype(np.float64), u.cpu().numpy()
    col = lambda v, r: v[r].item() if torch.is_tensor(v) else np.float32(v) if isinstance(v, float) else v  # noqa: E731
    q = min(51, 62 - int(np.ceil(np.log2(max(S.shape[1], 1)))))
    for r in range(S.shape[0]):
        want, wl, w = definition(S0[r], np.atleast_1d(un[r]), col(T, r), col(k, r), float(col(p, r)), float(col(mp, r)))
        got, gl = np.atleast_1d(idx[r]), np.atleast_1d(logp[r])
        assert np.array_equal(got, want), (r, got, want)
        with np.errstate(invalid="ignore"):
            off = np.abs(gl - wl)
        tol = 2.0 ** -24 * np.abs(np.where(np.isfinite(wl), wl, 0)) + 2.0 ** -(q + 1) * (1 / w + S.shape[1]) + 1e-14
        assert np.all((gl == wl) | (off <= tol)), (r, gl, wl)
    return idx


def scores(rng, n, M, dtype, spread=1.0):
    return torch.from_numpy((spread * rng.normal(size=(n, M))).astype(np.float32)).cuda().to(TYPES[dtype])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,M", [(1, 1), (3, 2), (2, 7), (5, 63), (4, 64), (3, 65), (7, 1023), (2, 4097), (3, 9724), (2, 40001),
                                 (2, 70003), (1, 262147)])
def test_sizes_types_and_filters(ops, dtype, n, M):
    rng = np.random.default_rng(M + 7 * n)
    S = scores(rng, n, M, dtype, 1.5)
    u = torch.from_numpy(rng.random((n, 3))).cuda()
    for kw in [dict(), dict(T=0.3, k=50), dict(T=0.7, p=0.9), dict(T=2.0, mp=0.05), dict(T=0.5, k=max(1, M // 3), p=0.8, mp=1e-3),
               dict(T=1.0, k=1), dict(T=1.0, p=0.0), dict(T=0.0)]:
        check(ops, S, u, **kw)


def test_one_random_number_per_row_in_float32(ops):
    rng = np.random.default_rng(3)
    S = scores(rng, 33, 1000, "f32")
    u = torch.from_numpy(rng.random(33).astype(np.float32)).cuda()
    idx = check(ops, S, u, T=0.5, p=0.7)
    assert idx.shape == (33,)


def test_every_row_its_own_parameters(ops):
    rng = np.random.default_rng(4)
    n, M = 64, 3001
    S = scores(rng, n, M, "f32")
    u = torch.from_numpy(rng.random((n, 2))).cuda()
    T = torch.from_numpy(np.where(rng.random(n) < 0.2, 0.0, rng.uniform(0.01, 3, n)).astype(np.float32)).cuda()
    k = torch.from_numpy(np.where(rng.random(n) < 0.5, 0, rng.integers(1, M + 10, n)).astype(np.int32)).cuda()
    p = torch.from_numpy(np.where(rng.random(n) < 0.5, 1.0, rng.uniform(0, 1, n)).astype(np.float32)).cuda()
    m = torch.from_numpy(np.where(rng.random(n) < 0.5, 0.0, rng.uniform(0, 0.3, n)).astype(np.float32)).cuda()
    check(ops, S, u, T=T, k=k, p=p, mp=m)
    check(ops, S, u, T=0.25, k=k)


def test_parameters_per_row_outside_their_range(ops):
    """A tensor's values are not looked at on the host: NaN and out-of-range values act as documented."""
    rng = np.random.default_rng(5)
    S = scores(rng, 6, 500, "f32")
    u = torch.from_numpy(rng.random((6, 4))).cuda()
    nan = float("nan")
    f = lambda *v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    a = ops.sample_rows(S, u, temperature=f(nan, -1, 0, 1, 1, 1), top_p=f(1, 1, 1, nan, 7, 1), min_p=f(0, 0, 0, nan, -3, 9))
    b = ops.sample_rows(S, u, temperature=f(0, 0, 0, 1, 1, 1), top_p=1.0, min_p=f(0, 0, 0, 0, 0, 1))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    k = torch.tensor([-1, 0, -2 ** 31, 2 ** 31 - 1, 600, 500], dtype=torch.int32, device="cuda")
    c, d = ops.sample_rows(S, u, top_k=k), ops.sample_rows(S, u)
    assert torch.equal(c[0], d[0]) and torch.equal(c[1], d[1])


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_equal_scores_rank_by_column(ops, dtype):
    """Constant rows (every item in one bucket with one key), rows of few values, and more equal scores than the list of
    one bucket holds."""
    rng = np.random.default_rng(6)
    for M in (5, 1024, 1025, 5000, 40003):
        S = torch.full((2, M), 0.5, device="cuda", dtype=TYPES[dtype])
        u = torch.from_numpy(np.stack([[0.0, 0.25, 0.5, 0.999999, 0.123456], rng.random(5)])).cuda()
        check(ops, S, u, T=0.7)
        check(ops, S, u, k=max(1, M // 2))
        check(ops, S, u, p=0.31)
        few = torch.from_numpy(rng.integers(0, 3, (2, M)).astype(np.float32)).cuda().to(TYPES[dtype])
        check(ops, few, u, T=0.9, k=M - 1, p=0.93)
        check(ops, few, u, T=2.0, k=max(1, (2 * M) // 3))
    signed = torch.zeros((1, 3000), device="cuda", dtype=TYPES[dtype])
    signed[0, ::2] = -0.0                                       # one score as the definition sees it
    check(ops, signed, torch.tensor([[0.0, 0.0004, 0.5, 0.9999]], device="cuda", dtype=torch.float64))


def test_an_outlier_that_stretches_the_buckets(ops):
    """One item far above or below the rest puts everything else into one bucket, which is then cut by the keys' digits."""
    rng = np.random.default_rng(7)
    u = torch.from_numpy(rng.random((1, 6))).cuda()
    S = scores(rng, 1, 30000, "f32", 1e-3)
    S[0, 77] = 9.0
    check(ops, S, u, T=10.0)
    check(ops, S, u, T=10.0, k=15000, p=0.5)
    S[0, 77] = -9.0
    check(ops, S, u, T=10.0, p=0.9)
    S[0] = torch.from_numpy(1.0 + 1e-6 * rng.integers(0, 50, 30000).astype(np.float32)).cuda()
    S[0, 5] = -20.0
    check(ops, S, u, T=5.0, k=20000, p=0.77)


def test_masked_rows_infinities_and_nan(ops):
    rng = np.random.default_rng(8)
    inf, low = float("inf"), torch.finfo(torch.float32).min
    S = scores(rng, 10, 2500, "f32")
    S[0] = -inf
    S[1] = float("nan")
    S[2, 1:] = -inf
    S[3, ::2] = float("nan")
    S[4] = low                                       # a mask value everywhere: one score, uniform
    S[5, :2400] = low
    S[6, [3, 9, 2000]] = inf                         # they share everything
    S[7, 100:] = -inf
    S[8] = torch.where(torch.rand(2500, device="cuda") < 0.5, torch.tensor(low, device="cuda"), torch.tensor(-inf, device="cuda"))
    S[9] *= 1e37
    u = torch.from_numpy(rng.random((10, 5))).cuda()
    for kw in [dict(), dict(T=0.1, k=7), dict(p=0.6), dict(mp=0.3), dict(T=float("inf")), dict(T=1e-30), dict(T=0.0)]:
        check(ops, S, u, **kw)


def test_random_numbers_at_and_outside_the_ends(ops):
    rng = np.random.default_rng(9)
    S = scores(rng, 1, 4000, "f32")
    u = torch.tensor([[0.0, -0.5, float("nan"), 1.0, 7.0, 1 - 2.0 ** -53, float("inf")]], dtype=torch.float64, device="cuda")
    idx = check(ops, S, u, k=100)
    order = torch.sort(S[0], descending=True, stable=True).indices
    assert (idx[0, :3] == int(order[0])).all() and (idx[0, 3:] == int(order[99])).all()


def test_strided_and_misaligned_rows(ops):
    rng = np.random.default_rng(10)
    for dtype in sorted(TYPES):
        big = scores(rng, 9, 5011, dtype)
        u = torch.from_numpy(rng.random((9, 2))).cuda()
        for a in range(0, 9):
            check(ops, big[:, a:a + 4001], u, T=0.5, p=0.9)
        check(ops, big[::2, 3:], u[::2].contiguous(), k=20)
        check(ops, big[4:5, 1:2], u[4:5])


def test_exclusions_are_dropped_and_written_as_topk_does(ops):
    rng = np.random.default_rng(11)
    n, M = 6, 1200
    S = scores(rng, n, M, "f32")
    lens = [0, 5, 300, 1200, 1, 40]
    ptr = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    col = np.concatenate([np.sort(rng.choice(M, size=l, replace=False)) for l in lens]).astype(np.int32)
    rows = torch.tensor([5, 4, 3, 2, 1, 0], device="cuda")
    ex = (torch.from_numpy(ptr).cuda(), torch.from_numpy(col).cuda())
    u = torch.from_numpy(rng.random((n, 3))).cuda()
    masked = S.clone()
    for r in range(n):
        c = 5 - r
        masked[r, torch.from_numpy(col[ptr[c]:ptr[c + 1]]).long().cuda()] = float("-inf")
    got = S.clone()
    a = ops.sample_rows(got, u, 0.8, exclude=ex, exclude_rows=rows)
    b = ops.sample_rows(masked, u, 0.8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(got, masked)
    assert (a[0][2] == -1).all()                     # every item excluded
    plain = S.clone()
    ops.sample_rows(plain, u, exclude=ex)
    assert torch.equal(torch.isinf(plain).sum(1).cpu(), torch.tensor(lens))


def test_draws_follow_the_distribution(ops):
    """u on an even grid of 2^16 values: every column's share is its probability to within one step."""
    rng = np.random.default_rng(12)
    S = scores(rng, 1, 50, "f32")
    N = 1 << 16
    u = ((torch.arange(N, dtype=torch.float64, device="cuda") + 0.5) / N)[None]
    idx, logp = ops.sample_rows(S, u.contiguous(), temperature=0.8)
    share = torch.bincount(idx[0].long(), minlength=50).double() / N
    want = torch.softmax(S[0].double() / 0.800000011920929, 0)
    assert float((share - want).abs().max()) <= 1.0 / N + 1e-12
    assert float((logp[0].double().exp() - want[idx[0].long()]).abs().max()) < 1e-6


def test_same_bits_alone_in_a_block_on_another_stream_and_in_a_graph(ops):
    rng = np.random.default_rng(13)
    S = scores(rng, 40, 20011, "f32")
    u = torch.from_numpy(rng.random((40, 2))).cuda()
    kw = dict(temperature=0.4, top_k=500, top_p=0.9, min_p=1e-3)
    want = ops.sample_rows(S, u, **kw)
    for r in (0, 17, 39):
        one = ops.sample_rows(S[r:r + 1], u[r:r + 1], **kw)
        assert torch.equal(one[0], want[0][r:r + 1]) and torch.equal(one[1], want[1][r:r + 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = ops.sample_rows(S, u, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there[0], want[0]) and torch.equal(there[1], want[1])
    Sg, ug = S.clone(), u.clone()
    ops.sample_rows(Sg, ug, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_rows(Sg, ug, **kw)
    for step in range(4):
        Sg.copy_(S.roll(step, 1)); ug.copy_(u.flip(0) if step % 2 else u)
        graph.replay()
        eager = ops.sample_rows(Sg, ug, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1]), step


def test_no_rows(ops):
    idx, logp = ops.sample_rows(torch.empty(0, 5, device="cuda"), torch.empty(0, 2, device="cuda"))
    assert idx.shape == (0, 2) and logp.shape == (0, 2)


def test_refusals(ops):
    S = torch.zeros(4, 10, device="cuda")
    u = torch.zeros(4, device="cuda")
    ok = torch.zeros(4, device="cuda")
    for bad in [lambda: ops.sample_rows(S.cpu(), u), lambda: ops.sample_rows(S, u.cpu()), lambda: ops.sample_rows(S.double(), u),
                lambda: ops.sample_rows(S[0], u), lambda: ops.sample_rows(S.t(), u), lambda: ops.sample_rows(S[:, :0], u),
                lambda: ops.sample_rows(S[:1].expand(4, 10), u), lambda: ops.sample_rows(S, u[:3]),
                lambda: ops.sample_rows(S, u.half()), lambda: ops.sample_rows(S, torch.zeros(4, 0, device="cuda")),
                lambda: ops.sample_rows(S, torch.zeros(4, 4, device="cuda").t()),
                lambda: ops.sample_rows(S, u, temperature=-1.0), lambda: ops.sample_rows(S, u, temperature=float("nan")),
                lambda: ops.sample_rows(S, u, top_k=-1), lambda: ops.sample_rows(S, u, top_k=2 ** 31),
                lambda: ops.sample_rows(S, u, top_p=1.5), lambda: ops.sample_rows(S, u, min_p=-0.1),
                lambda: ops.sample_rows(S, u, temperature=ok[:3]), lambda: ops.sample_rows(S, u, temperature=ok.double()),
                lambda: ops.sample_rows(S, u, top_k=ok), lambda: ops.sample_rows(S, u, top_p=ok.cpu()),
                lambda: ops.sample_rows(S, u, exclude_rows=torch.zeros(4, dtype=torch.int64, device="cuda")),
                lambda: ops.sample_rows(S, u, exclude=(torch.zeros(3, dtype=torch.int64, device="cuda"),
                                                       torch.zeros(1, dtype=torch.int32, device="cuda")))]:
        with pytest.raises(ValueError):
            bad()


def test_more_rows_than_one_axis_of_a_launch_takes(ops):
    rng = np.random.default_rng(31)
    n = (1 << 21) + 37
    S = torch.from_numpy(rng.normal(size=(n, 6)).astype(np.float16)).cuda()
    u = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
    idx, logp = ops.sample_rows(S, u)
    assert int(idx.min()) >= 0 and int(idx.max()) < 6
    for part in (slice(0, 100), slice(n - 100, n)):
        i, l = ops.sample_rows(S[part].clone(), u[part])
        assert torch.equal(i, idx[part]) and torch.equal(l, logp[part])


def test_more_draws_than_are_taken(ops):
    S = torch.zeros((1, 10), device="cuda")
    with pytest.raises(ValueError, match="draws"):
        ops.sample_rows(S, torch.zeros((1, (1 << 16) + 1), device="cuda"))


def test_a_thousand_draws_of_a_row(ops):
    rng = np.random.default_rng(32)
    check(ops, scores(rng, 2, 5000, "f32"), torch.from_numpy(rng.random((2, 1000))).cuda(), T=2.0, p=0.95)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M", [30011, 131071])
def test_16_bit_rows_counted_by_value(ops, dtype, M):
    """Rows of which much counts: few values, one value more often than 16 bits count, zeros of both signs, magnitudes too
    small for the table of values, more of them than their list takes, masks, only negative scores, one binade."""
    rng = np.random.default_rng(M)
    base = rng.normal(size=M).astype(np.float32)
    rows = [base, np.where(rng.random(M) < 0.7, 1.0, base), np.where(rng.random(M) < 0.5, -np.inf, base),
            np.where(rng.random(M) < 0.02, np.where(rng.random(M) < 0.5, 0.0, -0.0), base),
            np.where(rng.random(M) < 0.005, base * 2.0 ** -12, base), np.where(rng.random(M) < 0.3, base * 2.0 ** -12, base),
            -np.abs(base) - 0.25, 1.0 + rng.random(M) * 0.5, np.where(rng.random(M) < 0.6, 0.0, base),
            np.where(rng.random(M) < 0.3, -65504.0, base), np.full(M, 0.5), base * 1000.0, base * 2.0 ** -14]
    S = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda().to(TYPES[dtype])
    u = torch.from_numpy(rng.random((len(rows), 5))).cuda()
    for kw in (dict(T=0.5), dict(T=3.0, p=0.7), dict(T=0.5, k=M // 2), dict(T=1e30), dict(T=0.01, p=0.999)):
        check(ops, S, u, **kw)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("M", [700, 40001, 70003])
def test_best_item_at_temperature_zero(ops, dtype, M):
    """Many equal best items (more than a list holds), an infinite one at the start, the end and late, masks, NaN: the lowest
    column of the largest score, whatever the filters say."""
    rng = np.random.default_rng(M)
    base = rng.normal(size=M).astype(np.float32)
    rows = [base, np.zeros(M), np.where(rng.random(M) < 0.5, 7.0, base), np.where(np.arange(M) == M - 3, np.inf, base),
            np.where(np.arange(M) == 1, np.inf, base), np.where(np.arange(M) >= M // 2, np.inf, base), np.full(M, -np.inf),
            np.where(np.arange(M) % 2 == 0, np.nan, base), np.arange(M) / 64.0, -np.arange(M) / 64.0, np.full(M, -65504.0)]
    S = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda().to(TYPES[dtype])
    s = S.float().cpu().numpy()
    s = np.where(np.isnan(s), -np.inf, s)
    want = np.where(s.max(1) == -np.inf, -1, s.argmax(1))
    u = torch.from_numpy(rng.random((len(rows), 2))).cuda()
    for kw in (dict(), dict(top_k=5, top_p=0.5), dict(min_p=0.5)):
        idx, logp = ops.sample_rows(S, u, temperature=0.0, **kw)
        assert np.array_equal(idx.cpu().numpy(), np.stack([want, want], 1))
        assert torch.equal(logp, torch.where(idx < 0, -torch.inf, 0.0).float())
