"""GPU tests of many draws from rows that no list of candidates holds: equal scores, +inf scores, flat rows.  Columns have to be
the definition's in float64, and the time of a draw must not be that of a pass over the row.

Where all weights that count are alike (equal scores), a draw's column follows from u by a product and a floor; it is compared
where u n is not within 1e-6 of a whole number (the roundings of float64 weights and of the kernel's integers lie far below)."""
import time

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


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


def timed(call):
    """Its answer, and the milliseconds of a second run of it."""
    out = call()
    torch.cuda.synchronize()
    t = time.perf_counter()
    call()
    torch.cuda.synchronize()
    return out, (time.perf_counter() - t) * 1e3


def check_equal_items(idx, logp, u, places, kept):
    """places: the columns that share everything, in order, of which `kept` stay."""
    x = u * kept
    want = places[x.floor().long().clamp(max=kept - 1)]
    sure = (x - x.round()).abs() > 1e-6
    assert bool(sure.float().mean() > 0.9)
    assert torch.equal(idx[sure].long(), want[sure])
    assert torch.allclose(logp, -torch.log(torch.tensor(float(kept), device="cuda")).expand_as(logp), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n, M, some", [(2, 300, 5), (3, 9724, 9000), (2, 40001, 7), (1, 1000003, 1000003), (2, 262147, 250000)])
def test_many_draws_of_infinite_scores(ops, dtype, n, M, some):
    g = gen(M)
    S = torch.randn(n, M, generator=g, device="cuda").to(TYPES[dtype])
    places = torch.sort(torch.randperm(M, generator=g, device="cuda")[:some]).values
    S[:, places] = INF
    u = torch.rand(n, 1000, generator=g, device="cuda", dtype=torch.float64)
    u[0, 0], u[0, 1] = 0.0, 1.0 - 2.0 ** -53
    for kw, kept in ((dict(), some), (dict(top_k=3), min(3, some)), (dict(top_p=0.5), -(-some // 2))):
        (idx, logp), ms = timed(lambda: ops.sample_rows(S, u, temperature=0.7, **kw))
        for r in range(n):
            check_equal_items(idx[r], logp[r], u[r], places, kept)
        assert ms < 50.0, ms                             # a pass over a million items per draw: some hundred


def definition(s, u, T, top_k=0, top_p=1.0):
    """One row in float64: columns, ln q, and whether u W lies clear of a border (weights are integers of 2^-39 of the largest
    at the least, sums of a million of them within 2^-20 of that)."""
    s = s.double()
    rank = torch.sort(s, descending=True, stable=True)
    w = torch.exp((rank.values - rank.values[0]) / T)
    w[torch.isnan(w) | (rank.values == -INF)] = 0.0
    if top_k:
        w[top_k:] = 0.0
    sure = True
    if top_p < 1:
        cum = torch.cumsum(w, 0)
        p = float(torch.tensor(top_p, dtype=torch.float32))
        sure = float(((cum - p * cum[-1]).abs() / cum[-1]).min()) > 1e-12 or bool((w == w[0]).all())
        w = torch.where(cum - w < p * cum[-1], w, 0.0)
    cum = torch.cumsum(w, 0)
    at = torch.searchsorted(cum, u * cum[-1], right=True).clamp(max=int((w > 0).sum()) - 1)
    gap = torch.minimum((cum[at] - u * cum[-1]).abs(), (u * cum[-1] - (cum[at] - w[at])).abs()) / cum[-1]
    return rank.indices[at], torch.log(w[at] / cum[-1]), (gap > 1e-11) & sure


def rows_of_kind(kind, n, M, g):
    if kind == "equal":                                  # a user whose factors are 0
        S = torch.full((n, M), 0.25, device="cuda")
    elif kind == "five":                                 # quantised scores
        S = torch.randint(0, 5, (n, M), generator=g, device="cuda").float() * 0.125
    elif kind == "close":                                # all within a bucket of the histogram, one far below
        S = 1.0 + 1e-3 * torch.rand(n, M, generator=g, device="cuda")
        S[:, 3] = -1e20
    elif kind == "signs":                                # zeros of either sign are one score
        S = torch.where(torch.rand(n, M, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    else:
        S = torch.randn(n, M, generator=g, device="cuda")
    S[torch.rand(n, M, generator=g, device="cuda") < 0.01] = -INF
    return S


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("kind", ["equal", "five", "close", "signs", "normal"])
@pytest.mark.parametrize("n, M", [(3, 3001), (2, 40001), (1, 200003), (2, 600001)])
def test_many_draws_where_thousands_of_items_matter(ops, dtype, kind, n, M):
    g = gen(M)
    S = rows_of_kind(kind, n, M, g).to(TYPES[dtype])
    T = 1e22 if kind == "close" else 1.0
    draws = 700
    u = torch.rand(n, draws, generator=g, device="cuda", dtype=torch.float64)
    u[0, 0], u[0, 1] = 0.0, 1.0 - 2.0 ** -53
    for kw in (dict(), dict(top_k=M // 3), dict(top_p=0.6), dict(top_k=M // 2, top_p=0.7), dict(top_k=M), dict(top_k=5000)):
        idx, logp = ops.sample_rows(S, u, temperature=T, **kw)
        for r in range(n):
            want, wl, sure = definition(S[r].float(), u[r], T, **kw)
            assert bool(sure.float().mean() > 0.95) or kw.get("top_p"), (kw, r)
            assert torch.equal(idx[r][sure].long(), want[sure]), (kw, r)
            assert torch.allclose(logp[r][sure].double(), wl[sure], rtol=2.0 ** -23, atol=1e-7), (kw, r)
        one, _ = ops.sample_rows(S, u[:, 5].contiguous(), temperature=T, **kw)     # the same draws, however many are made
        assert torch.equal(one, idx[:, 5])


@pytest.mark.parametrize("kind", ["equal", "five", "normal", "close"])
def test_a_draw_does_not_cost_a_pass(ops, kind):
    """As many draws as are taken, of long rows: a second or two at the most (one pass per draw would be minutes)."""
    g = gen(8)
    for n, M in ((1, 1000003), (4, 70001)):
        S = rows_of_kind(kind, n, M, g)
        u = torch.rand(n, 1 << 16, generator=g, device="cuda", dtype=torch.float64)
        (idx, _), ms = timed(lambda: ops.sample_rows(S, u, temperature=1.0))
        print(kind, n, M, "%.1f ms" % ms)
        for r in range(n):
            want, _, sure = definition(S[r], u[r], 1.0)
            assert torch.equal(idx[r][sure].long(), want[sure])
        assert ms < 5000.0, ms


def test_more_draws_of_a_long_row_than_a_call_takes(ops):
    """They go in several calls: the same answers as by hand, the exclusions made once or more."""
    M, draws = (1 << 22) + 77, 5000
    g = gen(11)
    S = torch.randn(1, M, generator=g, device="cuda")
    u = torch.rand(1, draws, generator=g, device="cuda", dtype=torch.float64)
    ex = (torch.tensor([0, 3], device="cuda"), torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda"))
    S[0, 5:8] = 50.0
    idx, logp = ops.sample_rows(S, u, temperature=0.5, top_k=3000, exclude=ex)
    assert bool((S[0, 5:8] == -INF).all())
    for a, b in ((0, 100), (4050, 4150), (4900, 5000)):
        i, l = ops.sample_rows(S, u[:, a:b].contiguous(), temperature=0.5, top_k=3000)
        assert torch.equal(i, idx[:, a:b]) and torch.equal(l, logp[:, a:b])
    want, wl, sure = definition(S[0], u[0], 0.5, top_k=3000)
    assert torch.equal(idx[0][sure].long(), want[sure]) and bool(sure.float().mean() > 0.95)


def test_windows_in_a_graph_and_on_two_streams(ops):
    """Rows cut over workgroups and rows of one, many draws each; replays with the program's own work between them."""
    g = gen(12)
    cases = []
    for n, M, kind in ((1, 200003, "equal"), (2, 300007, "normal"), (3, 40001, "five"), (2, 40001, "normal")):
        S = rows_of_kind(kind, n, M, g)
        u = torch.rand(n, 500, generator=g, device="cuda")
        cases.append((S, u))
    calls = [lambda S=S, u=u: ops.sample_rows(S, u, temperature=1.0, top_p=0.99) for S, u in cases]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [c() for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        graph.replay()
        (torch.randn(700, 700, device="cuda") * 2).sum()
        torch.cuda.synchronize()
        for (i, l), (wi, wl) in zip(out, want):
            assert torch.equal(i, wi) and torch.equal(l, wl)
            i.zero_(); l.zero_()
        got = []
        for k, c in enumerate(calls):
            with torch.cuda.stream(streams[k % 2]):
                got.append(c())
        torch.cuda.synchronize()
        for (i, l), (wi, wl) in zip(got, want):
            assert torch.equal(i, wi) and torch.equal(l, wl)
