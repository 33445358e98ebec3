"""GPU tests of the paths that use the softmax operators together: ops.recommend_sample, RecommenderALS.sample and
RecommenderALS.distill - a model trained, its lists followed by a smaller one, and items drawn from that.  No reference
counterpart; draws are compared with sample_rows of the materialised scores, steps with ops.distill_topk."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ra():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import recommender_amd
    return recommender_amd


def matrix(rng, N, M, per):
    import scipy.sparse as sps
    rows = np.repeat(np.arange(N), per)
    cols = np.concatenate([rng.choice(M, size=per, replace=False) for _ in range(N)])
    U = sps.csr_matrix((rng.integers(1, 6, len(rows)).astype(np.float64), (rows, cols)), shape=(N, M))
    U.sort_indices()
    return U


@pytest.mark.parametrize("prepared", [False, True])
@pytest.mark.parametrize("excluded", [False, True])
def test_recommend_sample_is_sample_rows_of_the_scores(ra, prepared, excluded):
    from recommender_amd import ops
    rng = np.random.default_rng(1)
    N, M, f = 90, 1500, 32
    X = torch.from_numpy(rng.normal(size=(N, f)).astype(np.float32)).cuda()
    Y = torch.from_numpy(rng.normal(size=(M, f)).astype(np.float32)).cuda()
    users = torch.from_numpy(rng.integers(0, N, 70)).cuda()
    u = torch.from_numpy(rng.random((70, 3))).cuda()
    items = ops.prepare_items(Y) if prepared else Y
    U = matrix(rng, N, M, 40)
    ex = (U.indptr, U.indices) if excluded else None
    T = torch.from_numpy(rng.uniform(0.3, 2, 70).astype(np.float32)).cuda()
    k = torch.from_numpy(rng.integers(0, 100, 70).astype(np.int32)).cuda()
    for kw in [dict(temperature=2.0), dict(temperature=T, top_p=0.8), dict(temperature=1.0, top_k=50, min_p=0.01, top_p=0.9),
               dict(temperature=T, top_k=k), dict(temperature=3.0, top_k=M), dict(temperature=0.0, top_k=7)]:
        for block in (4096, 16):
            idx, logp = ops.recommend_sample(X, items, users, u, exclude_csr=ex, block_users=block, **kw)
            sc = ops.scores(X, items, users)
            e = ops.device_exclusions(ex, X.device) if excluded else None
            want, wlog = ops.sample_rows(sc, u, exclude=e, exclude_rows=users if excluded else None, **kw)
            assert torch.equal(idx, want)
            assert torch.allclose(logp, wlog, rtol=1e-6, atol=1e-6)
    one, _ = ops.recommend_sample(X, items, users, u[:, 0].contiguous(), temperature=1.0, top_k=20)
    assert one.shape == (70,)


def test_recommender_sample(ra):
    rng = np.random.default_rng(2)
    U = matrix(rng, 60, 200, 20)
    rec = ra.RecommenderALS(als_kwargs=dict(f=16, epochs=2, lamb=0.1))
    rec.input_data(U)
    rec.train()
    users = np.arange(60)
    idx, logp = rec.sample(users, n=5, temperature=0.2, seed=3)
    again, _ = rec.sample(users, n=5, temperature=0.2, seed=3)
    assert idx.shape == logp.shape == (60, 5) and np.array_equal(idx, again)
    assert ((idx >= 0) & (idx < 200)).all() and (logp <= 0).all()
    best, _ = rec.sample(users, temperature=0.0)
    top, _ = rec.recommend(users, k=1)
    assert np.array_equal(best, top)
    seen, _ = rec.sample(users, n=50, temperature=5.0, top_k=0, filter_rated=True, seed=1)
    assert all(not set(seen[u]) & set(U.indices[U.indptr[u]:U.indptr[u + 1]]) for u in users)
    few, lq = rec.sample(users[:2], n=4, temperature=[0.1, 0.5], top_k=[1, 3], u=np.full((2, 4), 0.999))
    assert (few[0] == few[0, 0]).all() and lq[0, 0] == 0.0
    with pytest.raises(ValueError):
        rec.sample(users, n=0)
    with pytest.raises(ValueError):
        rec.sample([60], filter_rated=True)


def test_distill_step_and_the_run_of_all_three(ra):
    """A teacher's lists followed by a smaller model for one step: the step is the gradients of ops.distill_topk, the loss
    it returns that of the factors before; and items are then drawn from the new factors."""
    from recommender_amd import ops
    rng = np.random.default_rng(4)
    U = matrix(rng, 80, 300, 25)
    teacher = ra.RecommenderALS(als_kwargs=dict(f=32, epochs=2, lamb=0.1)).input_data(U)
    teacher.train()
    student = ra.RecommenderALS(als_kwargs=dict(f=8, epochs=1, lamb=0.1, phantom_rows=1)).input_data(U)
    student.train()
    users = rng.permutation(80)[:50]
    ti, tv = teacher.recommend(users, k=20)
    ti[3, 10:] = -1
    X0, Y0 = student.X.clone(), student.Y.clone()
    before, _ = student.sample(users, temperature=0.0)
    loss = student.distill(ti, tv, users, lr=0.5, temperature=0.3)
    uid = torch.from_numpy(users).cuda()
    w = torch.full((50,), 1 / 50, device="cuda")
    wl, dX, dY = ops.distill_topk(X0, Y0, uid, torch.from_numpy(ti.astype(np.int32)).cuda(), torch.from_numpy(tv).cuda(), temperature=0.3,
                                  weight=w, M=300)
    assert abs(loss - float(wl.double().mean())) < 1e-6
    X1, Y1 = X0.clone(), Y0.clone()
    X1[uid] -= 0.5 * dX
    Y1[:300] -= 0.5 * dY
    assert torch.allclose(student.X, X1, rtol=1e-6, atol=1e-7) and torch.allclose(student.Y, Y1, rtol=1e-6, atol=1e-7)
    assert torch.equal(student.Y[300:], Y0[300:])
    idx, _ = student.sample(users, temperature=0.0)
    want = torch.argmax(student.X[uid].double() @ student.Y[:300].double().t(), 1)
    assert np.array_equal(idx[:, 0], want.cpu().numpy())         # the prepared item table has followed the step
    with pytest.raises(ValueError):
        student.distill(ti[:2], tv[:2], [1, 1], lr=0.1)
    with pytest.raises(ValueError):
        student.distill(ti[:2], tv[:2], [1, 80], lr=0.1)
    with pytest.raises(ValueError):
        student.distill(ti[:2], tv[:1], [1, 2], lr=0.1)


def test_no_users(ra):
    from recommender_amd import ops
    X = torch.randn(5, 8, device="cuda"); Y = torch.randn(30, 8, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    for kw in (dict(top_k=3), dict(top_k=0), dict(top_k=0, top_p=0.5)):
        idx, logp = ops.recommend_sample(X, Y, none, torch.empty((0, 4), device="cuda"), **kw)
        assert idx.shape == (0, 4) and logp.shape == (0, 4)


def work(ops, rng):
    """One call of every operator, of the forms with a workspace: few long rows, rows in parts, split passes."""
    long_rows = torch.from_numpy(rng.normal(size=(2, 100001)).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.random((2, 3))).cuda()
    idx = torch.from_numpy(rng.integers(0, 100001, (2, 50)).astype(np.int32)).cuda()
    val = torch.from_numpy(rng.normal(size=(2, 50)).astype(np.float32)).cuda()
    X = torch.from_numpy(rng.normal(size=(40, 24)).astype(np.float32)).cuda()
    Y = torch.from_numpy(rng.normal(size=(5000, 24)).astype(np.float32)).cuda()
    li = torch.from_numpy(rng.integers(0, 5000, (40, 30)).astype(np.int32)).cuda()
    lv = torch.from_numpy(rng.normal(size=(40, 30)).astype(np.float32)).cuda()
    torch.cuda.synchronize()

    def call():
        return [*ops.sample_rows(long_rows, u, top_k=500, top_p=0.9), *ops.distill_rows(long_rows, idx, val),
                *ops.distill_topk(X, Y, None, li, lv)]
    return call


def test_two_streams_at_once(ra):
    from recommender_amd import ops
    rng = np.random.default_rng(7)
    a, b = work(ops, rng), work(ops, rng)
    want_a, want_b = a(), b()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        with torch.cuda.stream(sa):
            got.append((a(), want_a))
        with torch.cuda.stream(sb):
            got.append((b(), want_b))
    torch.cuda.synchronize()
    for g, w in got:
        assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_two_graphs_of_one_pool(ra):
    from recommender_amd import ops
    rng = np.random.default_rng(8)
    a, b = work(ops, rng), work(ops, rng)
    want_a, want_b = a(), b()
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        out_a = a()
    with torch.cuda.graph(gb, pool=ga.pool()):
        out_b = b()
    for _ in range(4):
        for g in (ga, gb, gb, ga):
            g.replay()
        (torch.randn(1000, 1000, device="cuda") * 2).sum()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out_a, want_a))
        assert all(torch.equal(x, y) for x, y in zip(out_b, want_b))
        for o in out_a + out_b:
            o.zero_()
