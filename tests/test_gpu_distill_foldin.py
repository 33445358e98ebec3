"""GPU test of fold-in after RecommenderALS.distill: the cached item Gram is the new items', in the process that trained the model
as in one that loaded it."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_fold_in_after_a_distillation_step(tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import scipy.sparse as sps

    import recommender_amd as ra
    rng = np.random.default_rng(5)
    rows = np.repeat(np.arange(60), 20)
    cols = np.concatenate([rng.choice(200, size=20, replace=False) for _ in range(60)])
    U = sps.csr_matrix((rng.integers(1, 6, len(rows)).astype(np.float64), (rows, cols)), shape=(60, 200))
    kw = dict(f=16, epochs=2, lamb=0.1, phantom_rows=0)
    model = ra.RecommenderALS(als_kwargs=kw).input_data(U)
    model.train()
    lists, values = model.recommend(np.arange(60), k=10)
    step = lambda m: m.distill(lists[:, ::-1].copy(), values, np.arange(60), lr=20.0, temperature=0.2)  # noqa: E731
    triplets = (np.array([7, 7, 7, 30, 30]), np.array([1, 50, 199, 3, 8]), np.array([5.0, 3.0, 4.0, 5.0, 1.0]))

    step(model)
    model.save(str(tmp_path))
    loaded = ra.RecommenderALS(mode="predict", model_path=str(tmp_path))
    fresh = ra.RecommenderALS(mode="predict", model_path=str(tmp_path))
    model.update_user(*triplets, refresh_gram=False)
    loaded.update_user(*triplets, refresh_gram=False)
    fresh.update_user(*triplets, refresh_gram=True)
    for m in (model, loaded):
        assert torch.allclose(m.X[[7, 30]], fresh.X[[7, 30]], rtol=1e-5, atol=1e-6)

    # a training epoch leaves its own Gram, as ever
    step(model)
    model.train(epochs=3)
    want = model.engine.cache_Y
    x = model.X.clone()
    model.update_user(*triplets, refresh_gram=False)
    from recommender_amd import ops
    csr = model.make_update_data(triplets)
    ops.half_sweep(csr, model.Y, want, x, model.config["alpha"], info=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert torch.equal(model.X, x)


def test_a_step_of_many_users_goes_in_several_calls(monkeypatch):
    """Workspace for a few users only: the same step, within the roundings of sums in another order."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import scipy.sparse as sps

    import recommender_amd as ra
    from recommender_amd import ops
    rng = np.random.default_rng(6)
    U = sps.csr_matrix(rng.integers(0, 2, (300, 500)).astype(np.float64))
    lists = np.stack([rng.choice(500, size=12, replace=False) for _ in range(300)])
    values = rng.normal(size=(300, 12))
    users = rng.permutation(300)
    results = []
    for limit in (None, ops.distill_topk_workspace(64, 500, 16, 12)):
        model = ra.RecommenderALS(als_kwargs=dict(f=16, epochs=1, lamb=0.1)).input_data(U)
        model.train()
        if limit:
            model.DISTILL_BYTES = limit
        calls = []
        real = ops.distill_topk
        monkeypatch.setattr(ops, "distill_topk", lambda X, Y, u, *a, **k: calls.append(len(u)) or real(X, Y, u, *a, **k))
        loss = model.distill(lists, values, users, lr=0.5)
        monkeypatch.setattr(ops, "distill_topk", real)
        results.append((loss, model.X, model.Y))
        assert sum(calls) == 300 and (calls == [300] if limit is None else max(calls) <= 64 and len(calls) > 4)
    (l0, x0, y0), (l1, x1, y1) = results
    assert abs(l0 - l1) < 1e-6
    assert torch.allclose(x0, x1, rtol=1e-5, atol=1e-7) and torch.allclose(y0, y1, rtol=1e-5, atol=1e-7)
    with pytest.raises(ValueError):
        model.distill(lists[:2], values[:2, :5], [1, 2], lr=0.1)
    with pytest.raises(ValueError):
        model.distill(lists[:2, 0], values[:2, 0], [1, 2], lr=0.1)


def test_a_model_without_sizes_is_refused():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import recommender_amd as ra
    with pytest.raises(RuntimeError):
        ra.RecommenderALS(als_kwargs=dict(f=8)).distill([[1]], [[1.0]], [0], lr=0.1)
    model = ra.RecommenderALS(n_users=5, n_items=9, als_kwargs=dict(f=8))
    assert np.isfinite(model.distill([[1, 2]], [[1.0, 0.5]], [3], lr=0.1))
