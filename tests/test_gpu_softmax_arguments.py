"""GPU tests of what the softmax operators make of their arguments: refusals at the entry, whatever path a call takes."""
import warnings

import warnings

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


@pytest.fixture
def model(ops):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    X = torch.randn(90, 16, generator=g, device="cuda")
    Y = torch.randn(1500, 16, generator=g, device="cuda")
    users = torch.randint(0, 90, (70,), generator=g, device="cuda")
    u = torch.rand(70, 3, generator=g, device="cuda")
    return X, Y, users, u


@pytest.mark.parametrize("block", [4096, 16])
@pytest.mark.parametrize("length", [69, 71, 1, 140])
@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
@pytest.mark.parametrize("top_k", [0, 20])
def test_recommend_sample_refuses_parameters_of_another_length(ops, model, name, length, block, top_k):
    """On the path through the list (one top_k) and through the scores, and whichever block a parameter would end in."""
    X, Y, users, u = model
    kw = dict(top_k=top_k, block_users=block)
    kw[name] = torch.full((length,), 3, dtype=torch.int32, device="cuda") if name == "top_k" else torch.full((length,), 0.5, device="cuda")
    with pytest.raises(ValueError):
        ops.recommend_sample(X, Y, users, u, **kw)


@pytest.mark.parametrize("top_k", [0, 20])
def test_recommend_sample_refuses_at_the_entry(ops, model, top_k):
    X, Y, users, u = model
    rows = torch.ones(70, device="cuda")
    for kw in (dict(u=u.half()), dict(u=u[:69]), dict(u=u.cpu()), dict(u=u.t().contiguous().t()), dict(u=u[:, :0]),
               dict(u=torch.zeros(70, (1 << 16) + 1, device="cuda")), dict(temperature=-1.0), dict(temperature=float("nan")),
               dict(top_p=1.5), dict(min_p=-0.1), dict(temperature=rows.double()), dict(temperature=rows.cpu()),
               dict(top_p=torch.ones(140, device="cuda")[::2]), dict(top_k=-1), dict(users=users.int()), dict(users=users + 50)):
        args = dict(dict(users=users, u=u, top_k=top_k), **kw)
        with pytest.raises(ValueError):
            ops.recommend_sample(X, Y, args.pop("users"), args.pop("u"), **args)


def waits_for_the_device(call):
    torch.cuda.synchronize()
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        torch.cuda.set_sync_debug_mode("warn")
        try:
            call()
        finally:
            torch.cuda.set_sync_debug_mode("default")
    return sum("called a synchronizing" in str(w.message) for w in seen)


@pytest.mark.parametrize("excluded", [False, True])
def test_recommend_sample_waits_as_often_for_many_blocks_as_for_one(ops, model, excluded):
    X, Y, users, u = model
    ex = ops.device_exclusions((np.arange(91, dtype=np.int64) * 5, np.tile(np.arange(5, dtype=np.int32), 90)), X.device) if excluded else None
    counts = []
    answers = []
    for block in (4096, 7):
        call = lambda: answers.append(ops.recommend_sample(X, Y, users, u, top_p=0.9, exclude_csr=ex, block_users=block))  # noqa: E731
        call()
        counts.append(waits_for_the_device(call))
    assert counts[0] == counts[1], counts
    assert torch.equal(answers[0][0], answers[-1][0]) and torch.equal(answers[0][1], answers[-1][1])
    if excluded:
        assert int(answers[0][0].min()) >= 5
        short = ops.device_exclusions((np.zeros(50, dtype=np.int64), np.zeros(0, dtype=np.int32)), X.device)
        with pytest.raises(ValueError):
            ops.recommend_sample(X, Y, users, u, top_p=0.9, exclude_csr=short)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("swap", [False, True])
def test_distill_rows_writes_beside_the_scores_in_one_buffer(ops, dtype, swap):
    """Scores and gradient as two column blocks of one buffer share no element; any that do are refused."""
    n, M = 9, 701
    buf = torch.randn(n, 2 * M + 3, device="cuda").to(dtype)
    idx = torch.randint(0, M, (n, 20), device="cuda", dtype=torch.int32)
    val = torch.randn(n, 20, device="cuda")
    S, out = buf[:, :M], buf[:, M + 3:]
    if swap:
        S, out = out, S
    kept = S.clone()
    want = ops.distill_rows(kept, idx, val)
    loss, grad = ops.distill_rows(S, idx, val, out=out)
    assert grad is out and torch.equal(S, kept) and torch.equal(loss, want[0])
    assert torch.allclose(out.float(), want[1].float(), rtol=2.0 ** -7, atol=1e-6)
    for a in (1, M // 2, M - 1):
        with pytest.raises(ValueError):
            ops.distill_rows(buf[:, :M], idx, val, out=buf[:, a:a + M])
        with pytest.raises(ValueError):
            ops.distill_rows(buf[:, a:a + M], idx, val, out=buf[:, :M])
    with pytest.raises(ValueError):                      # a row further down
        ops.distill_rows(buf[:-1, :M], idx[:-1], val[:-1], out=buf[1:, :M])
    flat = buf.flatten()
    with pytest.raises(ValueError):                      # other row strides, which meet somewhere
        ops.distill_rows(flat[: 4 * 1000].view(4, 1000)[:, :M], idx[:4], val[:4], out=flat[M: M + 4 * 1100].view(4, 1100)[:, :M])
    ops.distill_rows(flat[: 4 * M].view(4, M), idx[:4], val[:4], out=flat[4 * M: 8 * M].view(4, M))
