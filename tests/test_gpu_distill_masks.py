"""GPU tests of distill_rows on rows of which long stretches are masked (-inf): the share of such a stretch is 0 wherever the
rest of the row lies.  Against the formula in float64; tolerances: the argument of an exponential, |s - max| / T <= R, is rounded
to float32 (2^-24 R), and so a share is within (4 R + 16) 2^-24 of itself."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from recommender_amd import ops
    return ops


@pytest.mark.parametrize("level, T", [(-200.0, 1.0), (-3.0, 0.01), (200.0, 1.0), (-1e30, 1e28)])
@pytest.mark.parametrize("M", [9724, 59047, 200003])
def test_a_masked_stretch_of_a_row_far_from_zero(ops, M, level, T):
    """200 003 items are held by several workgroups, of which the first sees nothing but -inf."""
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    S = level + T * torch.randn(3, M, generator=g, device="cuda")
    S[:, : M * 7 // 10] = float("-inf")
    S[1, M * 9 // 10:] = float("-inf")
    idx = torch.randint(M * 7 // 10, M * 9 // 10, (3, 30), generator=g, device="cuda", dtype=torch.int32).sort(1).values
    idx[:, 1:][idx[:, 1:] == idx[:, :-1]] = -1
    val = T * torch.randn(3, 30, generator=g, device="cuda")
    w = torch.full((3,), T, device="cuda")
    loss, grad = ops.distill_rows(S, idx, val, temperature=T, weight=w)
    T64 = float(torch.tensor(T, dtype=torch.float32))
    log_q = torch.log_softmax(S.double() / T64, 1)
    t = torch.softmax(torch.where(idx >= 0, val.double() / T64, float("-inf")), 1)
    at = idx.clamp(min=0).long()
    terms = torch.where(t > 0, t * (torch.log(t) - log_q.gather(1, at)), 0.0)
    want = log_q.exp().scatter_add(1, at, -t)
    R = 12.0                                             # s / T spreads by six standard deviations on either side
    assert torch.isfinite(grad).all()
    tol = (4 * R + 16) * 2.0 ** -24
    mag = log_q.exp().scatter_add(1, at, t)
    assert ((grad.double() - want).abs() <= tol * mag).all()
    assert ((loss.double() - terms.sum(1)).abs() <= tol * terms.abs().sum(1) + tol).all()
    assert not grad[:, : M * 7 // 10].any()


@pytest.mark.parametrize("M", [700, 200003])
def test_lists_with_nan_are_not_empty_lists(ops, M):
    """softmax of a list that holds a NaN or +inf is NaN, also where it holds nothing else; the items off the list keep their
    slopes, and a list of -inf alone is the empty one."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    S = torch.randn(5, M, generator=g, device="cuda")
    idx = torch.arange(5, 15, device="cuda", dtype=torch.int32).repeat(5, 1)
    val = torch.randn(5, 10, generator=g, device="cuda")
    val[0] = float("nan")
    val[1, 3] = float("nan")
    val[2] = float("inf")
    val[3] = float("-inf")
    loss, grad = ops.distill_rows(S, idx, val)
    want, slopes = ops.distill_rows(S, idx, torch.zeros_like(val))
    assert torch.isnan(loss[:3]).all() and torch.isnan(grad[:3, 5:15]).all()
    assert float(loss[3]) == 0.0 and not grad[3].any() and torch.isfinite(loss[4])
    off = torch.ones(M, dtype=torch.bool, device="cuda")
    off[5:15] = False
    assert torch.equal(grad[[0, 1, 2, 4]][:, off], slopes[[0, 1, 2, 4]][:, off])


@pytest.mark.parametrize("n, M", [(4, 700), (40, 700), (8, 70001)])
def test_factor_form_lists_with_nan_are_not_empty_lists(ops, n, M):
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    X, Y = torch.randn(n, 20, generator=g, device="cuda"), torch.randn(M, 20, generator=g, device="cuda")
    idx = torch.arange(5, 15, device="cuda", dtype=torch.int32).repeat(n, 1)
    val = torch.randn(n, 10, generator=g, device="cuda")
    val[0] = float("nan")
    val[1] = float("-inf")
    loss, dX, dY = ops.distill_topk(X, Y, None, idx, val)
    assert torch.isnan(loss[0]) and torch.isnan(dX[0]).all() and torch.isnan(dY[5:15]).all()
    assert float(loss[1]) == 0.0 and not dX[1].any()
    rest = torch.cat([dY[:5], dY[15:]])
    assert torch.isfinite(rest).all() and torch.isfinite(loss[1:]).all() and torch.isfinite(dX[1:]).all()
