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
