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
