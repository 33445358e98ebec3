"""CPU tests of the temperatures als_distill_rows refuses - those whose reciprocal, or that times log2(e), float32 does not hold -
and of how many draws als_sample_rows takes.  Nothing is launched; the addresses are never read."""
import pytest

from recommender_amd._lib import lib

P = 1 << 20                        # an address: aligned, never read


@pytest.mark.parametrize("T", [3.5e-39, 4.0e-39, 1e-31, 2e30, 3e38, float("inf"), float("nan"), 0.0, -1.0])
def test_distill_rows_refuses_temperatures_without_a_reciprocal(T):
    rc = lib.als_distill_rows(P, 0, 100, 4, 100, P, P, 10, 10, T, None, P, P, 100, None, 0, None)
    assert rc == 1 and "temperature" in lib.als_last_error_string().decode()


def test_draws_per_call():
    """2^16, and fewer of rows so long that a pass per draw would hold the GPU: the limit refuses one more, and the sizes als_sample_rows
    refuses have none."""
    import ctypes

    from recommender_amd import _lib
    opts = _lib.SampleOpts(1.0, 0, 1.0, 0.0, None, None, None, None)
    most = lib.als_sample_rows_max_draws
    assert most(1) == most(1 << 22) == 1 << 16 and most(0) == 0 and most((1 << 31) - 1) == 0
    last = 1 << 16
    for M in ((1 << 22) + 1, 10 ** 7, 1 << 24, 1 << 28, (1 << 31) - (1 << 16)):
        d = most(M)
        assert 8 <= d <= last and d * M <= 1 << 34
        last = d
        rc = lib.als_sample_rows(P, 0, M, 1, M, None, None, None, ctypes.byref(opts), P, 0, d + 1, P, P, None, 0, None)
        assert rc == 1 and "sizes" in lib.als_last_error_string().decode()
