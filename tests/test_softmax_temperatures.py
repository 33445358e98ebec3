"""CPU tests of the temperatures als_distill_rows refuses: those whose reciprocal, or that times log2(e), float32 does not hold.
Nothing is launched; the addresses are never read."""
import pytest

from recommender_amd._lib import lib

P = 1 << 20                        # an address: aligned, never read


@pytest.mark.parametrize("T", [3.5e-39, 4.0e-39, 1e-31, 2e30, 3e38, float("inf"), float("nan"), 0.0, -1.0])
def test_distill_rows_refuses_temperatures_without_a_reciprocal(T):
    rc = lib.als_distill_rows(P, 0, 100, 4, 100, P, P, 10, 10, T, None, P, P, 100, None, 0, None)
    assert rc == 1 and "temperature" in lib.als_last_error_string().decode()
