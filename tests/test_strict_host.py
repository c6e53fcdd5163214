"""The comparison of tests/strict.py, on mistakes planted in what it is given."""
import numpy as np
import pytest

from tests import operator_refs as refs
from tests.strict import wrong

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("got,want,tol,bad", [
    (1.0, 1.0, 0.0, False), (1.0, 1.25, 0.25, False), (1.0, 1.26, 0.25, True), (NAN, 1.0, 10.0, True), (1.0, NAN, 10.0, True), (NAN, NAN, 0.0, False),
    (INF, 1.0, 1e30, True), (1.0, INF, INF, True), (INF, INF, INF, False), (INF, INF, NAN, False), (-INF, INF, INF, True), (NAN, INF, INF, True)])
def test_one_value(got, want, tol, bad):
    assert wrong(got, want, tol).item() is bad


@pytest.mark.parametrize("tol", [INF, NAN, -1.0])
def test_a_finite_value_needs_a_finite_tolerance(tol):
    with pytest.raises(AssertionError):
        wrong(1.0, 1.0, tol)


@pytest.mark.parametrize("planted", [NAN, INF, 0.0])
def test_one_element_of_a_rotation(planted):
    r = np.random.default_rng(1)
    x = r.normal(0, 1, (3, 2, 8))
    x[1, 0, 6] = INF                                     # passed on
    want, size = refs.rope(x, np.array([1, 5, 9]), np.array([1.0, 0.1]), False, 1.0, None, 0.0, 0.0)
    tol = np.where(np.isfinite(want), size * 2.0 ** -20, 0.0)
    assert not wrong(want.copy(), want, tol).any()
    got = want.copy()
    got[2, 1, 1] = planted
    assert np.argwhere(wrong(got, want, tol)).tolist() == [[2, 1, 1]]
