"""A comparison that only values which are right can pass."""
import numpy as np


def wrong(got, want, tol):
    """Where `got` is not within `tol` of `want`: a NaN is right only where a NaN is wanted, an infinity only where that infinity is."""
    got, want, tol = np.broadcast_arrays(np.asarray(got, np.float64), np.asarray(want, np.float64), np.asarray(tol, np.float64))
    finite = np.isfinite(want)
    assert np.isfinite(tol[finite]).all() and (tol[finite] >= 0).all(), "a finite value needs a finite tolerance"
    with np.errstate(invalid="ignore"):
        near = finite & (np.abs(got - want) <= tol)
    return ~(near | (got == want) | (np.isnan(got) & np.isnan(want)))
