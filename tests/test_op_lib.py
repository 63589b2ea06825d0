"""The comparison that the operators' tests go by: what it has to refuse."""
import numpy as np
import pytest

from op_lib import close


@pytest.mark.parametrize("got", [np.nan, np.inf, -np.inf, 1.5])
def test_close_refuses(got):
    want = np.ones((2, 3))
    a = want.copy()
    close(a, want, 0)
    a[1, 2] = got
    with pytest.raises(AssertionError):
        close(a, want, 0.25)


@pytest.mark.parametrize("want", [np.nan, np.inf])
def test_close_refuses_values_for_what_is_not_finite(want):
    w = np.ones((2, 3))
    w[0, 1] = want
    close(w.copy(), w, 0)
    for got in (1.0, -np.inf, np.inf if np.isnan(want) else np.nan):
        a = w.copy()
        a[0, 1] = got
        with pytest.raises(AssertionError):
            close(a, w, 0.25)
