"""q35_matmul_q4 with infinities and NaN in X, and with entries and scales next to the largest that there are: outputs are what
the formula's products and sums give."""
import numpy as np
import pytest

import pyq35
from q4_ref import bytes_of, nibbles, weights64
from test_gpu_matmul_q4 import make
from test_gpu_matmul_q4_outliers import bound, multiply

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


FORMS = [(1, 90, 300, 64, False), (1, 70, 256, 128, True), (5, 60, 515, 32, True), (8, 8300, 130, 64, False), (21, 12600, 128, 128, True),
         (19, 14000, 100, 32, False), (12, 22000, 100, 64, False), (7, 8400, 200, 32, True)]


@pytest.mark.parametrize("M,N,K,G,zeros", FORMS)
@pytest.mark.parametrize("bad", [[np.inf], [-np.inf], [np.nan], [np.inf, np.inf], [np.inf, -np.inf]])
def test_infinities_and_nan(hip, M, N, K, G, zeros, bad):
    """An infinity times a weight is one with the product's sign, times 0 a NaN; other rows, and groups of scale 0, as ever."""
    x = make(M, N, K, G, zeros, M + N)
    row = M // 2
    x["X"][row, 3] = 3e38               # a finite neighbour with the largest exponent
    for i, v in enumerate(bad):
        x["X"][row, 7 + i * (K - 20)] = v
    x["scales"][1, 0] = 0
    w = weights64(x["codes"], x["scales"], x["zeros"], K, G)
    got = multiply(hip, x)
    off = ~np.isfinite(x["X"][row])
    with np.errstate(all="ignore"):
        want = (x["X"][row, off].astype(np.float64) * w[:, off]).sum(-1)
    assert np.array_equal(np.isnan(got[row]), np.isnan(want))
    inf = ~np.isnan(want)
    assert np.array_equal(got[row][inf], want[inf].astype(np.float32)) and np.isinf(got[row][inf]).all()
    rest = np.arange(M) != row
    y = dict(x, X=x["X"][rest])
    exact = y["X"][:, :K].astype(np.float64) @ w.T
    assert (np.abs(got[rest] - exact) <= bound(y, w, exact)).all()


@pytest.mark.parametrize("M,N,K,G,zeros", FORMS)
def test_largest_entries_and_scales(hip, M, N, K, G, zeros):
    """An entry of 3e38 meets weights of 0 in groups of scale 60000: what it leaves of the others is finite."""
    x = make(M, N, K, G, zeros, M + N)
    c = nibbles(x["codes"])[:, :K].copy()
    x["X"][:, 9] = np.float32(3e38)
    c[:, 9] = 8 if x["zeros"] is None else x["zeros"][:, 0] & 15
    x["codes"] = bytes_of(c)
    x["scales"][:, 0] = np.float16(60000.0).view(np.uint16)
    w = weights64(x["codes"], x["scales"], x["zeros"], K, G)
    want = x["X"][:, :K].astype(np.float64) @ w.T
    got = multiply(hip, x)
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound(x, w, want)).all()
