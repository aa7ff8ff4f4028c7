"""q35_attn_q4 with a query entry, or a value row, far above the others: errors stay within what the header says operands keep.

Tolerance. Query entries, q, are off by 2^-23 of their row's largest, Q. A score is formed by groups of 64 dims as step x sum of
q code + least x sum of q: two sums of whole numbers, rounded twice and once, two products added up with one rounding
each, four groups, and a product by the unit: 8 roundings of 2^-24 of terms that are at most sum |q| (|least| + 15 step). With
the factor 1 / 16 of a score this is
    D = (2^-23 Q sum |k| + 2^-21 sum |q| (|least| + 15 step)) / 16,
and exp2 adds less than 2^-22: weights are off by E = D + 2^-22 of themselves, outputs by 2 E max |v|. Weights times steps are off by
2^-23 of the largest of a tile of 64 rows, times |code - 8| <= 8, 64 rows: 2^-14 of that largest a tile; sums of a
sequence's weights, least values and tiles add some roundings of 2^-24 a tile of what they add, max |v| at most."""
import numpy as np
import pytest

import pyq35
from batch_ref import HD, attn64, rms64, rope64
from q4_ref import row_values
from test_gpu_attn_q4 import make, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def check(x, got):
    B, nq = x["qg"].shape[:2]
    nkv = x["k"].shape[1]
    for b in range(B):
        n = int(x["len"][b]) + 1
        sc = {c: got[c + "_scale"][b, :, :n].astype(np.float64) for c in ("k", "v")}
        rows = {c: row_values(got[c][b, :, :n], got[c + "_scale"][b, :, :n]) for c in ("k", "v")}
        out, wts = attn64(x, b, rows["k"], rows["v"])
        q = rope64(rms64(x["qg"][b, :, :HD], x["q_norm"]), x["pos"][b], x["rot"])
        gate = 1.0 / (1.0 + np.exp(-x["qg"][b, :, HD:].astype(np.float64)))
        tiles = (n + 63) // 64
        for h in range(nq):
            g = h // (nq // nkv)
            span = np.repeat(np.abs(sc["k"][g, :, :, 1]) + 15.0 * sc["k"][g, :, :, 0], 64, -1)
            d = (2.0 ** -23 * np.abs(q[h]).max() * np.abs(rows["k"][g]).sum(-1) + 2.0 ** -21 * (np.abs(q[h]) * span).sum(-1)).max() / 16.0
            most = np.abs(rows["v"][g]).max()
            wide = np.zeros(4)
            for t in range(tiles):
                part = slice(64 * t, min(64 * t + 64, n))
                wide += (wts[h, part, None] * sc["v"][g, part, :, 0]).max(0)
            tol = 2.0 * (d + 2.0 ** -22) * most + np.repeat(2.0 ** -14 * wide, 64) + 2.0 ** -24 * (4 * tiles + 16) * most
            err = np.abs(got["out"][b, h] - out[h])
            assert (err <= tol * gate[h] + 2.0 ** -22 * np.abs(out[h])).all(), f"sequence {b} head {h}: {(err / tol).max()}"


@pytest.mark.parametrize("size", [30.0, 300.0, 3000.0])
@pytest.mark.parametrize("lens", [[200, 64], [900]])
def test_query_entry(hip, lens, size):
    """A norm weight makes one entry of every query row `size` times the others; keys are small there."""
    x = make(8, 2, lens, max(lens) + 1, 3)
    x["q_norm"][70] = size - 1.0
    x["k_scale"][..., 1, :] *= np.float16(2.0 / size)
    x["k_norm"][64:128] = 2.0 / size - 1.0
    check(x, run(hip, x, bar=None))


@pytest.mark.parametrize("size", [30.0, 300.0])
@pytest.mark.parametrize("lens", [[200, 64], [900]])
def test_value_row(hip, lens, size):
    """One value row stands far above the others in one group of 64 dims."""
    x = make(8, 2, lens, max(lens) + 1, 4)
    x["v_scale"][:, :, 33, 2] *= np.float16(size)
    check(x, run(hip, x, bar=None))
