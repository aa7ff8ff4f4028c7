"""q35_attn_batch over the range of fp32: finite inputs whose definition in float64 is a float give
that float, whatever sizes of keys and values follow one another.

Tolerances are those of test_gpu_attn_batch.py, times what a test says."""
import numpy as np
import pytest

import pyq35
from batch_ref import HD, rms64
from helpers import REL_L2
from test_gpu_attn_batch import make, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


@pytest.mark.parametrize("large", [2.0 ** 80, 2.0 ** 70])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -80])
def test_large_values_before_small_ones(hip, small, large):
    """Every eighth tile of 32 keys has large value rows, the others have tiny ones or zeros, and scores
    rise by 8.5 a tile, from -64 to 64: the maximum moves with every tile, seven times in a row
    with nothing to add. Half of the heads see that, the others random scores.
    A score of 64 is a sum of 256 products: its additions are off by 256^0.5 * 64 * 2^-24 = 6e-5 where
    errors are independent, its products by 64 * 2^-21 = 3e-5, and a weight depends on two of them:
    1.3e-4, against a bar of 1.5e-4."""
    nkv, P = 16, 512
    x = make(16 * nkv, nkv, P, [3] * 17, 8, seed=21, rot=0)
    tile = np.arange(P) // 32
    for kv in range(nkv):
        x["qg"][:, 16 * kv:16 * kv + 16:2, :HD] = x["qg"][0, 16 * kv, :HD]
        q = rms64(x["qg"][0, 16 * kv:16 * kv + 1, :HD], x["q_norm"])[0]
        u = q / np.linalg.norm(q)
        k = x["k_prefix"][kv] - np.outer(x["k_prefix"][kv] @ u, u)
        x["k_prefix"][kv] = k + np.outer(8.5 * (tile - 7.5) * 16.0 / np.linalg.norm(q), u)
    x["v_prefix"] *= np.where(tile % 8 == 0, large, small).astype(np.float32)[None, :, None]
    run(hip, x, P, False, bar=15 * REL_L2)


@pytest.mark.parametrize("nq", [16, 2])
@pytest.mark.parametrize("power", [60, 100, 110, 112])
def test_large_keys(hip, power, nq):
    """One key row, or every one, times 2^power: entries up to 2^114, scores up to 2^113. The softmax is
    then 1 at one key and 0 at all others (for scores of that size to be within 2^7 of one another
    they would have to agree in 50 bits), so that no rounding reaches the outputs."""
    x = make(nq, 2, 500, [20, 40, 0, 30, 12, 9, 5, 3], 64, seed=22)
    rows = x["k_prefix"].copy()
    x["k_prefix"][:, 77] *= np.float32(2.0 ** power)
    run(hip, x, 500, False)
    x["k_prefix"] = rows * np.float32(2.0 ** power)
    run(hip, x, 500, False)


@pytest.mark.parametrize("nq", [16, 2])
@pytest.mark.parametrize("size", [2.0 ** 114, -2.0 ** 114])
def test_key_entry_along_the_query(hip, size, nq):
    """A key entry of 2^114 where the queries have their largest entry."""
    x = make(nq, 2, 300, [20, 40, 0, 30, 12, 9, 5, 3], 64, seed=23)
    x["qg"][..., 200] = 12.0
    x["k_prefix"][1, 40, 200] = size
    run(hip, x, 300, False)
