"""q35_attn_batch where the definition in float64 is finite beside infinities or values near the
largest float in the caches: the output has to be finite too, and the definition's. (What may be lost
is stated with the entry point: sums over an fp32 prefix of more than 16 query rows with such an
entry, and infinities in bf16 caches.) Tolerances are those of test_gpu_attn_batch.py."""
import numpy as np
import pytest

import pyq35
from helpers import bf16_bits, bf16_to_f32
from test_gpu_attn_batch import make, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("nq", [16, 2])
@pytest.mark.parametrize("size", [3e38, -3e38])
def test_key_entry_near_the_largest(hip, size, nq, where, bf16):
    """Weights of 1 for that key or of 0, whatever the other entries: no rounding reaches the outputs."""
    if nq == 16 and where == "prefix" and not bf16:
        size = np.copysign(2.0 ** 114, size)   # the largest that this form takes
    x = make(nq, 2, 500, [20, 40, 0, 30, 12, 9, 5, 3], 64, seed=31, bf16=bf16)
    val = np.array([size], np.float32)
    val = bf16_to_f32(bf16_bits(val)) if bf16 else val
    if where == "prefix":
        x["k_prefix"][1, 77, 5] = val[0]
    else:
        x["k_own"][3, 1, 11, 5] = val[0]
    got = run(hip, x, 500, bf16)
    assert np.isfinite(got["out"]).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("nq", [16, 2])
def test_large_values(hip, nq, where, bf16):
    """A value row of up to 2^114 among ordinary ones: the others do not show beside it."""
    x = make(nq, 2, 500, [20, 40, 0, 30, 12, 9, 5, 3], 64, seed=32, bf16=bf16)
    if where == "prefix":
        x["v_prefix"][1, 77] *= np.float32(2.0 ** 111)
    else:
        x["v_own"][3, 1, 11] *= np.float32(2.0 ** 111)
    got = run(hip, x, 500, bf16)
    assert np.isfinite(got["out"]).all()


@pytest.mark.parametrize("P,lens", [(0, [20, 40, 0, 200]), (33, [17, 4, 0, 1]), (49, [0, 0])])
@pytest.mark.parametrize("nq,nkv", [(2, 2), (4, 2), (8, 2)])
def test_keys_of_weight_zero(hip, nq, nkv, P, lens):
    """Keys with a score of minus infinity have a weight of 0: single ones, and all old rows of the own
    caches and the last of the prefix, whole groups of 16 of them (fp32 rows multiplied as they are)."""
    x = make(nq, nkv, P, lens, 256, seed=33)
    x["qg"][..., 200] = np.abs(x["qg"][..., 200]) + 0.1   # (not rotated: every query's entry is positive)
    for some in (True, False):
        k = -np.inf
        if P:
            x["k_prefix"][:, (P - 1) // 16 * 16:P, 200] = k
            x["k_prefix"][:, 5, 200] = k
        for b, n in enumerate(lens):
            x["k_own"][b, :, slice(3, 4) if some else slice(0, n), 200] = np.where(n > 3 or not some, k, np.nan)
        got = run(hip, x, P, False)
        assert np.isfinite(got["out"]).all()
