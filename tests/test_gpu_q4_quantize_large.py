"""q35_q4_quantize where a group's scale is more than fp16 holds: such a group has no values, its scale is a NaN."""
import numpy as np
import pytest

import pyq35
from batch_ref import Buffers
from helpers import bf16_bits, bf16_to_f32
from q4_ref import quantize_weights, weights64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("K,G", [(256, 64), (100, 32), (300, 128)])
def test_scales_beyond_fp16(hip, K, G, bf16, asym):
    rng = np.random.default_rng(K)
    N, groups = 12, (K + G - 1) // G
    W = rng.standard_normal((N, K)).astype(np.float32)
    last = 65519.0 * (15.0 if asym else 8.0)        # the largest whose scale is rounded to 65504
    W[0, 5], W[1, 5], W[2, 5] = last, 2 * last, -2 * last
    W[3, 5], W[4, 5], W[5, 5] = 3e38, -3e38, 1.001 * last
    W[6, 4], W[6, 5] = 3e38, -3e38
    W[7, G:] *= np.float32(1e7)
    W[0, :G] = np.minimum(np.abs(W[0, :G]), last) if asym else W[0, :G]
    if bf16:
        W = bf16_to_f32(bf16_bits(W))
    with Buffers(hip, W=bf16_bits(W) if bf16 else W, codes=np.full((N, (K + 1) // 2), 0x55, np.uint8),
                 scales=np.zeros((N, groups), np.uint16), zeros=np.zeros((N, groups), np.uint8)) as bufs:
        pyq35.check(pyq35.lib.q35_q4_quantize(bufs.p["W"], int(bf16), N, K, G, bufs.p["codes"], bufs.p["scales"],
                                              bufs.p["zeros"] if asym else None, None))
        hip.sync()
        c, s, z = bufs.get("codes"), bufs.get("scales"), bufs.get("zeros")
    _, raw, _ = quantize_weights(W, K, G, asym)
    beyond = ~np.isfinite(raw.view(np.float16).astype(np.float32))
    assert beyond[[1, 2, 3, 4, 6], 0].all() and not beyond[8:].any()
    got = s.view(np.float16).astype(np.float32)
    assert np.array_equal(np.isnan(got), beyond) and np.array_equal(s[~beyond], raw[~beyond])
    values = weights64(c, s, z if asym else None, K, G)
    assert np.array_equal(np.isnan(values), beyond[:, np.arange(K) // G])
    if asym:
        assert (z[beyond] == 8).all()
