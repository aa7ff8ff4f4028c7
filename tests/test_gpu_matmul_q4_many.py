"""q35_matmul_q4 for many rows and tiles, where it multiplies on the fp16 matrix cores: against float64, with the cases of
the few rows' form.

Tolerance. An entry of X enters as two fp16 values, off by 2^-11 of 2^-11 of itself; a product instruction adds its 32
exact products to a group's sum with one rounding, eight in a group at most (2 of 128 / 32); a scale and its
product are rounded once each, and one addition a group and one a wave follow. Each of these terms is within its own of
the few rows' bound: 2^-22 of the largest entry for each, (K / 32 + 10) 2^-24 of the sum of the products, 2^-23 of the result."""
import numpy as np
import pytest

import pyq35
from batch_ref import Buffers, Graph
from test_gpu_matmul_q4 import arrays, bound, call, check, expect, make, pack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,G", [(17, 15600, 320, 64), (20, 13111, 515, 32), (33, 8000, 260, 128), (48, 8224, 255, 64), (64, 4101, 1000, 32),
                                     (100, 2700, 2600, 64), (600, 450, 4500, 128), (40, 6601, 1, 32), (257, 1040, 6144, 32), (1100, 241, 768, 64)])
def test_sizes(hip, M, N, K, G, zeros):
    check(hip, make(M, N, K, G, zeros, M + K))


@pytest.mark.parametrize("M", [19, 35])
def test_strides_and_residual(hip, M):
    check(hip, make(M, 13900, 515, 64, False, 1, ldx=517, ldy=13907, residual=True))
    check(hip, make(M, 13900, 512, 32, True, 2, ldx=540, ldy=13901, residual=True))
    check(hip, make(M, 13900, 512, 128, False, 3, ldy=13905), in_place=True)


def test_unlike_sizes(hip):
    """Entries from the smallest to the largest fp32 in one row, groups of zeros, rows of zeros."""
    M = 21
    x = make(M, 12600, 640, 64, False, 7)
    x["X"] = np.random.default_rng(7).standard_normal((M, 640)).astype(np.float32)
    x["X"][:, 64:128] *= np.float32(2.0 ** 60)
    x["X"][:, 128:192] *= np.float32(2.0 ** -60)
    x["X"][:, 192:256] = 0.0
    x["X"][:, 256] = np.float32(1e30)
    x["X"][0] *= np.float32(2.0 ** -100)
    x["X"][M // 2, 320:] = 0.0
    x["X"][2] = 0.0
    w, want = expect(x)
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        got = bufs.get("Y")
    # entries below 2^-100 may count as 0
    assert (np.abs(got - want) <= bound(x, w, want) + 2.0 ** -100 * np.abs(w).sum(1)).all()


@pytest.mark.parametrize("top", [32767.0, 32768.0, 65519.0, 65520.0, 16383.999, 16384.0, 2047.5, 2048.5])
def test_borders_of_the_parts(hip, top):
    """The largest entry of a group next to where fp16 rounds, overflows or changes its exponent, of both signs."""
    x = make(18, 14700, 256, 64, False, 9)
    x["X"][:, ::64], x["X"][:, 1::64] = np.float32(top), np.float32(-top)
    x["X"][1] *= np.float32(2.0 ** -30)
    x["X"][3] *= np.float32(2.0 ** 100)
    check(hip, x)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_not_finite(hip, bad):
    x = make(20, 13200, 300, 64, True, 11)
    keep = x["X"].copy()
    x["X"][7, 100] = bad
    x["scales"][5, 2] = 0x7E00
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        got = bufs.get("Y")
    assert not np.isfinite(got[7]).any() and np.isnan(got[:, 5]).all()
    x["X"] = keep
    x["scales"][5, 2] = 0
    w, want = expect(x)
    ok = np.ones_like(got, bool)
    ok[7], ok[:, 5] = False, False
    assert (np.abs(got - want) <= bound(x, w, want))[ok].all()


def test_graph(hip):
    """A captured call, replayed with other rows between eager calls."""
    x = make(33, 8224, 512, 64, True, 5)
    rng = np.random.default_rng(5)
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        g = Graph(hip, lambda s: call(bufs, x, stream=s))
        try:
            for _ in range(3):
                bufs.set("X", rng.standard_normal(x["X"].shape, dtype=np.float32))
                g.replay()
                first = bufs.get("Y")
                bufs.set("Y", x["Y"])
                call(bufs, x)
                hip.sync()
                assert np.array_equal(first, bufs.get("Y")) and np.isfinite(first).all()
        finally:
            g.close()
