"""q35_matmul_q4 where an entry of X stands far above its group's others and meets a weight of 0: the others keep what fp32
gives them, in every form of the product.

Tolerance. An entry times the power of two that brings its group's largest to [2^14, 2^15) is two fp16 values: the first is
off by half a step, 2^-11 of itself, the second by 2^-11 of what the first leaves, or by 2^-25 where fp16 has no smaller
values, 2^-39 of the largest. The rest as in test_gpu_matmul_q4.py: (K / 32 + 10) 2^-24 of the sum of the products, in
which a weight of 0 has no share, and 2^-23 of the result."""
import numpy as np
import pytest

import pyq35
from batch_ref import Buffers
from q4_ref import bytes_of, nibbles, weights64
from test_gpu_matmul_q4 import arrays, call, expect, make, pack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def bound(x, w, want):
    K, G = x["K"], x["G"]
    groups = (K + G - 1) // G
    X = np.abs(x["X"][:, :K].astype(np.float64))
    top = np.pad(X, ((0, 0), (0, groups * G - K))).reshape(len(X), groups, G).max(-1)
    each = np.pad(np.abs(w), ((0, 0), (0, groups * G - K))).reshape(len(w), groups, G).sum(-1)
    return (2.0 ** -39 * top @ each.T + (2.0 ** -22 + (K / 32 + 10) * 2.0 ** -24) * (X @ np.abs(w).T) + 2.0 ** -23 * np.abs(want)
            + 1e-37)


def outliers(x, size, rng):
    """One entry of every group of X is `size` times as large, and its weights are 0."""
    K, G = x["K"], x["G"]
    c = nibbles(x["codes"])[:, :K].copy()
    for g in range((K + G - 1) // G):
        at = g * G + rng.integers(0, min(G, K - g * G))
        x["X"][:, at] = np.float32(size) * np.sign(x["X"][:, at]) * (1.0 + rng.random(len(x["X"]), dtype=np.float32))
        c[:, at] = 8 if x["zeros"] is None else x["zeros"][:, g] & 15
    x["codes"] = bytes_of(c)
    return x


def multiply(hip, x):
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        return bufs.get("Y")


@pytest.mark.parametrize("size", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("M,N,K,G,zeros", [
    (1, 300, 2048, 64, False), (1, 64, 1000, 128, True), (1, 40, 511, 32, False), (3, 100, 2048, 64, True), (4, 33, 640, 32, True),
    (8, 8300, 256, 64, False), (13, 64, 6144, 32, False), (16, 9000, 513, 128, True), (24, 11000, 512, 64, True), (70, 50, 700, 64, False),
    (9, 30000, 130, 64, True), (12, 22000, 300, 128, False), (16, 16500, 260, 32, False), (6, 9000, 300, 128, True), (40, 5000, 640, 64, True)])
def test_beside_an_outlier(hip, M, N, K, G, zeros, size):
    rng = np.random.default_rng(M + K)
    x = outliers(make(M, N, K, G, zeros, M + N + K), size, rng)
    got = multiply(hip, x)
    w, want = expect(x)
    b = bound(x, w, want)
    err = np.abs(got - want)
    assert (err <= b).all(), f"worst {np.nanmax(err / b)}"


def test_a_row_alone_and_in_a_batch(hip):
    """One row's outputs are as near by itself as among many, whatever form multiplies them."""
    rng = np.random.default_rng(1)
    x = outliers(make(40, 7000, 512, 64, False, 3), 1e5, rng)
    w, want = expect(x)
    for M in (1, 2, 7, 16, 40):
        y = dict(x, X=x["X"][:M], Y=x["Y"][:M])
        assert (np.abs(multiply(hip, y) - want[:M]) <= bound(y, w, want[:M])).all(), M
