"""q35_attn_q4 where one workgroup has a head's cache whole: short caches, many heads of somewhat longer ones, on both
sides of each limit, for every number of query heads that a key head may have; and few long sequences, whose rows larger
workgroups share. Tolerance as in test_gpu_attn_q4.py."""
import numpy as np
import pytest

import pyq35
from test_gpu_attn_q4 import make, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


@pytest.mark.parametrize("nq,nkv", [(16, 2), (8, 2), (1, 1), (3, 1), (5, 1), (14, 2), (9, 1), (16, 1)])
@pytest.mark.parametrize("cap", [257, 300, 449, 511, 512, 513])
def test_short_caches(hip, nq, nkv, cap):
    run(hip, make(nq, nkv, [cap - 1, 0, 63, 64, -1, cap // 2, cap, 255, 256], cap, cap + nq))


@pytest.mark.parametrize("B,nkv,cap", [(64, 2, 1024), (63, 2, 1024), (64, 2, 1025), (32, 4, 700), (255, 1, 600), (256, 2, 300), (300, 2, 300),
                                       (520, 1, 513)])
def test_many_heads(hip, B, nkv, cap):
    rng = np.random.default_rng(B)
    lens = rng.integers(0, cap, B)
    lens[rng.permutation(B)[:6]] = [-1, cap - 1, cap, 0, 511 % cap, 512 % cap]
    run(hip, make(4 * nkv, nkv, lens.tolist(), cap, B + cap))


@pytest.mark.parametrize("nq,nkv,lens,cap", [(8, 2, [16399, 0, 700, -1], 16400), (16, 2, [9000, 511, 512, 16383], 16384), (16, 2, [5000], 65537),
                                             (16, 2, [65535], 65536), (5, 1, [3000], 131072), (3, 3, [43690], 43691), (8, 2, [0], 65536),
                                             (32, 4, [20000, 12800], 16384 + 4000), (16, 2, [6553, 6554, 1] * 6 + [3276, -1], 3277)])
def test_few_long_sequences(hip, nq, nkv, lens, cap):
    run(hip, make(nq, nkv, lens, cap, cap + nq))
