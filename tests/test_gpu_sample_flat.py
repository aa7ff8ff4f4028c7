"""q35_sample on rows whose borders lie among thousands of candidates of nearly one weight: a token far above a bulk that still
holds much of the mass, flat rows at high temperatures, bulks deep below the largest, equal logits by the thousand; large batches of a full vocabulary."""
import time

import numpy as np
import pytest

import pyq35
from batch_ref import Buffers
from q4_ref import sample_args
from test_gpu_sample import check, settings

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


@pytest.mark.parametrize("p", [0.95, 1.0])
@pytest.mark.parametrize("spread,t,above", [(0.8, 1.0, 14.0), (1.0, 1.0, 14.0), (1.3, 1.0, 14.0), (2.0, 1.3, 16.0), (1.0, 0.6, 8.0), (0.05, 1.0, 13.0),
                                            (1.0, 3.0, 0.0), (1.0, 5.0, 0.0), (1.0, 100.0, 0.0), (1e-6, 1.0, 0.0), (1e-6, 1.0, 12.5)])
@pytest.mark.parametrize("B,V", [(5, 151936), (3, 20000), (140, 4001)])
def test_bulk(hip, B, V, spread, t, above, p):
    rng = np.random.default_rng(B)
    x = dict(logits=(spread * rng.standard_normal((B, V))).astype(np.float32), **settings(B, rng, t=t, k=0, p=p, m=[0.0, 1e-7]))
    x["logits"][np.arange(B), rng.integers(0, V, B)] += np.float32(above)
    # min_p's border at 1e-7 lies in the bulk: of 20000 candidates, 1000 a unit of depth, some are within the 1.5e-10 of it
    # that check leaves open (2 V (unit / 2 + 2^-53), 1.5e-3 of a unit of depth), so all those rows may be
    check(hip, x, most_open=0.25 + (x["min_p"] > 0).mean())


@pytest.mark.parametrize("k", [3000, 40000])
def test_borders_of_a_count(hip, k):
    rng = np.random.default_rng(k)
    B, V = 6, 151936
    x = dict(logits=rng.standard_normal((B, V)).astype(np.float32), **settings(B, rng, t=4.0, k=k, p=[0.5, 0.9, 1.0], m=[0.0, 0.3]))
    check(hip, x, most_open=0.4)


def test_many_rows_of_a_full_vocabulary(hip):
    """More rows than are cut into slices."""
    rng = np.random.default_rng(2)
    B, V = 133, 151936
    x = dict(logits=(2 * rng.standard_normal((B, V), dtype=np.float32)), **settings(B, rng))
    x["logits"][:, 5] += 9.0
    check(hip, x, most_open=0.1)


@pytest.mark.parametrize("n", [64, 65, 66, 300, 1025, 2047, 2049, 3000, 8000, 8191, 8192, 8193, 9000])
@pytest.mark.parametrize("B,V", [(4, 151936), (130, 9100)])
def test_equal_ones_on_top(hip, B, V, n):
    """n equal logits far above the others, next to what a bucket, a wave and a list hold, with some of their own above them."""
    rng = np.random.default_rng(n)
    x = dict(logits=(rng.standard_normal((B, V)) - 50).astype(np.float32), **settings(B, rng, t=1.0, k=[0, 0, 40, 2000], p=[1.0, 0.9, 0.3], m=0.0))
    for b in range(B):
        at = rng.permutation(V)
        x["logits"][b, at[:n]] = 1.0
        x["logits"][b, at[n - 3:n]] = np.float32(1.0) + np.arange(3, dtype=np.float32) * np.float32(2.0 ** -20)
    # top_p of equal candidates: the border may fall within 2^-24 of a whole one
    check(hip, x, most_open=0.5)


def call_time(hip, x):
    """Seconds a call, the least of some runs of 20."""
    B, V = x["logits"].shape
    with Buffers(hip, **x, token=np.zeros(B, np.int32), prob=np.zeros(B, np.float32)) as bufs:
        a = sample_args(bufs, B, V, V)
        times = []
        for _ in range(6):
            hip.sync()
            t = time.perf_counter()
            for _ in range(20):
                pyq35.check(pyq35.lib.q35_sample(a, None))
            hip.sync()
            times.append((time.perf_counter() - t) / 20)
        return min(times)


@pytest.mark.parametrize("spread,t,above", [(1.0, 1.0, 14.0), (1.3, 1.0, 14.0), (1.0, 0.6, 8.0)])
def test_a_confident_row_is_no_slower(hip, spread, t, above):
    """One token far above a bulk that top_p reaches into: as an ordinary row, not by descent, which takes 20 times as long."""
    rng = np.random.default_rng(6)
    off = settings(1, rng, t=t, k=0, p=0.95, m=0.0, u=0.999)
    row = rng.standard_normal((1, 151936)).astype(np.float32)
    ordinary = call_time(hip, dict(off, logits=2 * row))
    row = np.float32(spread) * row
    row[0, 77] += np.float32(above)
    assert call_time(hip, dict(off, logits=row)) < 5 * ordinary


@pytest.mark.parametrize("t,equal", [(3.0, 0), (5.0, 0), (1.0, 2000), (1.0, 5000)])
def test_a_flat_row_is_little_slower(hip, t, equal):
    """Some thousand candidates beside the borders are listed and sorted, not counted one against the other or by descent."""
    rng = np.random.default_rng(7)
    row = rng.standard_normal((1, 151936)).astype(np.float32)
    ordinary = call_time(hip, dict(settings(1, rng, t=1.0, k=0, p=0.95, m=0.0, u=0.999), logits=2 * row))
    row[0, rng.permutation(151936)[:equal]] = 20.0
    assert call_time(hip, dict(settings(1, rng, t=t, k=0, p=0.95, m=0.0, u=0.7), logits=row)) < 6 * ordinary
