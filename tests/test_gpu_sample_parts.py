"""q35_sample for a small top_k, whose candidates are found by the largest logits of parts of the row: orders in which the
largest stand together, equal logits by the thousand, rows with fewer candidates than top_k, infinities, and
lists next to what one wave settles."""
import ctypes as C

import numpy as np
import pytest

import pyq35
from batch_ref import Buffers, Graph
from q4_ref import sample_args
from test_gpu_sample import check, run, settings

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def rows(rng, B, V, order):
    x = 3.0 * rng.standard_normal((B, V), dtype=np.float32)
    if order == "falling":
        return np.sort(x, -1)[:, ::-1].copy()
    if order == "rising":
        return np.sort(x, -1)
    if order == "heap":                  # the largest side by side somewhere
        at = V // 3
        x[:, at:at + 200] += 12.0
    if order == "one lane":              # the largest where they share a part
        x[:, 8:V:256] += 20.0
    return x


@pytest.mark.parametrize("order", ["any", "falling", "rising", "heap", "one lane"])
@pytest.mark.parametrize("k", [1, 2, 20, 63, 64, 65, 200])
@pytest.mark.parametrize("B,V", [(1, 151936), (7, 40001), (1, 4097)])
def test_orders(hip, B, V, k, order):
    rng = np.random.default_rng(V + k)
    x = settings(B, rng, k=k, t=[0.6, 1.0, 2.0], p=[1.0, 0.8, 0.95], m=[0.0, 0.05])
    x["logits"] = rows(rng, B, V, order)
    check(hip, x, most_open=0.5 if B == 1 else 0.3)


@pytest.mark.parametrize("k", [1, 40, 64])
def test_ties(hip, k):
    """More equal candidates than can be listed: the first by id are kept."""
    rng = np.random.default_rng(k)
    B, V = 5, 30000
    x = settings(B, rng, k=k, t=1.0, p=[1.0, 0.7], m=0.0)
    x["logits"] = np.round(rng.standard_normal((B, V)) * 0.5).astype(np.float32)
    x["logits"][0] = 1.5
    x["u"] = ((np.arange(B) + 0.37) / B).astype(np.float32)
    check(hip, x, most_open=0.2)


@pytest.mark.parametrize("left", [0, 1, 5, 30, 70])
def test_few_candidates(hip, left):
    """Rows of which a grammar, or the depth of their logits, leaves fewer candidates than top_k, or fewer parts."""
    rng = np.random.default_rng(left)
    B, V = 6, 20000
    x = settings(B, rng, k=[8, 64], t=[0.5, 1.0], p=[1.0, 0.9], m=[0.0, 0.01])
    x["logits"] = np.full((B, V), -np.inf, np.float32)
    for b in range(B):
        at = rng.permutation(V)[:left] if b % 2 else 4 * 256 * np.arange(left) % V + np.arange(left) // 19 * 7
        x["logits"][b, at] = 2 * rng.standard_normal(left).astype(np.float32)
    x["logits"][1][np.isinf(x["logits"][1])] = -100.0     # 36 temperatures below: without weight
    check(hip, x, most_open=0.4)


def test_infinities(hip):
    rng = np.random.default_rng(2)
    B, V = 6, 20000
    x = settings(B, rng, k=50, t=1.0, p=[1.0, 0.9], m=[0.0, 0.1])
    x["logits"] = rng.standard_normal((B, V), dtype=np.float32)
    x["logits"][:, ::3] = np.nan
    for b in range(B):
        x["logits"][b, rng.permutation(V)[:b * 15]] = np.inf
    check(hip, x, most_open=0.4)


@pytest.mark.parametrize("n", [60, 63, 64, 65, 66, 130])
def test_lists_of_a_wave(hip, n):
    """n candidates far above the others, all kept by top_k or by top_p alone."""
    rng = np.random.default_rng(n)
    for k in (64, 0):
        B, V = 4, 12000
        x = settings(B, rng, k=k, t=1.0, p=[0.5, 0.99], m=[0.0, 0.3])
        x["logits"] = rng.standard_normal((B, V), dtype=np.float32) - 60
        for b in range(B):
            x["logits"][b, rng.permutation(V)[:n]] = 0.01 * rng.standard_normal(n).astype(np.float32)
        check(hip, x, most_open=0.6)


def test_graph(hip):
    """A captured call whose rows change between small and large top_k, counts and lists, eagerly and replayed."""
    rng = np.random.default_rng(4)
    B, V = 3, 50000
    x = settings(B, rng, k=[20, 0, 500], t=1.0)
    x["logits"] = rows(rng, B, V, "any")
    with Buffers(hip, **x, token=np.zeros(B, np.int32), prob=np.zeros(B, np.float32)) as bufs:
        a = sample_args(bufs, B, V, V)
        g = Graph(hip, lambda s: pyq35.check(pyq35.lib.q35_sample(a, s)))
        try:
            for i in range(4):
                bufs.set("logits", rows(rng, B, V, ("falling", "any", "heap", "one lane")[i]))
                bufs.set("top_k", np.roll(np.array([20, 0, 500], np.int32), i))
                bufs.set("u", rng.random(B, dtype=np.float32))
                g.replay()
                first = bufs.get("token"), bufs.get("prob")
                bufs.set("token", np.full(B, -9, np.int32))
                pyq35.check(pyq35.lib.q35_sample(a, None))
                hip.sync()
                assert np.array_equal(first[0], bufs.get("token")) and np.array_equal(first[1], bufs.get("prob")) and (first[0] >= 0).all()
        finally:
            g.close()


def test_two_calls_at_once(hip):
    rng = np.random.default_rng(8)
    B, V = 6, 60000
    x = settings(B, rng, k=[0, 20, 300], t=[0.7, 1.5], p=[0.9, 1.0])
    x["logits"] = rows(rng, B, V, "any")
    y = dict(x, logits=rows(rng, B, V, "heap"), u=rng.random(B, dtype=np.float32))
    want = [run(hip, x), run(hip, y)]
    out = dict(token=np.zeros(B, np.int32), prob=np.zeros(B, np.float32))
    with Buffers(hip, **x, **out) as p, Buffers(hip, **y, **out) as q:
        s = [C.c_void_p(), C.c_void_p()]
        for i in s:
            hip._ck(hip.rt.hipStreamCreate(C.byref(i)), "hipStreamCreate")
        a, b = sample_args(p, B, V, V), sample_args(q, B, V, V)
        for _ in range(5):
            pyq35.check(pyq35.lib.q35_sample(a, s[0]))
            pyq35.check(pyq35.lib.q35_sample(b, s[1]))
        hip.sync()
        for d, w in ((p, want[0]), (q, want[1])):
            assert np.array_equal(d.get("token"), w[0]) and np.array_equal(d.get("prob"), w[1])
        for i in s:
            hip._ck(hip.rt.hipStreamDestroy(i), "hipStreamDestroy")
