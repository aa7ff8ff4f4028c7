"""q35_sample against its definition in float64: every filter alone and together, ties, ruled-out
candidates, infinities and NaN, extreme settings, one candidate to a full vocabulary, captured graphs.

Tolerance. Weights are whole multiples of 2^-S of the largest (S = 50, or 62 - n for 2^n candidates), so a
sum of V of them is off by at most V 2^-(S+1), and the float64 sums here by V 2^-53: a row whose
nearest border is closer than twice that, relative to the weight that is left, may go either way and is
not compared. A probability is off by a multiple of the weight left, the sum's error and its fp32 rounding."""
import numpy as np
import pytest

import pyq35
from batch_ref import Buffers, Graph
from q4_ref import sample64, sample_args

pytestmark = pytest.mark.gpu
lib = pyq35.lib


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def settings(B, rng, t=None, k=None, p=None, m=None, u=None):
    pick = lambda v, c: np.full(B, v) if np.isscalar(v) else rng.choice(c if v is None else v, B)  # noqa: E731
    return {"temperature": pick(t, [0.0, 0.3, 0.7, 1.0, 2.0]).astype(np.float32),
            "top_k": pick(k, [0, 1, 5, 40, 1000]).astype(np.int32), "top_p": pick(p, [1.0, 0.95, 0.5, 0.1]).astype(np.float32),
            "min_p": pick(m, [0.0, 0.01, 0.2]).astype(np.float32),
            "u": (rng.random(B, dtype=np.float32) if u is None else np.full(B, u) if np.isscalar(u) else np.asarray(u)).astype(np.float32)}


def run(hip, x, ld=None, drop=()):
    B, V = x["logits"].shape
    wide = np.full((B, ld or V), np.inf, np.float32)
    wide[:, :V] = x["logits"]
    arrays = dict(x, logits=wide, token=np.full(B, -7, np.int32), prob=np.full(B, -7, np.float32))
    for n in drop:
        arrays.pop(n)
    with Buffers(hip, **arrays) as bufs:
        pyq35.check(lib.q35_sample(sample_args(bufs, B, V, ld or V), None))
        hip.sync()
        return bufs.get("token"), bufs.get("prob") if "prob" not in drop else None


def check(hip, x, most_open=0.02, **kw):
    B, V = x["logits"].shape
    token, prob = run(hip, x, **kw)
    n = max(int(V - 1).bit_length(), 0)
    unit = 2.0 ** -min(50, 62 - n)
    near = 2 * V * (unit / 2 + 2.0 ** -53)
    left = 0
    for b in range(B):
        want, p, room = sample64(x["logits"][b], *(x[c][b] for c in ("temperature", "top_k", "top_p", "min_p", "u")))
        if room <= near:
            left += 1
            continue
        assert token[b] == want, f"row {b}: {token[b]} for {want}, room {room}, {[x[c][b] for c in x if c != 'logits']}"
        if prob is not None:
            assert abs(prob[b] - p) <= p * (2.0 ** -24 + near) + unit + 1e-45, f"row {b}: {prob[b]} for {p}"
    assert left <= most_open * B, f"{left} rows next to a border"
    return token, prob


def logits(B, V, rng, spread=2.0):
    return (spread * rng.standard_normal((B, V))).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 1000, 1024, 4095, 4097, 20011])
def test_all_filters(hip, V):
    rng = np.random.default_rng(V)
    check(hip, dict(logits=logits(60, V, rng), **settings(60, rng)))


@pytest.mark.parametrize("only", ["t", "k", "p", "m"])
@pytest.mark.parametrize("spread", [0.0001, 0.5, 3.0, 40.0])
def test_one_filter(hip, only, spread):
    rng = np.random.default_rng(5)
    off = dict(t=1.0, k=0, p=1.0, m=0.0)
    off[only] = None if only != "t" else [0.2, 0.9, 1.0, 1.7]
    check(hip, dict(logits=logits(50, 7001, rng, spread), **settings(50, rng, **off)))


@pytest.mark.parametrize("B", [1, 9, 70])
def test_full_vocabulary(hip, B):
    rng = np.random.default_rng(B)
    x = dict(logits=logits(B, 151936, rng, 2.0), **settings(B, rng, t=[0.6, 1.0, 1.3]))
    x["logits"][:, 77] += 9.0
    check(hip, x, most_open=0.1)


@pytest.mark.parametrize("V", [5, 3000, 151936])
def test_ties(hip, V):
    """Few distinct logits: most borders lie among equal ones, and the lower id comes first."""
    rng = np.random.default_rng(V)
    x = dict(logits=rng.integers(-2, 3, (40, V)).astype(np.float32), **settings(40, rng, t=[0.5, 1.0]))
    x["logits"][5] = 0.25
    x["logits"][6, ::2] = -0.0
    x["logits"][6, 1::2] = 0.0
    # top_k of 5, 40 or 1000 equal candidates and top_p of 0.95, 0.5 or 0.1 (to 2^-24) put the border within
    # 2^-24 of a whole candidate: 3 / 5 of 3 / 4 of the rows where the largest logit fills top_k
    check(hip, x, most_open=0.1 if V < 100000 else 0.5)


def test_equal_candidates_exactly(hip):
    """1024 equal candidates: every place's share is 1/1024, and borders belong to the next one."""
    B = 64
    x = dict(logits=np.full((B, 1024), 1.5, np.float32), **settings(B, np.random.default_rng(0), t=1.0, k=0, p=1.0, m=0.0))
    at = np.arange(B) * 16
    x["u"] = (at / 1024).astype(np.float32)
    token, prob = run(hip, x)
    assert np.array_equal(token, at) and np.allclose(prob, 1 / 1024, rtol=2.0 ** -23)
    x["top_k"][:] = 512
    x["top_p"][:] = 0.25                       # 128 are left
    x["u"] = (np.arange(B) / 64).astype(np.float32)
    token, prob = run(hip, x)
    assert np.array_equal(token, np.arange(B) * 2) and np.allclose(prob, 1 / 128, rtol=2.0 ** -23)


def test_ruled_out_and_not_finite(hip):
    rng = np.random.default_rng(3)
    B, V = 24, 3001
    x = dict(logits=logits(B, V, rng), **settings(B, rng, t=[0.0, 0.8, 1.0], k=[0, 30], p=[1.0, 0.9]))
    L = x["logits"]
    L[0], L[1] = -np.inf, np.nan
    L[2, :], L[2, 1234] = -np.inf, -5.0
    L[3, 100], L[3, 2000], L[3, 2500] = np.inf, np.inf, np.nan
    L[4, ::3] = np.nan
    L[5, 1:] = -np.inf
    L[6] = np.where(np.arange(V) % 2, -3.0e38, 3.0e38)
    L[7] = np.float32(1e-45) * rng.integers(0, 3, V)
    L[8, rng.random(V) < 0.95] = -np.inf
    L[9] = np.inf
    L[10] = -3.4028235e38
    x["temperature"][6], x["temperature"][10] = 1.0, 1.0
    token, prob = check(hip, x, most_open=0.1)
    assert token[0] == token[1] == -1 and prob[0] == prob[1] == 0 and token[2] == 1234 and token[5] == 0


def test_extreme_settings(hip):
    rng = np.random.default_rng(4)
    V = 500
    rows = [  # temperature, top_k, top_p, min_p, u
        (1e-38, 0, 1, 0, 0.9), (1e30, 0, 1, 0, 0.4999), (np.inf, 0, 1, 0, 0.123), (1, 2147483647, 1, 0, 0.3), (1, -2147483648, 1, 0, 0.3),
        (1, 0, 0, 0, 0.9), (1, 0, -1, 0, 0.9), (1, 0, 2, 0, 0.9), (1, 0, np.inf, 0, 0.9), (1, 0, 1, 1, 0.9), (1, 0, 1, 1.5, 0.9),
        (1, 0, 1, -1, 0.9), (1, 0, 1, np.inf, 0.9), (1, 0, 1e-30, 0, 0.9), (1, 500, 1, 0, 0.7), (1, 499, 1, 0, 0.9999999),
        (1, 501, 0.99999994, 1e-30, 0.7), (1, 1, 1, 0, 0.99), (0.0, 0, 0.5, 0.5, 0.5), (1e-45, 0, 0.7, 0.1, 0.6)]
    x = dict(logits=logits(len(rows), V, rng), **{c: np.array([r[i] for r in rows], np.int32 if c == "top_k" else np.float32)
                                                  for i, c in enumerate(("temperature", "top_k", "top_p", "min_p", "u"))})
    check(hip, x)


def test_numbers_outside_the_interval(hip):
    """u outside [0, 1): the nearest of it; not a number: 0. NaN filters are off."""
    rng = np.random.default_rng(5)
    one = logits(1, 300, rng)
    x = dict(logits=np.repeat(one, 8, 0), **settings(8, rng, t=1.0, k=0, p=1.0, m=0.0))
    x["u"] = np.array([0.0, -3.0, np.nan, -np.inf, 1.0, 7.0, np.inf, 0.0], np.float32)
    x["top_p"][7], x["min_p"][7] = np.nan, np.nan
    token, prob = run(hip, x)
    order = np.lexsort((np.arange(300), -one[0].astype(np.float64)))
    assert (token[[0, 1, 2, 3, 7]] == order[0]).all() and (token[4:7] == order[-1]).all()
    w = np.exp(one[0].astype(np.float64) - one.max())
    assert abs(prob[7] - 1 / w.sum()) < 1e-6


def test_empty_places_strides_and_no_filters(hip):
    rng = np.random.default_rng(6)
    x = dict(logits=logits(9, 1234, rng), **settings(9, rng, t=[0.7, 1.0]))
    x["temperature"][[1, 4]] = -1.0, np.nan
    token, prob = run(hip, x, ld=1300)
    assert (token[[1, 4]] == -7).all() and (prob[[1, 4]] == -7).all()
    on = [0, 2, 3, 5, 6, 7, 8]
    y = {n: a[on] for n, a in x.items()}
    t2, p2 = check(hip, y)
    assert np.array_equal(token[on], t2) and np.array_equal(prob[on], p2)
    y["top_k"][:], y["top_p"][:], y["min_p"][:] = 0, 1, 0
    a, _ = check(hip, y)
    b, _ = run(hip, y, drop=("top_k", "top_p", "min_p", "prob"))
    assert np.array_equal(a, b)


def test_graph(hip):
    """Logits, settings and numbers are read when the graph is replayed."""
    rng = np.random.default_rng(7)
    B, V = 6, 30000
    x = dict(logits=logits(B, V, rng), **settings(B, rng, t=1.0))
    with Buffers(hip, **x, token=np.zeros(B, np.int32), prob=np.zeros(B, np.float32)) as bufs:
        a = sample_args(bufs, B, V, V)
        g = Graph(hip, lambda s: pyq35.check(lib.q35_sample(a, s)))
        try:
            for i in range(5):
                y = dict(logits=logits(B, V, rng, 1.0 + i), **settings(B, rng))
                for n in y:
                    bufs.set(n, y[n])
                g.replay()
                token, prob = bufs.get("token"), bufs.get("prob")
                t2, p2 = check(hip, y, most_open=0.2)
                assert np.array_equal(token, t2) and np.array_equal(prob, p2)
        finally:
            g.close()


def test_frequencies(hip):
    """Over a grid of numbers every candidate is drawn as often as its share says."""
    rng = np.random.default_rng(8)
    V, n = 7, 4096
    one = logits(1, V, rng, 1.0)
    x = dict(logits=np.repeat(one, n, 0), **settings(n, rng, t=0.8, k=5, p=1.0, m=0.0, u=(np.arange(n) + 0.5) / n))
    token, _ = run(hip, x)
    w = np.exp((one[0].astype(np.float64) - one.max()) / np.float32(0.8))
    w[np.argsort(-one[0])[5:]] = 0
    assert (np.abs(np.bincount(token, minlength=V) - n * w / w.sum()) <= 1.0).all()
