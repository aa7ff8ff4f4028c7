"""q35_kv_evict against its definition: whole numbers and copies, so every bit has to agree.
Lengths around the budget, every kind of score, ties, protected rows, empty places, in place
and into other arrays, one row to 131072."""
import numpy as np
import pytest

import pyq35
from batch_ref import HD, Buffers, Graph, evict_args, evict_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def make(B, NKV, cap, lens, seed, bf16=False, kind="exp"):
    rng = np.random.default_rng(seed)
    shape = (B, NKV, cap)
    if kind == "exp":
        score = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
        score[rng.random(shape) < 0.1] = 0.0
    elif kind == "ties":
        score = rng.integers(0, 3, shape).astype(np.float32)
    elif kind == "same":
        score = np.full(shape, 0.25, np.float32)
    elif kind == "close":   # neighbours in the last bits
        score = (np.float32(1.0).view(np.uint32) + rng.integers(0, 50, shape).astype(np.uint32)).view(np.float32)
    else:                   # any bits: NaN, infinities, both zeros, subnormals, negative
        score = rng.integers(0, 1 << 32, shape, dtype=np.uint64).astype(np.uint32).view(np.float32)
        special = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45], np.float32)
        pick = rng.random(shape) < 0.5
        score[pick] = special[rng.integers(0, len(special), int(pick.sum()))]
    bits = np.uint16 if bf16 else np.uint32
    kv = [rng.integers(0, np.iinfo(bits).max, (B, NKV, cap, HD), dtype=bits) for _ in range(2)]
    pos = np.argsort(rng.random(shape), -1).astype(np.int32)
    return {"len": np.array(lens, np.int32), "next_pos": np.full(B, cap + 3, np.int32), "score": score, "pos": pos,
            "k": kv[0], "v": kv[1], "score_out": np.full(shape, 7.0, np.float32), "pos_out": np.full(shape, -7, np.int32),
            "new_len": np.full(B, -9, np.int32)}


def same(a, b):
    return np.array_equal(a.view(np.uint32) if a.dtype == np.float32 else a, b.view(np.uint32) if b.dtype == np.float32 else b)


def expect(x, keep, n_sink, n_recent, in_place):
    B, NKV, cap = x["score"].shape
    w = {c: x[c].copy() for c in ("k", "v")}
    w["score"] = x["score" if in_place else "score_out"].copy()
    w["pos"] = x["pos" if in_place else "pos_out"].copy()
    w["new_len"] = x["len"].copy()
    for b in range(B):
        n = int(x["len"][b])
        if n < 0 or n > cap:
            continue
        w["new_len"][b] = min(n, keep)
        for h in range(NKV):
            take = evict_rows(x["score"][b, h], x["pos"][b, h], n, keep, n_sink, n_recent, x["next_pos"][b])
            m = len(take)
            for c in ("k", "v", "score", "pos"):
                w[c][b, h, :m] = x[c][b, h][take]
    return w


def run(hip, x, keep, n_sink=0, n_recent=0, bf16=False, in_place=False):
    B, NKV, cap = x["score"].shape
    names = {"score_out": "score", "pos_out": "pos", "new_len": "len"} if in_place else {}
    with Buffers(hip, **x) as bufs:
        a = evict_args(bufs, B, NKV, cap, keep, n_sink, n_recent, bf16, **names)
        pyq35.check(pyq35.lib.q35_kv_evict(a, None))
        hip.sync()
        want = expect(x, keep, n_sink, n_recent, in_place)
        for c in want:
            got = bufs.get(names.get(c + "_out" if c in ("score", "pos") else c, c + "_out" if c in ("score", "pos") else c))
            assert same(got, want[c]), c
        if not in_place:
            assert same(bufs.get("score"), x["score"]) and same(bufs.get("pos"), x["pos"])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cap,keep", [(1, 1), (2, 1), (3, 2), (5, 5), (5, 9), (64, 63), (64, 1), (65, 32), (100, 64), (1000, 900),
                                      (1024, 1023), (1025, 512), (2304, 2048), (4099, 77)])
def test_lengths(hip, cap, keep, in_place):
    lens = [cap, min(cap, keep), min(cap, keep + 1), max(keep - 1, 0) if keep <= cap else cap, 0, cap - 1, -1, cap + 1, -2147483648,
            2147483647]
    x = make(len(lens), 2, cap, lens, seed=cap * 7 + keep)
    run(hip, x, keep, in_place=in_place, n_sink=min(2, keep // 2), n_recent=min(5, keep // 2))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", ["exp", "ties", "same", "close", "bits"])
def test_scores(hip, kind, bf16):
    for cap, keep in ((300, 200), (3001, 1500), (700, 3)):
        run(hip, make(3, 3, cap, [cap, cap - 7, cap // 2], seed=cap, bf16=bf16, kind=kind), keep, bf16=bf16)
        run(hip, make(1, 1, cap, [cap], seed=cap + 1, bf16=bf16, kind=kind), keep, 1, 2, bf16=bf16, in_place=True)


def test_protected_rows(hip):
    x = make(2, 2, 400, [400, 390], seed=3)
    for sink, recent in ((0, 0), (4, 60), (100, 0), (0, 100), (50, 50), (99, 1)):
        run(hip, x, 100, sink, recent)
    # more protected rows than stay (positions given twice): the lower slots stay
    x["pos"][:] = 2
    run(hip, x, 100, 4, 60)
    x["next_pos"][:] = [2147483647, -2147483648]
    run(hip, x, 100, 0, 100)


@pytest.mark.parametrize("cap,keep,bf16", [(131072, 32768, False), (131072, 100000, True), (70001, 5, False), (40000, 39999, True)])
def test_long(hip, cap, keep, bf16):
    x = make(1, 1, cap, [cap], seed=cap, bf16=bf16)
    run(hip, x, keep, min(4, keep // 2), min(64, keep // 2), bf16=bf16)


@pytest.mark.parametrize("kind", ["ties", "same", "close", "bits"])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_with_equal_scores(hip, kind, in_place):
    """More equal keys than the selection holds in LDS, and lengths that end within a slice."""
    cap = 40961
    x = make(3, 2, cap, [cap, 20000, 33000], seed=len(kind), bf16=True, kind=kind)
    for keep in (30000, 1):
        run(hip, x, keep, min(3, keep // 2), min(100, keep // 2), bf16=True, in_place=in_place)


@pytest.mark.parametrize("cap", [4096, 4097, 16384, 16385])
def test_around_the_forms_of_the_selection(hip, cap):
    lens = [cap, cap - 1, 2049, 2048, 2047, 0, -1, cap + 1]
    run(hip, make(len(lens), 1, cap, lens, seed=cap, bf16=True), 2048, 4, 64, bf16=True)
    run(hip, make(len(lens), 1, cap, lens, seed=cap, bf16=True, kind="close"), cap - 1, 4, 64, bf16=True, in_place=True)
    run(hip, make(2, 1, cap, [cap, 5], seed=cap, bf16=True), cap + 5, bf16=True)


def test_many_sequences(hip):
    rng = np.random.default_rng(4)
    x = make(64, 2, 96, rng.integers(-1, 98, 64), seed=4, bf16=True)
    run(hip, x, 64, 4, 16, bf16=True, in_place=True)


def test_again_on_the_result(hip):
    """An eviction of a cache that is within its budget changes nothing; in place, twice."""
    x = make(2, 2, 200, [200, 150], seed=6)
    with Buffers(hip, **x) as bufs:
        a = evict_args(bufs, 2, 2, 200, 128, 2, 8, False, score_out="score", pos_out="pos", new_len="len")
        pyq35.check(pyq35.lib.q35_kv_evict(a, None))
        once = {c: bufs.get(c) for c in ("k", "v", "score", "pos", "len")}
        pyq35.check(pyq35.lib.q35_kv_evict(a, None))
        assert all(same(bufs.get(c), once[c]) for c in once) and once["len"].tolist() == [128, 128]


def test_captured(hip):
    """A graph replayed on new scores and lengths, with eager work between, against the definition."""
    x = make(3, 2, 500, [500, 450, 100], seed=7)
    with Buffers(hip, **x) as bufs:
        a = evict_args(bufs, 3, 2, 500, 256, 4, 16, False)
        g = Graph(hip, lambda s: pyq35.check(pyq35.lib.q35_kv_evict(a, s)))
        for i in range(4):
            y = make(3, 2, 500, [500 - i, 257 + i, 500 - 100 * i], seed=70 + i)
            for c in y:
                bufs.set(c, y[c])
            g.replay()
            w = expect(y, 256, 4, 16, False)
            for c, n in (("k", "k"), ("v", "v"), ("score", "score_out"), ("pos", "pos_out"), ("new_len", "new_len")):
                assert same(bufs.get(n), w[c]), (i, c)
        g.close()
