"""q35_attn_batch against its definition in float64: head groups, cache types, prefix and own
lengths from nothing to several tiles and pieces, empty and full places, garbage behind the
lengths, rotary widths, accumulated weights, captured graphs and concurrent calls.

Tolerance. A score is a sum of 256 products, |q k| about 1 each for the normal rows here,
times 1/16: with each addition off by at most half a step of a partial sum of at most about 48
(3 sigma of sqrt(256)) the error is 256^0.5 * 48 * 2^-24 / 16 = 3e-6 at most where errors are
independent, plus the rounding of the query and the exponent (a score of 6 carries
6 * 2^-24 = 4e-7). The weights are off by that much relatively and the output is their mean of
rows: below the 1e-5 (REL_L2) that the other attention entry points are held to. Norm weights that
scale the scores by c scale the error by c. Appended rows are compared on their own: fp32 rows
to 8 * 2^-24 (norm, factor, rotation of two terms), bf16 ones to half a step, 2^-8, more, and the
definition then reads the row that the call appended, as a rounding may go either way."""
import numpy as np
import pytest

import pyq35
from batch_ref import (HD, Buffers, Graph, attn64, attn_args, cache_in, cache_out, rms64, rope64)
from helpers import REL_L2, bf16_bits, bf16_to_f32, rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def make(nq, nkv, P, lens, cap, seed, bf16=False, rot=64, prefix_cap=None, norm=0.1, pos=None):
    """Inputs; everything behind a length is NaN."""
    rng = np.random.default_rng(seed)
    B, pc = len(lens), P if prefix_cap is None else prefix_cap
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
    rnd = (lambda v: bf16_to_f32(bf16_bits(v))) if bf16 else (lambda v: v)
    x = {"qg": n(B, nq, 2 * HD), "k_new": n(B, nkv, HD), "v_new": n(B, nkv, HD), "q_norm": norm * n(HD),
         "k_norm": norm * n(HD), "rot": rot, "own_len": np.array(lens, np.int32),
         "pos": np.array([P + min(max(v, 0), cap) for v in lens] if pos is None else pos, np.int32),
         "k_prefix": rnd(n(nkv, pc, HD)), "v_prefix": rnd(n(nkv, pc, HD)),
         "k_own": rnd(n(B, nkv, cap, HD)), "v_own": rnd(n(B, nkv, cap, HD)),
         "own_score": np.abs(n(B, nkv, cap)), "own_pos": rng.integers(0, 1000, (B, nkv, cap)).astype(np.int32),
         "out": n(B, nq, HD)}
    for c in ("k_prefix", "v_prefix"):
        x[c][:, P:] = np.nan
    for b, v in enumerate(lens):
        for c in ("k_own", "v_own", "own_score"):
            x[c][b, :, max(v, 0):] = np.nan
    return x


def upload(hip, x, bf16):
    skip = ("rot",) + (() if x["k_prefix"].size else ("k_prefix", "v_prefix"))
    return Buffers(hip, **{k: cache_in(v, bf16) if k in ("k_prefix", "v_prefix", "k_own", "v_own") else v
                           for k, v in x.items() if k not in skip})


def check(x, got, P, bf16, scores=True, bar=REL_L2):
    B, nq, nkv, cap = x["qg"].shape[0], x["qg"].shape[1], x["k_new"].shape[1], x["k_own"].shape[2]
    G = nq // nkv
    for b in range(B):
        n = int(x["own_len"][b])
        same = lambda c, idx: np.array_equal(got[c][idx], x[c][idx], equal_nan=True)  # noqa: E731
        if n < 0 or n >= cap:
            assert all(same(c, b) for c in ("k_own", "v_own", "own_score", "own_pos")), f"place {b}"
            assert same("out", b) if n < 0 else np.isnan(got["out"][b]).all(), f"place {b}"
            continue
        # rows: the new one in its slot, the others as they were
        keep = np.arange(cap) != n
        assert same("k_own", (b, slice(None), keep)) and same("v_own", (b, slice(None), keep)), f"sequence {b}"
        k = rope64(rms64(x["k_new"][b], x["k_norm"]), x["pos"][b], x["rot"])
        step = 2.0 ** -8 if bf16 else 0.0
        big = np.abs(k).max(-1, keepdims=True)
        assert (np.abs(got["k_own"][b, :, n] - k) <= np.abs(k) * step + 8 * 2.0 ** -24 * big * (1 + step)).all()
        v = bf16_to_f32(bf16_bits(x["v_new"][b])) if bf16 else x["v_new"][b]
        assert np.array_equal(got["v_own"][b, :, n], v)
        rk = np.concatenate([x["k_prefix"][:, :P], got["k_own"][b, :, :n + 1]], 1)
        rv = np.concatenate([x["v_prefix"][:, :P], got["v_own"][b, :, :n + 1]], 1)
        out, w = attn64(x, b, rk, rv)
        for h in range(nq):
            assert rel_l2(got["out"][b, h], out[h]) < bar, f"sequence {b} head {h}"
        if not scores:
            assert same("own_score", b) and same("own_pos", b)
            continue
        own = w[:, P:].reshape(nkv, G, n + 1).sum(1)
        want = x["own_score"][b, :, :n + 1].astype(np.float64)
        want[:, n] = 0.0
        # the weight's relative error, and the rounding of the sum
        err = np.abs(got["own_score"][b, :, :n + 1] - (want + own))
        assert (err <= bar * own + 2.0 ** -24 * (want + own) + 1e-37).all(), f"sequence {b}"
        assert same("own_score", (b, slice(None), slice(n + 1, None)))
        assert (got["own_pos"][b, :, n] == x["pos"][b]).all() and same("own_pos", (b, slice(None), keep))


def run(hip, x, P, bf16, scores=True, bar=REL_L2):
    B, cap = x["qg"].shape[0], x["k_own"].shape[2]
    with upload(hip, x, bf16) as bufs:
        a = attn_args(bufs, x, bf16, cap, P, x["k_prefix"].shape[1], scores)
        pyq35.check(pyq35.lib.q35_attn_batch(a, None))
        hip.sync()
        got = {c: bufs.get(c) for c in ("out", "k_own", "v_own", "own_score", "own_pos")}
    got["k_own"], got["v_own"] = cache_out(got["k_own"]), cache_out(got["v_own"])
    check(x, got, P, bf16, scores, bar)
    return got


HEADS = [(16, 2), (8, 2), (2, 1), (4, 1), (2, 2), (16, 1), (6, 2), (5, 1), (10, 1), (39, 3)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("nq,nkv", HEADS)
def test_head_groups(hip, nq, nkv, bf16):
    x = make(nq, nkv, 77, [0, 1, 30, 5, -1], 40, seed=nq * 31 + nkv, bf16=bf16, prefix_cap=100)
    run(hip, x, 77, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 500, 2047, 4133])
def test_prefix_lengths(hip, P, bf16):
    x = make(8, 2, P, [0, 3, 33], 34, seed=P, bf16=bf16, prefix_cap=P + (P % 3))
    run(hip, x, P, bf16, scores=P % 2 == 1)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("lens,cap", [([0], 1), ([0, 1, 2], 3), ([14, 15, 16, 17], 18), ([30, 31, 32, 33], 64),
                                      ([62, 63, 64, 65, 66], 67), ([127, 128, 200, 0], 1000), ([999, 500, 998], 1000),
                                      ([3000], 3001), ([2303, 100, -1, 1700], 2304)])
def test_own_lengths(hip, lens, cap, bf16):
    for P in (0, 40):
        run(hip, make(8, 2, P, lens, cap, seed=cap + P, bf16=bf16), P, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B", [1, 2, 3, 4, 7, 8, 9, 16, 17, 33, 64, 65])
def test_batch_sizes(hip, B, bf16):
    rng = np.random.default_rng(B)
    for nq in (16, 8):
        lens = rng.integers(0, 70, B).tolist()
        run(hip, make(nq, 2, 301, lens, 70, seed=B, bf16=bf16), 301, bf16, scores=B % 2 == 0)


@pytest.mark.parametrize("bf16", [False, True])
def test_empty_and_full_places(hip, bf16):
    for lens in ([-1, 3, -5, 0, -2147483648], [-1, -1], [7, 8, 9, 2147483647, 6], [8]):
        for P in (0, 50):
            run(hip, make(4, 1, P, lens, 8, seed=P + len(lens), bf16=bf16), P, bf16)


@pytest.mark.parametrize("rot", [0, 2, 18, 64, 96, 256])
def test_rotary_widths_and_far_positions(hip, rot):
    pos = [0, 5, 131071, 2147483600]
    run(hip, make(8, 2, 60, [0, 4, 9, 20], 21, seed=rot, rot=rot, pos=pos), 60, False)


@pytest.mark.parametrize("bf16", [False, True])
def test_peaked_scores(hip, bf16):
    # norm weights of 2: queries and keys three times as long, scores of nine times the spread
    x = make(16, 2, 700, [0, 40, 300], 301, seed=5, bf16=bf16)
    x["q_norm"][:] = 2.0
    x["k_norm"][:] = 2.0
    for c in ("k_prefix", "k_own"):
        x[c] *= 4.0   # a power of two: bf16 rows stay exact
    run(hip, x, 700, bf16, bar=12 * REL_L2)


def test_rows_far_below_the_others(hip):
    """Keys whose scores underflow against the largest: their weights are 0, others' exact."""
    x = make(4, 1, 200, [0, 64, 100], 128, seed=6)
    x["k_prefix"] *= 2.0 ** -20
    x["k_own"] *= 2.0 ** 6
    run(hip, x, 200, False, bar=64 * REL_L2)


def test_nothing_else_is_written(hip):
    """Outputs and rows of a second batch directly behind the first one's stay as they are."""
    x = make(8, 2, 50, [3, 9, 0, 5], 10, seed=8)
    with upload(hip, x, False) as bufs:
        full = {c: bufs.get(c) for c in ("out", "k_own", "v_own", "own_score", "own_pos")}
        a = attn_args(bufs, x, False, 10, 50, 50)
        a.batch = 2
        pyq35.check(pyq35.lib.q35_attn_batch(a, None))
        hip.sync()
        for c, was in full.items():
            assert np.array_equal(bufs.get(c)[2:], was[2:], equal_nan=True), c


@pytest.mark.parametrize("bf16", [False, True])
def test_same_bits_again(hip, bf16):
    x = make(16, 2, 1000, [5, 200, 64, 0, 90], 256, seed=9, bf16=bf16)
    a, b = run(hip, x, 1000, bf16), run(hip, x, 1000, bf16)
    assert all(np.array_equal(a[c], b[c], equal_nan=True) for c in a)


@pytest.mark.parametrize("bf16", [False, True])
def test_captured_steps(hip, bf16):
    """One graph of the call replayed over steps whose lengths and positions change on the device,
    against eager calls of the same steps."""
    x = make(8, 2, 333, [0, 7, -1, 62], 80, seed=10, bf16=bf16)
    steps = 5
    rng = np.random.default_rng(1)
    qs = [rng.standard_normal(x["qg"].shape, dtype=np.float32) for _ in range(steps)]
    res = []
    for graph in (False, True):
        with upload(hip, x, bf16) as bufs:
            a = attn_args(bufs, x, bf16, 80, 333, 333)
            g = Graph(hip, lambda s: pyq35.check(pyq35.lib.q35_attn_batch(a, s))) if graph else None
            outs = []
            for i in range(steps):
                bufs.set("qg", qs[i])
                bufs.set("own_len", np.where(x["own_len"] >= 0, x["own_len"] + i, -1))
                bufs.set("pos", x["pos"] + i)
                if g:
                    g.replay()
                else:
                    pyq35.check(pyq35.lib.q35_attn_batch(a, None))
                    hip.sync()
                outs.append({c: bufs.get(c) for c in ("out", "k_own", "v_own", "own_score", "own_pos")})
            if g:
                g.close()
            res.append(outs)
    for i in range(steps):
        for c in res[0][i]:
            assert np.array_equal(res[0][i][c], res[1][i][c], equal_nan=True), (i, c)


def test_two_calls_at_once(hip):
    """Two batches on two streams, each with a workspace of its own."""
    import ctypes as C
    xs = [make(16, 2, 2000, [5, 60, 33], 64, seed=s) for s in (1, 2)]
    alone = [run(hip, x, 2000, False) for x in xs]
    streams = [C.c_void_p() for _ in xs]
    bufs = [upload(hip, x, False) for x in xs]
    for s in streams:
        hip._ck(hip.rt.hipStreamCreate(C.byref(s)), "hipStreamCreate")
    args = [attn_args(b, x, False, 64, 2000, 2000) for b, x in zip(bufs, xs)]
    hip.sync()
    for a, s in zip(args, streams):
        pyq35.check(pyq35.lib.q35_attn_batch(a, s))
    hip.sync()
    for b, ref in zip(bufs, alone):
        assert all(np.array_equal(b.get(c), ref[c], equal_nan=True) for c in ref)
    for s, b in zip(streams, bufs):
        hip._ck(hip.rt.hipStreamDestroy(s), "hipStreamDestroy")
        b.__exit__()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("order", [1, -1])
def test_value_rows_of_every_size(hip, order, bf16):
    """Value rows of one sequence over 2^-60 .. 2^60, rising or falling, with scores that make the small
    ones count: each row's size is undone by its score, 0.69 a power of two, so that the weights
    move by e^83. The keys' errors (a score of 40 carries 40 * 2^-24 and 3e-6 a unit of its norm)
    set the bar: 40 times the usual one. Next to them a sequence of ordinary rows."""
    x = make(16, 2, 640, [0, 100, 70, 3, 33, 20, 64], 101, seed=12, bf16=bf16)
    p = np.linspace(-60, 60, 640)[::order]
    q = rope64(rms64(x["qg"][2, :, :HD], x["q_norm"]), x["pos"][2], x["rot"])
    for kv in range(2):
        u = q[8 * kv] / np.linalg.norm(q[8 * kv])
        k = x["k_prefix"][kv] - np.outer(x["k_prefix"][kv] @ u, u)
        k = k + np.outer(-np.round(p) * np.log(2.0) * 16.0 / np.linalg.norm(q[8 * kv]), u)
        x["k_prefix"][kv] = bf16_to_f32(bf16_bits(k.astype(np.float32))) if bf16 else k.astype(np.float32)
        x["v_prefix"][kv] *= np.exp2(np.round(p))[:, None].astype(np.float32)
    run(hip, x, 640, bf16, bar=40 * REL_L2)


@pytest.mark.parametrize("big", [2.0 ** 40, 2.0 ** -40, 2.0 ** 100, 2.0 ** -90])
def test_scales_of_values(hip, big):
    """All value rows times a power of two, and every other row: results scale with them."""
    x = make(16, 2, 300, [5, 40, 0, 12, 9, 22, 7, 1], 64, seed=13)
    for c in ("v_prefix", "v_own", "v_new"):
        x[c] *= np.float32(big)
    run(hip, x, 300, False)
    x["v_prefix"][:, ::2] *= np.float32(1.0 / big)
    run(hip, x, 300, False)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan, 3e38])
@pytest.mark.parametrize("where", ["v_prefix", "k_prefix", "v_own", "k_own", "qg"])
@pytest.mark.parametrize("nq", [16, 2])
def test_no_wrong_finite_outputs(hip, nq, where, what, bf16):
    """One infinity, NaN or value near the type's largest: an output that depends on it is the
    definition's or not finite (a square of 3e38 is no float, so not that in a query), all others are
    as without it. The bar: ten times that of a run, of the value or of the outputs' mean size."""
    if where == "qg" and what == 3e38:
        what = -np.nan
    x = make(nq, 2, 500, [20, 40, 0, 30, 12, 9, 5, 3], 64, seed=14, bf16=bf16)
    clean = run(hip, x, 500, bf16)["out"]
    at = {"v_prefix": (1, 77, 5), "k_prefix": (1, 77, 5), "v_own": (3, 1, 11, 5), "k_own": (3, 1, 11, 5), "qg": (3, nq - 1, 5)}[where]
    val = np.array([what], np.float32)
    x[where][at] = bf16_to_f32(bf16_bits(val))[0] if bf16 and where != "qg" else val[0]
    with upload(hip, x, bf16) as bufs:
        pyq35.check(pyq35.lib.q35_attn_batch(attn_args(bufs, x, bf16, 64, 500, 500), None))
        hip.sync()
        got, ko, vo = bufs.get("out"), cache_out(bufs.get("k_own")), cache_out(bufs.get("v_own"))
    seen = np.zeros(got.shape[:2], bool)
    if where == "qg":
        seen[3, nq - 1] = True
    elif where.endswith("own"):
        seen[3, nq // 2:] = True
    else:
        seen[:, nq // 2:] = True
    assert np.array_equal(got[~seen], clean[~seen])
    size = np.sqrt(np.mean(clean.astype(np.float64) ** 2))
    for b in range(8):
        n = x["own_len"][b] + 1
        with np.errstate(all="ignore"):
            want = attn64(x, b, np.concatenate([x["k_prefix"], ko[b, :, :n]], 1), np.concatenate([x["v_prefix"], vo[b, :, :n]], 1))[0]
        fine = np.isfinite(got[b]) & seen[b][:, None]
        assert (np.abs(got[b] - want) <= 10 * REL_L2 * np.maximum(np.abs(want), size))[fine].all(), f"sequence {b}"


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("nq,nkv,P,lens,cap", [(8, 1, 20000, [63], 64), (16, 1, 20000, [10, 63, -1, 5], 64), (2, 2, 1, [4999, 70], 5000),
                                               (1, 1, 0, [59999], 60000), (4, 1, 9000, [8000, 3], 9000)])
def test_many_pieces(hip, nq, nkv, P, lens, cap, bf16):
    """More pieces of a row than a wave has lanes (its merge then takes several a lane)."""
    run(hip, make(nq, nkv, P, lens, cap, seed=P + cap, bf16=bf16), P, bf16)
