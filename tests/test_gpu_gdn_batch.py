"""q35_gdn_batch against the recurrence in float64 (the bar of the other GDN entry points): one
token and ragged ones, in place and forked from one prompt's state, shared and own k-heads, with
and without the gated norm, padded rows, strides, empty places; and bit for bit against itself
when tokens come in one call or in several."""
import numpy as np
import pytest

import pyq35
from batch_ref import D, Buffers, Graph, gdn64, gdn_args
from helpers import REL_L2, rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def make(KH, VH, counts, seed, one=False, norm=True, fork=False, spare=3, pos=None):
    """Rows of the tokens and `spare` behind the last; leading dimensions wider than the rows."""
    rng = np.random.default_rng(seed)
    B, rows = len(counts), int(np.sum(counts)) + spare
    CONV, VD = (2 * KH + VH) * D, VH * D
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
    x = {"KH": KH, "VH": VH, "qkv": n(rows, CONV + 5), "z": n(rows, VD + 2), "b": n(rows, VH + 1), "a": n(rows, VH + 1),
         "conv_w": 0.5 * n(CONV, 4), "A_log": n(VH), "dt_bias": n(VH), "norm_w": 1 + 0.1 * n(D) if norm else None,
         "ring": n(B, 4, CONV), "state": 0.1 * n(B, VH, D, D), "out": n(rows, VD),
         "pos": np.array(rng.integers(0, 50, B) if pos is None else pos, np.int32),
         "row0": None if one else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), "counts": list(counts)}
    if fork:
        x["ring_in"], x["state_in"] = n(4, CONV), 0.1 * n(VH, D, D)
    return x


def call(hip, bufs, x, rows, fork=False, **over):
    a = gdn_args(bufs, x, len(x["counts"]), rows, fork)
    for k, v in over.items():
        setattr(a, k, v)
    pyq35.check(pyq35.lib.q35_gdn_batch(a, None))
    hip.sync()
    return {c: bufs.get(c) for c in ("out", "ring", "state")}


def device(hip, x):
    return Buffers(hip, **{k: v for k, v in x.items() if k not in ("KH", "VH", "counts")})


def check(x, got, fork=False):
    first = 0
    done = np.zeros(len(x["out"]), bool)
    for b, n in enumerate(x["counts"]):
        pos = int(x["pos"][b])
        if pos < 0:
            assert all(np.array_equal(got[c][b], x[c][b]) for c in ("ring", "state")), f"place {b}"
        else:
            ring, state = (x["ring_in"], x["state_in"]) if fork else (x["ring"][b], x["state"][b])
            out, ring, state = gdn64(x, b, first, n, pos, ring, state)
            for t in range(n):
                assert rel_l2(got["out"][first + t], out[t]) < REL_L2, f"sequence {b} token {t}"
            done[first:first + n] = True
            assert rel_l2(got["state"][b], state) < REL_L2, f"sequence {b}"
            assert np.array_equal(got["ring"][b], ring.astype(np.float32)), f"sequence {b}"
        first += n
    assert np.array_equal(got["out"][~done], x["out"][~done])


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("fork", [False, True])
@pytest.mark.parametrize("KH,VH,B", [(16, 16, 1), (2, 2, 5), (2, 4, 7), (1, 3, 4), (16, 16, 9), (8, 16, 33)])
def test_one_token(hip, KH, VH, B, fork, norm):
    x = make(KH, VH, [1] * B, seed=B + VH, one=True, norm=norm, fork=fork)
    with device(hip, x) as bufs:
        check(x, call(hip, bufs, x, B, fork), fork)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("fork", [False, True])
@pytest.mark.parametrize("KH,VH,counts", [(2, 2, [1]), (2, 2, [0, 1, 2, 3, 4, 5]), (2, 4, [7, 8, 9, 0, 16, 17]), (1, 3, [0, 0]),
                                          (4, 4, [40, 1, 0, 23]), (16, 16, [3, 1, 5])])
def test_ragged(hip, KH, VH, counts, fork, norm):
    x = make(KH, VH, counts, seed=sum(counts) + VH, norm=norm, fork=fork)
    with device(hip, x) as bufs:
        check(x, call(hip, bufs, x, len(x["out"]), fork), fork)


@pytest.mark.parametrize("one", [True, False])
def test_empty_places(hip, one):
    counts = [1, 1, 1, 1] if one else [2, 0, 3, 1]
    for fork in (False, True):
        x = make(2, 4, counts, seed=1, one=one, fork=fork, pos=[5, -1, -2147483648, 2147483647])
        if not one:
            x["pos"][3] = 2147483640
        with device(hip, x) as bufs:
            check(x, call(hip, bufs, x, len(x["out"]), fork), fork)


def test_rows_beyond_the_buffer(hip):
    """Offsets past `rows` are cut there: what lies behind is neither read nor written."""
    x = make(2, 2, [2, 3], seed=2, spare=0)
    with device(hip, x) as bufs:
        got = call(hip, bufs, x, 4)
    x["counts"] = [2, 2]
    check(x, got)


def test_strides_of_rings_and_states(hip):
    """Sequences' rings and states apart from each other, read from other ones of another stride."""
    KH, VH, B = 2, 2, 3
    CONV, S = (2 * KH + VH) * D, VH * D * D
    x = make(KH, VH, [1, 4, 0], seed=3)
    rng = np.random.default_rng(0)
    wide = {"ring": rng.standard_normal((B, 4 * CONV + 12), dtype=np.float32),
            "state": rng.standard_normal((B, S + 4), dtype=np.float32),
            "ring_in": rng.standard_normal((B, 4 * CONV + 4), dtype=np.float32),
            "state_in": 0.1 * rng.standard_normal((B, S + 64), dtype=np.float32)}
    with device(hip, {**x, **wide}) as bufs:
        got = call(hip, bufs, x, len(x["out"]), True, stride_ring=4 * CONV + 12, stride_state=S + 4,
                   stride_ring_in=4 * CONV + 4, stride_state_in=S + 64)
        assert all(np.array_equal(bufs.get(c), wide[c]) for c in ("ring_in", "state_in"))
    assert np.array_equal(got["ring"][:, 4 * CONV:], wide["ring"][:, 4 * CONV:])
    assert np.array_equal(got["state"][:, S:], wide["state"][:, S:])
    x["ring"], x["state"] = wide["ring_in"][:, :4 * CONV].reshape(B, 4, CONV), wide["state_in"][:, :S].reshape(B, VH, D, D)
    got["ring"], got["state"] = got["ring"][:, :4 * CONV].reshape(B, 4, CONV), got["state"][:, :S].reshape(B, VH, D, D)
    check(x, got)


def test_extreme_gates(hip):
    """Decays of nearly 1 and of 0, beta of 0 and 1, and rows of zeros (norms of eps)."""
    x = make(2, 2, [3, 2], seed=4)
    x["a"][0], x["a"][1], x["a"][2] = 50.0, -50.0, 0.0
    x["b"][0], x["b"][1] = -100.0, 100.0
    x["qkv"][3] = 0.0
    x["z"][4] = -90.0
    x["ring"][1] = 0.0
    with device(hip, x) as bufs:
        got = call(hip, bufs, x, len(x["out"]))
    out, ring, state = gdn64(x, 0, 0, 3, int(x["pos"][0]), x["ring"][0], x["state"][0])
    assert all(rel_l2(got["out"][t], out[t]) < REL_L2 for t in range(3)) and rel_l2(got["state"][0], state) < REL_L2
    assert np.isfinite(got["out"]).all() and np.isfinite(got["state"]).all()


def test_tokens_at_once_or_one_by_one(hip):
    x = make(2, 4, [6, 6], seed=5)
    with device(hip, x) as bufs:
        whole = call(hip, bufs, x, 12)
    with device(hip, x) as bufs:
        for t in range(6):
            bufs.set("pos", x["pos"] + t)
            # row t of both sequences: the second one's rows lie six further on
            for b in range(2):
                bufs.set("row0", np.where(np.arange(3) <= b, b * 6 + t, b * 6 + t + 1).astype(np.int32))
                call(hip, bufs, x, 12)
        parts = {c: bufs.get(c) for c in ("out", "ring", "state")}
    # the call for sequence b gives sequence 0 no token (equal offsets) or the other way round
    assert all(np.array_equal(whole[c][:12] if c == "out" else whole[c], parts[c][:12] if c == "out" else parts[c]) for c in whole)


def test_one_token_forms_agree(hip):
    x = make(4, 8, [1] * 6, seed=6, one=True)
    with device(hip, x) as bufs:
        a = call(hip, bufs, x, 6)
    x["row0"] = np.arange(7, dtype=np.int32)
    with device(hip, x) as bufs:
        b = call(hip, bufs, x, 6)
    assert all(np.array_equal(a[c], b[c]) for c in a)


def test_against_the_decode_entry(hip):
    """One sequence: the same results as q35_gdn_decode to its rounding."""
    x = make(16, 16, [1], seed=7, one=True, spare=0, pos=[11])
    with device(hip, x) as bufs:
        got = call(hip, bufs, x, 1)
    with device(hip, x) as bufs:
        a = pyq35.GdnDecodeArgs(n_layers=1, k_heads=16, v_heads=16, head_dim_k=D, head_dim_v=D, conv_kernel=4, pos=11,
                                eps=1e-6, conv_ring=bufs.p["ring"],
                                **{n: bufs.p[n] for n in ("qkv", "z", "b", "a", "conv_w", "A_log", "dt_bias", "norm_w", "state",
                                                          "out")})
        pyq35.check(pyq35.lib.q35_gdn_decode(a, None))
        hip.sync()
        ref = {c: bufs.get(c) for c in ("out", "ring", "state")}
    assert np.array_equal(got["ring"], ref["ring"])
    assert rel_l2(got["out"], ref["out"]) < REL_L2 and rel_l2(got["state"], ref["state"]) < REL_L2


def test_captured(hip):
    """A graph of a ragged call replayed on new rows, offsets and positions, against eager calls."""
    x = make(2, 4, [2, 0, 3], seed=8)
    rng = np.random.default_rng(2)
    feeds = [(rng.standard_normal(x["qkv"].shape, dtype=np.float32), r0) for r0 in ([0, 2, 2, 5], [0, 0, 4, 8], [0, 1, 2, 3])]
    res = []
    for graph in (False, True):
        with device(hip, x) as bufs:
            a = gdn_args(bufs, x, 3, 8)
            g = Graph(hip, lambda s: pyq35.check(pyq35.lib.q35_gdn_batch(a, s))) if graph else None
            pos, outs = x["pos"].copy(), []
            for qkv, r0 in feeds:
                bufs.set("qkv", qkv)
                bufs.set("row0", r0)
                bufs.set("pos", pos)
                if g:
                    g.replay()
                else:
                    pyq35.check(pyq35.lib.q35_gdn_batch(a, None))
                    hip.sync()
                pos = pos + np.diff(r0)
                outs.append({c: bufs.get(c) for c in ("out", "ring", "state")})
            if g:
                g.close()
            res.append(outs)
    for i, (u, v) in enumerate(zip(*res)):
        assert all(np.array_equal(u[c], v[c]) for c in u), i


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("fork", [False, True])
@pytest.mark.parametrize("KH,VH", [(8, 16), (16, 16)])
def test_many_sequences(hip, KH, VH, fork, norm):
    """More workgroups than the chip holds at three a compute unit: four waves a head."""
    counts = np.random.default_rng(VH + KH).integers(0, 12, 60).tolist()
    x = make(KH, VH, counts, seed=KH, norm=norm, fork=fork)
    x["pos"][[3, 59]] = -1
    with device(hip, x) as bufs:
        check(x, call(hip, bufs, x, len(x["out"]), fork), fork)
