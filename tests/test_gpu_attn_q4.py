"""q35_attn_q4 against its definition in float64 over the rows as the cache holds them: head groups,
lengths from nothing to many pieces, empty and full places, garbage behind the lengths, rotary widths,
peaked and flat weights, rows without values, offsets beyond 32 bits, captured graphs, concurrent calls.

Tolerance. Scores are sums of 256 products of about 1 each, times 1/16: with every addition off by half a
step of partial sums of at most about 48, 3e-6 at most, and 24-bit multiples of a query's largest entry add
2^-23 of 256 products' largest, less than that. Weights enter to 2^-23 of the largest beside them, so the
output, their mean of rows, keeps within the 1e-5 (REL_L2) that the other attention entry points are
held to. Appended rows are whole numbers and fp16 values from 64-bit sums: every bit has to agree."""
import ctypes as C

import numpy as np
import pytest

import pyq35
from batch_ref import HD, Buffers, Graph, attn64
from helpers import REL_L2, rel_l2
from q4_ref import attn_q4_args, row_codes, row_values, same_rows, turned

pytestmark = pytest.mark.gpu
lib = pyq35.lib


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def cache(rng, *shape, size=1.0):
    step = size * (0.30 + 0.05 * rng.standard_normal((*shape, 4)))
    least = -7.5 * step + 0.2 * size * rng.standard_normal((*shape, 4))
    return rng.integers(0, 256, (*shape, 128), dtype=np.uint8), np.stack([step, least], -1).astype(np.float16)


def make(nq, nkv, lens, cap, seed, rot=64, norm=0.1, pos=None, size=1.0):
    """Inputs; scales behind a length are NaN, codes there are whatever they are."""
    rng = np.random.default_rng(seed)
    B = len(lens)
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
    x = {"qg": n(B, nq, 2 * HD), "k_new": n(B, nkv, HD), "v_new": n(B, nkv, HD), "q_norm": norm * n(HD), "k_norm": norm * n(HD),
         "rot": rot, "len": np.array(lens, np.int32),
         "pos": np.array([min(max(v, 0), cap) + 5 for v in lens] if pos is None else pos, np.int32), "out": n(B, nq, HD)}
    for c in ("k", "v"):
        x[c], x[c + "_scale"] = cache(rng, B, nkv, cap, size=size)
        for b, v in enumerate(lens):
            x[c + "_scale"][b, :, max(v, 0):] = np.nan
    return x


def check(x, got, bar=REL_L2):
    B, nq, cap = x["qg"].shape[0], x["qg"].shape[1], x["k"].shape[2]
    for b in range(B):
        n = int(x["len"][b])
        if n < 0 or n >= cap:
            for c in ("k", "v"):
                assert np.array_equal(got[c][b], x[c][b]) and same_rows(got[c + "_scale"][b], x[c + "_scale"][b]), f"place {b}"
            assert np.array_equal(got["out"][b], x["out"][b]) if n < 0 else np.isnan(got["out"][b]).all(), f"place {b}"
            continue
        rows = {}
        for c, new in (("k", turned(x, b, x["k_new"][b], x["k_norm"])), ("v", x["v_new"][b])):
            want, scale = x[c][b].copy(), x[c + "_scale"][b].copy()
            want[:, n], scale[:, n] = row_codes(new)
            assert np.array_equal(got[c][b], want) and same_rows(got[c + "_scale"][b], scale), f"sequence {b} {c}"
            rows[c] = row_values(got[c][b, :, :n + 1], got[c + "_scale"][b, :, :n + 1])
        out, _ = attn64(x, b, rows["k"], rows["v"])
        for h in range(nq):
            assert rel_l2(got["out"][b, h], out[h]) < bar, f"sequence {b} head {h}: {rel_l2(got['out'][b, h], out[h])}"


def upload(hip, x):
    return Buffers(hip, **{n: a for n, a in x.items() if n != "rot"})


OUT = ("out", "k", "v", "k_scale", "v_scale")


def run(hip, x, bar=REL_L2):
    with upload(hip, x) as bufs:
        a = attn_q4_args(bufs, x, x["k"].shape[2])
        pyq35.check(lib.q35_attn_q4(a, None))
        hip.sync()
        got = {c: bufs.get(c) for c in OUT}
    if bar:
        check(x, got, bar)
    return got


@pytest.mark.parametrize("nq,nkv", [(16, 2), (8, 2), (2, 1), (4, 1), (2, 2), (16, 1), (6, 2), (5, 1), (10, 1), (39, 3), (14, 2), (24, 2)])
def test_head_groups(hip, nq, nkv):
    run(hip, make(nq, nkv, [0, 3, 77, -1, 130], 131, nq))


@pytest.mark.parametrize("cap", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 500, 511, 513, 1025])
def test_lengths(hip, cap):
    run(hip, make(8, 2, [cap - 1, cap // 2, 0, cap, -1], cap, cap))


@pytest.mark.parametrize("rot", [0, 2, 6, 32, 62, 64, 128, 254, 256])
def test_rotary_widths(hip, rot):
    run(hip, make(4, 2, [5, 60], 70, rot, rot=rot, pos=[123456, 7]))


def test_every_place_empty_or_full(hip):
    run(hip, make(8, 2, [-1, -5, 40, 41, 2147483647], 40, 1))
    run(hip, make(8, 2, [-1], 40, 1))


@pytest.mark.parametrize("lens", [[2999], [3000 - 1, 100, 0, 1700, -1, 2500, 64], [2048 - 1] * 20])
def test_long(hip, lens):
    run(hip, make(16, 2, lens, 3001, 2))


def test_very_long(hip):
    run(hip, make(8, 1, [40000], 40001, 3))


@pytest.mark.parametrize("norm", [0.0, 1.0, 3.0])
def test_peaked_and_flat(hip, norm):
    """Norm weights scale the scores and their error; flat weights: a query of zeros."""
    x = make(8, 2, [400, 39], 401, 4, norm=norm)
    big = (1 + np.abs(x["q_norm"]).max())
    run(hip, x, REL_L2 * max(1.0, big * big))
    x = make(8, 2, [400, 39], 401, 4, norm=0.1)
    x["q_norm"][:] = -1.0
    run(hip, x)


@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_sizes_of_rows(hip, size):
    x = make(8, 2, [300, 17], 301, 6, size=size)
    if size > 1:
        x["k_scale"] = (x["k_scale"].astype(np.float32) / size).astype(np.float16)   # large values, scores as they were
    run(hip, x)


def test_rows_of_one_value(hip):
    """Steps of zero; a single group that stands out; equal rows."""
    x = make(8, 2, [200, 90], 201, 7)
    x["k_scale"][0, :, :90, :, 0] = 0
    x["v_scale"][0, :, 20:120, :, 0] = 0
    x["k"][1], x["k_scale"][1, :, :90] = x["k"][1, :, :1], x["k_scale"][1, :, :1]
    x["v_new"][1] = 2.5
    x["v_scale"][0, 0, 150, 2] = [200.0, -1500.0]
    run(hip, x)


def test_rows_without_values(hip):
    """A key row with a NaN group has no score: its head's outputs are NaN, the others are as without
    it. A value row's NaN group takes its 64 dims. Infinities and NaN in the inputs stay where they are."""
    x = make(8, 2, [200, 90, 300, 31], 301, 8)
    x["k_scale"][0, 1, 130, 2] = np.nan
    x["v_scale"][1, 0, 60, 1] = np.nan
    x["qg"][2, 3, 7] = np.inf
    x["qg"][2, 5, 8] = np.nan
    x["v_new"][3, 1, 255] = np.nan
    got = run(hip, x, None)
    assert np.isnan(got["out"][0, 4:]).all() and np.isnan(got["out"][1, :4, 64:128]).all()
    assert np.isnan(got["out"][2, 3]).all() and np.isnan(got["out"][2, 5]).all()
    assert np.isnan(got["out"][3, 4:, 192:]).all()
    bad = np.isnan(got["out"])
    assert bad.sum() == 4 * HD + 4 * 64 + 2 * HD + 4 * 64
    y = {n: np.copy(a) for n, a in x.items() if n != "rot"}
    y["rot"] = 64
    y["k_scale"][0, 1, 130, 2] = 0.1
    y["v_scale"][1, 0, 60, 1] = 0.1
    y["qg"][2, 3, 7] = y["qg"][2, 5, 8] = 1.0
    y["v_new"][3, 1, 255] = 0.0
    ref = run(hip, y)
    clean = np.ones_like(bad)
    clean[0, 4:], clean[1, :4, 64:128], clean[2, 3], clean[2, 5], clean[3, 4:, 192:] = False, False, False, False, False
    # group 3 of the appended row is another row's: its other groups, and every other place, keep their bits
    assert np.array_equal(got["out"][clean], ref["out"][clean])


def test_bits_do_not_depend_on_the_batch(hip):
    """Twice the same call, and equal sequences in one batch, give the same bits."""
    x = make(8, 2, [700, 700, 3, 700], 901, 9)
    for c in ("qg", "k_new", "v_new", "k", "v", "k_scale", "v_scale"):
        x[c][3] = x[c][0]
    x["pos"][3] = x["pos"][0]
    a, b = run(hip, x), run(hip, x)
    assert np.array_equal(a["out"], b["out"]) and np.array_equal(a["out"][0], a["out"][3])


def test_offsets_beyond_32_bits(hip):
    """The last cache of a batch whose caches take more than 2^32 bytes each for K and V."""
    B, nkv, cap, n = 17, 2, 1 << 20, 70
    x = make(8, nkv, [n], n + 1, 10)
    big = {"len": np.full(B, -1, np.int32), "pos": np.zeros(B, np.int32), "out": np.zeros((B, 8, HD), np.float32),
           "q_norm": x["q_norm"], "k_norm": x["k_norm"], "rot": 64}
    big["len"][-1], big["pos"][-1] = n, x["pos"][0]
    for c in ("qg", "k_new", "v_new"):
        big[c] = np.zeros((B,) + x[c].shape[1:], np.float32)
        big[c][-1] = x[c][0]
    with upload(hip, big) as bufs:
        for c, row in (("k", 128), ("v", 128), ("k_scale", 16), ("v_scale", 16)):
            bufs.p[c] = hip.malloc(B * nkv * cap * row)
            for h in range(nkv):
                hip.copy_in(bufs.p[c] + ((B - 1) * nkv + h) * cap * row, x[c][0, h])
        pyq35.check(lib.q35_attn_q4(attn_q4_args(bufs, big, cap), None))
        hip.sync()
        got = {"out": bufs.get("out")[-1:]}
        for c, row in (("k", 128), ("v", 128), ("k_scale", 16), ("v_scale", 16)):
            got[c] = np.stack([hip.download(bufs.p[c] + ((B - 1) * nkv + h) * cap * row, x[c][0, h].shape, x[c].dtype) for h in range(nkv)])[None]
    check(x, got)


def test_graph_over_steps(hip):
    """One graph decodes step after step: lengths and positions move on the device's arrays."""
    B, cap = 3, 80
    x = make(8, 2, [0, 60, -1], cap, 11)
    with upload(hip, x) as bufs, upload(hip, x) as eager:
        a, e = attn_q4_args(bufs, x, cap), attn_q4_args(eager, x, cap)
        g = Graph(hip, lambda s: pyq35.check(lib.q35_attn_q4(a, s)))
        rng = np.random.default_rng(0)
        try:
            for step in range(6):
                for c in ("qg", "k_new", "v_new"):
                    v = rng.standard_normal(x[c].shape, dtype=np.float32)
                    bufs.set(c, v)
                    eager.set(c, v)
                n = np.array([step, 60 + step, -1 if step < 3 else step], np.int32)
                for d in (bufs, eager):
                    d.set("len", n)
                    d.set("pos", n + 5)
                g.replay()
                pyq35.check(lib.q35_attn_q4(e, None))
                hip.sync()
                for c in OUT:
                    assert np.array_equal(bufs.get(c).view(np.uint8), eager.get(c).view(np.uint8)), (step, c)
        finally:
            g.close()


def test_two_calls_at_once(hip):
    x = make(16, 2, [900, 44, 300], 901, 12)
    want = run(hip, x)
    with upload(hip, x) as p, upload(hip, x) as q:
        s = [C.c_void_p(), C.c_void_p()]
        for i in s:
            hip._ck(hip.rt.hipStreamCreate(C.byref(i)), "hipStreamCreate")
        a, b = attn_q4_args(p, x, 901), attn_q4_args(q, x, 901)
        for _ in range(4):
            pyq35.check(lib.q35_attn_q4(a, s[0]))
            pyq35.check(lib.q35_attn_q4(b, s[1]))
        hip.sync()
        assert np.array_equal(p.get("out"), want["out"]) and np.array_equal(q.get("out"), want["out"])
        for i in s:
            hip._ck(hip.rt.hipStreamDestroy(i), "hipStreamDestroy")
