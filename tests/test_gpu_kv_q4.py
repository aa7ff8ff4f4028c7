"""q35_kv_q4_store and q35_kv_q4_load against their definition: whole numbers and fp16 values, every bit
has to agree (any NaN for another); loaded values within half a step of their type. Ranges of rows of
every kind, shared prompts, values that fp16 does not hold, infinities and NaN."""
import numpy as np
import pytest

import pyq35
from batch_ref import HD, Buffers, Graph, cache_in, cache_out
from q4_ref import kv_q4_args, row_codes, row_values, same_rows

pytestmark = pytest.mark.gpu
lib = pyq35.lib


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def make(B, NKV, rows_cap, cap, begin, end, seed, bf16=False, shared=False):
    rng = np.random.default_rng(seed)
    x = {"begin": None if begin is None else np.array(begin, np.int32), "end": np.array(end, np.int32)}
    for c in ("k", "v"):
        r = rng.standard_normal((1 if shared else B, NKV, rows_cap, HD)).astype(np.float32) * np.exp(rng.standard_normal(HD)).astype(np.float32)
        x[c + "_rows"] = cache_out(cache_in(r, bf16))
        x[c] = rng.integers(0, 256, (B, NKV, cap, 128), dtype=np.uint8)
        x[c + "_scale"] = rng.standard_normal((B, NKV, cap, 4, 2)).astype(np.float16)
    return x


def ranges(x, rows_cap, cap):
    for b, e in enumerate(x["end"]):
        i = 0 if x["begin"] is None else int(x["begin"][b])
        if 0 <= i < e <= min(rows_cap, cap):
            yield b, i, int(e)


def run(hip, x, B, NKV, rows_cap, cap, bf16, shared, store):
    with Buffers(hip, **{n: cache_in(a, bf16) if n.endswith("_rows") else a for n, a in x.items()}) as bufs:
        a = kv_q4_args(bufs, B, NKV, rows_cap, cap, bf16, shared, x["begin"] is not None)
        pyq35.check((lib.q35_kv_q4_store if store else lib.q35_kv_q4_load)(a, None))
        hip.sync()
        return {n: cache_out(bufs.get(n)) if n.endswith("_rows") else bufs.get(n) for n in x if n not in ("begin", "end")}


def check_store(hip, x, rows_cap, cap, bf16=False, shared=False):
    B, NKV = x["k"].shape[:2]
    got = run(hip, x, B, NKV, rows_cap, cap, bf16, shared, True)
    for c in ("k", "v"):
        want, scale = x[c].copy(), x[c + "_scale"].copy()
        for b, i, e in ranges(x, rows_cap, cap):
            want[b, :, i:e], scale[b, :, i:e] = row_codes(x[c + "_rows"][0 if shared else b, :, i:e])
        assert np.array_equal(got[c], want) and same_rows(got[c + "_scale"], scale)
        assert np.array_equal(got[c + "_rows"], x[c + "_rows"], equal_nan=True)


def check_load(hip, x, rows_cap, cap, bf16=False):
    B, NKV = x["k"].shape[:2]
    got = run(hip, x, B, NKV, rows_cap, cap, bf16, False, False)
    for c in ("k", "v"):
        want, new = x[c + "_rows"].astype(np.float64), np.zeros(x[c + "_rows"].shape, bool)
        for b, i, e in ranges(x, rows_cap, cap):
            want[b, :, i:e], new[b, :, i:e] = row_values(x[c][b, :, i:e], x[c + "_scale"][b, :, i:e]), True
        assert np.array_equal(got[c + "_rows"][~new], x[c + "_rows"][~new])
        # a value is one fp32 rounding, bf16 another half step
        err = np.abs(got[c + "_rows"] - want)[new]
        assert (err <= np.abs(want[new]) * (2.0 ** -24 + (2.0 ** -8 if bf16 else 0)) * 1.01).all()
        assert np.array_equal(got[c], x[c]) and same_rows(got[c + "_scale"], x[c + "_scale"])


CASES = [(1, 2, 64, 64, None, [64]), (1, 1, 1, 1, None, [1]), (3, 2, 40, 50, [0, 7, 39], [40, 33, 40]),
         (5, 3, 70, 60, [0, -1, 5, 60, 0], [60, 10, 5, 61, 61]), (4, 1, 1000, 1300, None, [1000, 0, -1, 1001]), (2, 2, 5000, 5000, [0, 4000], [5000, 4999])]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,NKV,rows_cap,cap,begin,end", CASES)
def test_store(hip, B, NKV, rows_cap, cap, begin, end, bf16):
    check_store(hip, make(B, NKV, rows_cap, cap, begin, end, B + cap, bf16), rows_cap, cap, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,NKV,rows_cap,cap,begin,end", CASES)
def test_load(hip, B, NKV, rows_cap, cap, begin, end, bf16):
    check_load(hip, make(B, NKV, rows_cap, cap, begin, end, B + cap, bf16), rows_cap, cap, bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_shared_prompt(hip, bf16):
    check_store(hip, make(7, 2, 90, 128, [0, 0, 0, 3, 0, 89, 0], [90, 90, 0, 50, 1, 90, 91], 3, bf16, True), 90, 128, bf16, True)


@pytest.mark.parametrize("bf16", [False, True])
def test_values_of_every_kind(hip, bf16):
    x = make(1, 1, 16, 16, None, [16], 5, bf16)
    r = x["k_rows"][0, 0]
    r[0], r[1], r[2] = 0.0, 1.5, -3.0                              # no span
    r[3, 5], r[3, 70], r[3, 200] = np.nan, np.inf, -np.inf
    r[4, :64], r[4, 64:128], r[4, 128:192] = 70000.0, np.linspace(-70000, 0, 64), np.linspace(0, 1.2e6, 64)   # beyond fp16
    r[5] = np.linspace(-65504, 65504, 256)
    r[6] = 3.0e38
    r[7] = np.where(np.arange(256) % 2, 3.0e38, -3.0e38)
    r[8] *= np.float32(1e-6)                                         # steps among fp16's smallest, or none
    r[9] *= np.float32(1e-30)
    r[10] = np.float32(1000.0) + r[10]                               # least values far from the span
    r[11] = np.arange(256) % 16                                      # exactly the codes
    r[12] = (np.arange(256) % 31) * 0.5                              # halfway between two codes
    r[13, 1:] = 0.0
    x["k_rows"] = cache_out(cache_in(x["k_rows"], bf16))
    if bf16:
        x["k_rows"][0, 0, 3, 5] = np.nan
    check_store(hip, x, 16, 16, bf16)


def test_there_and_back(hip):
    """Half a step of each group, and the rounding of its step and least value."""
    x = make(2, 2, 300, 300, None, [300, 120], 8)
    got = run(hip, x, 2, 2, 300, 300, False, False, True)
    y = dict(x, **{c: got[c] for c in ("k", "v", "k_scale", "v_scale")}, k_rows=np.zeros_like(x["k_rows"]), v_rows=np.zeros_like(x["v_rows"]))
    back = run(hip, y, 2, 2, 300, 300, False, False, False)
    for c in ("k_rows", "v_rows"):
        for b, e in enumerate((300, 120)):
            a, z = x[c][b, :, :e].reshape(2, e, 4, 64).astype(np.float64), back[c][b, :, :e].reshape(2, e, 4, 64)
            span, size = a.max(-1) - a.min(-1), np.abs(a).max(-1)
            # half a step; codes that end early or late by the roundings of least (2^-11) and 15 steps (2^-11)
            assert (np.abs(a - z).max(-1) <= span / 30 * 1.001 + 2.0 ** -11 * (2 * size + span)).all()
        assert not back[c][1, :, 120:].any()


def test_graph(hip):
    """Ranges are read when the graph is replayed."""
    x = make(3, 2, 60, 60, [0, 0, 0], [10, 20, 30], 9)
    with Buffers(hip, **x) as bufs:
        a = kv_q4_args(bufs, 3, 2, 60, 60, False)
        g = Graph(hip, lambda s: pyq35.check(lib.q35_kv_q4_store(a, s)))
        try:
            for end in ([10, 20, 30], [60, -1, 0], [0, 60, 61]):
                for c in ("k", "v", "k_scale", "v_scale"):
                    bufs.set(c, x[c])
                bufs.set("end", end)
                g.replay()
                for c in ("k", "v"):
                    want = x[c].copy()
                    for b, i, e in ranges(dict(x, end=end), 60, 60):
                        want[b, :, i:e] = row_codes(x[c + "_rows"][b, :, i:e])[0]
                    assert np.array_equal(bufs.get(c), want)
        finally:
            g.close()
