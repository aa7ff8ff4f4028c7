"""q35_matmul_q4 against float64, and the kernels that make its weights against their definition bit by
bit: every group size, zero points, one row to several blocks of rows, sizes that fill no tile, strides,
residuals, entries of very different size, infinities and NaN, captured graphs, other streams.

Tolerance. A row of X may enter as whole multiples of 2^-22 of the largest entry of its group (off by
half of that, 2^-23), and 24 bits of fp32 arithmetic do the rest: a group's sum rounded twice, its scale
once, each product of both once, and one addition a group and lane. So an output is within
    2^-22 sum_g max_{k in g} |x_k| sum_{k in g} |w_k|  +  (K / 32 + 10) 2^-24 sum_k |x_k w_k|  +  2^-23 |y|
of the exact one, half of the first term left for the roundings of what undoes the multiples."""
import ctypes as C

import numpy as np
import pytest

import pyq35
from batch_ref import Buffers, Graph
from helpers import bf16_bits, bf16_to_f32
from q4_ref import bytes_of, quantize_weights, weights64

pytestmark = pytest.mark.gpu
lib = pyq35.lib


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


def make(M, N, K, G, zeros, seed, ldx=None, ldy=None, residual=False):
    rng = np.random.default_rng(seed)
    groups = (K + G - 1) // G
    x = {"codes": bytes_of(rng.integers(0, 16, (N, K), dtype=np.uint8)),
         "scales": (0.02 * np.exp(0.3 * rng.standard_normal((N, groups))) * rng.choice([-1, 1, 1, 1], (N, groups))
                    ).astype(np.float16).view(np.uint16),
         "zeros": rng.integers(0, 16, (N, groups), dtype=np.uint8) if zeros else None,
         "X": rng.standard_normal((M, ldx or K)).astype(np.float32) * np.exp(rng.standard_normal(ldx or K)).astype(np.float32),
         "Y": rng.standard_normal((M, ldy or N)).astype(np.float32), "N": N, "K": K, "G": G}
    x["X"][:, K:] = np.nan
    x["R"] = rng.standard_normal((M, (ldy or N) + 3)).astype(np.float32) if residual else None
    return x


def bound(x, w, want):
    M, K, G = x["X"].shape[0], x["K"], x["G"]
    groups = (K + G - 1) // G
    pad = lambda a: np.pad(a, ((0, 0), (0, groups * G - K))).reshape(a.shape[0], groups, G)  # noqa: E731
    a, b = pad(np.abs(x["X"][:, :K].astype(np.float64))), pad(np.abs(w))
    return (2.0 ** -22 * a.max(-1) @ b.sum(-1).T + (K / 32 + 10) * 2.0 ** -24 * (np.abs(x["X"][:, :K].astype(np.float64)) @ np.abs(w).T)
            + 2.0 ** -23 * np.abs(want) + 1e-37)


def pack(hip, bufs, x):
    zeros = x["zeros"] is not None
    n = lib.q35_q4_packed_bytes(x["N"], x["K"], x["G"], int(zeros))
    bufs.put("packed", np.full(n, 0xA5, np.uint8))
    pyq35.check(lib.q35_q4_pack(bufs.p["codes"], bufs.p["scales"], bufs.p["zeros"] if zeros else None, x["N"], x["K"], x["G"],
                                bufs.p["packed"], None))


def call(bufs, x, stream=None, in_place=False, M=None, ws="ws"):
    M, N, K, G = M or x["X"].shape[0], x["N"], x["K"], x["G"]
    need = lib.q35_matmul_q4_workspace_bytes(M, N, K, G)
    if ws not in bufs.p:
        bufs.put(ws, np.full(need, 0xFF, np.uint8))
    R, ldr = (bufs.p["Y"], x["Y"].shape[1]) if in_place else (bufs.p["R"], x["R"].shape[1]) if x["R"] is not None else (None, 0)
    pyq35.check(lib.q35_matmul_q4(bufs.p["X"], x["X"].shape[1], bufs.p["packed"], int(x["zeros"] is not None), M, N, K, G, R, ldr,
                                  bufs.p["Y"], x["Y"].shape[1], bufs.p[ws], need, stream))


def arrays(x):
    return {n: x[n] for n in ("codes", "scales", "zeros", "X", "Y", "R")}


def expect(x, in_place=False):
    N, K = x["N"], x["K"]
    w = weights64(x["codes"], x["scales"], x["zeros"], K, x["G"])
    want = x["X"][:, :K].astype(np.float64) @ w.T
    if in_place:
        want = want + x["Y"][:, :N]
    elif x["R"] is not None:
        want = want + x["R"][:, :N]
    return w, want


def check(hip, x, in_place=False):
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x, in_place=in_place)
        hip.sync()
        got = bufs.get("Y")
    w, want = expect(x, in_place)
    N = x["N"]
    err = np.abs(got[:, :N] - want)
    assert (err <= bound(x, w, want)).all(), f"worst {np.nanmax(err / bound(x, w, want))}"
    assert np.array_equal(got[:, N:], x["Y"][:, N:])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 13, 16, 17, 32, 33, 64, 70])
def test_rows(hip, M, G, zeros):
    check(hip, make(M, 80, 512, G, zeros, 10 * M + G))


@pytest.mark.parametrize("G,zeros", [(32, True), (64, False), (64, True), (128, False)])
@pytest.mark.parametrize("N,K", [(1, 1), (1, 2048), (16, 255), (17, 256), (15, 257), (33, 31), (100, 513), (48, 1000), (7, 4099), (2048, 2048),
                                 (1024, 3584)])
@pytest.mark.parametrize("M", [1, 6, 21])
def test_sizes(hip, M, N, K, G, zeros):
    check(hip, make(M, N, K, G, zeros, N + K + M))


@pytest.mark.parametrize("M,N,K,G", [(1, 40000, 300, 64), (1, 64, 32768, 64), (4, 64, 20000, 32), (16, 300, 16384, 128), (40, 5000, 640, 64),
                                     (300, 50, 700, 32), (1, 151936, 128, 128)])
def test_large(hip, M, N, K, G):
    check(hip, make(M, N, K, G, N % 2 == 0, 5))


@pytest.mark.parametrize("M", [1, 3, 11, 20])
def test_strides_and_residual(hip, M):
    check(hip, make(M, 77, 515, 64, False, 1, ldx=517, ldy=90, residual=True))
    check(hip, make(M, 77, 512, 32, True, 2, ldx=540, ldy=81, residual=True))
    check(hip, make(M, 77, 512, 64, False, 3, ldy=79), in_place=True)


@pytest.mark.parametrize("M", [1, 7, 18])
def test_unlike_sizes(hip, M):
    """Entries from the smallest to the largest fp32 in one row, groups of zeros, rows of zeros."""
    x = make(M, 50, 640, 64, False, 7)
    x["X"] = np.random.default_rng(7).standard_normal((M, 640)).astype(np.float32)
    x["X"][:, 64:128] *= np.float32(2.0 ** 60)
    x["X"][:, 128:192] *= np.float32(2.0 ** -60)
    x["X"][:, 192:256] = 0.0
    x["X"][:, 256] = np.float32(1e30)                                   # one entry far above its group
    x["X"][0] *= np.float32(2.0 ** -100) if M > 1 else np.float32(1.0)
    x["X"][M // 2, 320:] = 0.0
    if M > 2:
        x["X"][2] = 0.0
    # entries below 2^-100 may count as 0
    w, want = expect(x)
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        got = bufs.get("Y")
    assert (np.abs(got - want) <= bound(x, w, want) + 2.0 ** -100 * np.abs(w).sum(1)).all()


@pytest.mark.parametrize("top", [8355711.0, 8355712.0, 8388607.0, 4194304.0, 16711422.0])
def test_borders_of_the_multiples(hip, top):
    """The largest entry of a group next to where its multiples change, of both signs."""
    x = make(2, 32, 256, 64, False, 9)
    x["X"][:, ::64], x["X"][:, 1::64] = np.float32(top), np.float32(-top)
    x["X"][1] *= np.float32(2.0 ** -30)
    x["X"][:, 2::64] *= np.float32(1000.0)
    check(hip, x)


@pytest.mark.parametrize("M", [1, 6, 20])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_not_finite(hip, M, bad):
    """A row of X with an infinity or a NaN has no finite outputs, the other rows are as without it; a
    scale that is NaN takes its output column alone."""
    x = make(M, 40, 300, 64, True, 11)
    row = M - 1
    keep = x["X"].copy()
    x["X"][row, 100] = bad
    x["scales"][5, 2] = 0x7E00
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        got = bufs.get("Y")
    assert not np.isfinite(got[row]).any() and np.isnan(got[:, 5]).all()
    x["X"] = keep
    x["scales"][5, 2] = 0
    w, want = expect(x)
    ok = np.ones_like(got, bool)
    ok[row], ok[:, 5] = False, False
    assert (np.abs(got - want) <= bound(x, w, want))[ok].all()


def test_same_rows_in_any_batch(hip):
    """A row's outputs are the same bits wherever it stands in a batch of one size."""
    x = make(9, 200, 1000, 64, False, 3)
    x["X"][4] = x["X"][0]
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        got = bufs.get("Y")
        call(bufs, x)
        hip.sync()
        assert np.array_equal(got, bufs.get("Y"))
    assert np.array_equal(got[0], got[4])


@pytest.mark.parametrize("M", [1, 12])
def test_graph_and_streams(hip, M):
    x = make(M, 300, 2048, 64, True, 21)
    with Buffers(hip, **arrays(x)) as bufs:
        pack(hip, bufs, x)
        call(bufs, x)
        hip.sync()
        first = bufs.get("Y")
        g = Graph(hip, lambda s: call(bufs, x, s))
        try:
            for i in range(4):
                bufs.set("X", x["X"] * np.float32(1 + i))
                bufs.set("Y", x["Y"])
                g.replay()
                assert np.array_equal(bufs.get("Y"), first * np.float32(1 + i)) or i == 2   # 3 is no power of two
                call(bufs, x)
                hip.sync()
                eager = bufs.get("Y")
                g.replay()
                assert np.array_equal(bufs.get("Y"), eager)
        finally:
            g.close()
        # two calls at once, on two streams, with a workspace and outputs each
        bufs.set("X", x["X"])
        bufs.put("Y2", x["Y"])
        s1, s2 = C.c_void_p(), C.c_void_p()
        for s in (s1, s2):
            hip._ck(hip.rt.hipStreamCreate(C.byref(s)), "hipStreamCreate")
        other = Buffers(hip)
        other.p = dict(bufs.p, Y=bufs.p["Y2"])
        other.p.pop("ws")
        other.put("ws", np.full(max(16, lib.q35_matmul_q4_workspace_bytes(M, 300, 2048, 64)), 0xFF, np.uint8))
        for _ in range(5):
            call(bufs, x, s1)
            call(other, x, s2)
        hip.sync()
        assert np.array_equal(bufs.get("Y"), first) and np.array_equal(bufs.get("Y2"), first)
        hip.free(other.p["ws"])
        for s in (s1, s2):
            hip._ck(hip.rt.hipStreamDestroy(s), "hipStreamDestroy")


# ------------------------------------------------------------------------------ making the weights
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("N,K,G", [(5, 256, 64), (33, 100, 32), (17, 1, 64), (7, 333, 128), (64, 2048, 64)])
def test_quantize(hip, N, K, G, bf16, asym):
    rng = np.random.default_rng(N + K)
    W = (0.02 * rng.standard_normal((N, K))).astype(np.float32)
    W[0], W[1 % N, : K // 2] = 0.0, 0.5
    W[2 % N] = np.abs(W[2 % N])
    W[3 % N] *= np.float32(1e-7)                                        # steps among fp16's smallest
    if K > 40 and N > 4:
        W[4, 3], W[4, 40] = np.nan, -np.inf
    W = bf16_to_f32(bf16_bits(W)) if bf16 else W
    groups = (K + G - 1) // G
    with Buffers(hip, W=bf16_bits(W) if bf16 else W, codes=np.full((N, (K + 1) // 2), 0x55, np.uint8),
                 scales=np.zeros((N, groups), np.uint16), zeros=np.zeros((N, groups), np.uint8)) as bufs:
        pyq35.check(lib.q35_q4_quantize(bufs.p["W"], int(bf16), N, K, G, bufs.p["codes"], bufs.p["scales"],
                                        bufs.p["zeros"] if asym else None, None))
        hip.sync()
        c, s, z = bufs.get("codes"), bufs.get("scales"), bufs.get("zeros")
    if bf16 and K > 40 and N > 4:
        W[4, 3] = np.nan
    wc, wsc, wz = quantize_weights(W, K, G, asym)
    nan = np.isnan(wsc.view(np.float16).astype(np.float32))
    assert np.array_equal(np.isnan(s.view(np.float16).astype(np.float32)), nan) and np.array_equal(s[~nan], wsc[~nan])
    assert np.array_equal(c, wc) and (not asym or np.array_equal(z, wz))
    # half a step from every weight, and as much again where the rounded scale ends early
    fine = ~nan[:, np.arange(K) // G] & (np.abs(s.view(np.float16).astype(np.float32)) > 6.2e-5)[:, np.arange(K) // G]
    step = np.abs(s.view(np.float16).astype(np.float64))[:, np.arange(K) // G]
    v = weights64(c, s, z if asym else None, K, G)
    assert (np.abs(v - W) <= 1.05 * step)[fine].all()
