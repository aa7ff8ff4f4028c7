"""The operators of a decode step held in 4 bits together, as a program uses them: weights quantized and packed once, a
prompt's rows stored into every sequence's cache, then steps of one captured graph (queries, keys and values from 4-bit
weights, attention over the 4-bit caches, the output product onto the residual, the head, the draw), replayed with
new inputs between eager work; at the end the caches are read back.

Each operator is held to its own tolerance on what it was given: what it is given is the one before's output."""
import numpy as np
import pytest

import pyq35
from batch_ref import HD, Buffers, Graph
from helpers import bf16_bits, bf16_to_f32
from q4_ref import attn_q4_args, kv_q4_args, quantize_weights, row_codes, row_values, same_rows, sample64, sample_args, weights64
from test_gpu_attn_q4 import check as check_attention
from test_gpu_matmul_q4 import bound

pytestmark = pytest.mark.gpu
lib = pyq35.lib


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


class Weights:
    def __init__(self, bufs, name, N, K, G, asym, rng, M):
        self.bufs, self.name, self.N, self.K, self.G, self.asym = bufs, name, N, K, G, asym
        W = bf16_bits(rng.standard_normal((N, K), dtype=np.float32) / np.sqrt(K))
        groups = (K + G - 1) // G
        for n, a in (("w", W), ("c", np.zeros((N, (K + 1) // 2), np.uint8)), ("s", np.zeros((N, groups), np.uint16)),
                     ("z", np.zeros((N, groups), np.uint8)), ("p", np.zeros(lib.q35_q4_packed_bytes(N, K, G, int(asym)), np.uint8))):
            bufs.put(name + n, a)
        bufs.put(name + "ws", np.full(lib.q35_matmul_q4_workspace_bytes(M, N, K, G), 0xFF, np.uint8))
        p = lambda n: bufs.p[name + n]  # noqa: E731
        z = p("z") if asym else None
        pyq35.check(lib.q35_q4_quantize(p("w"), 1, N, K, G, p("c"), p("s"), z, None))
        pyq35.check(lib.q35_q4_pack(p("c"), p("s"), z, N, K, G, p("p"), None))
        bufs.hip.sync()
        c, s, z = bufs.get(name + "c"), bufs.get(name + "s"), bufs.get(name + "z")
        want = quantize_weights(bf16_to_f32(W), K, G, asym)
        assert np.array_equal(c, want[0]) and np.array_equal(s, want[1]) and (not asym or np.array_equal(z, want[2]))
        self.w = weights64(c, s, z if asym else None, K, G)

    def multiply(self, X, Y, M, stream, R=None):
        b = self.bufs
        need = lib.q35_matmul_q4_workspace_bytes(M, self.N, self.K, self.G)
        pyq35.check(lib.q35_matmul_q4(b.p[X], self.K, b.p[self.name + "p"], int(self.asym), M, self.N, self.K, self.G,
                                      b.p[R] if R else None, self.N, b.p[Y], self.N, b.p[self.name + "ws"], need, stream))

    def check(self, X, Y, R=None):
        x = {"X": X, "K": self.K, "G": self.G}
        want = X.astype(np.float64) @ self.w.T + (0 if R is None else R)
        assert (np.abs(Y - want) <= bound(x, self.w, want)).all(), f"{self.name}: {np.abs(Y - want).max()}"


@pytest.mark.parametrize("B,nq,nkv,prompt,steps", [(1, 8, 2, 37, 5), (5, 8, 2, 300, 4), (13, 4, 1, 0, 4)])
def test_steps(hip, B, nq, nkv, prompt, steps):
    rng = np.random.default_rng(B)
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
    H, V, cap, idle = 320, 3001, prompt + 9, B > 1
    lens = np.full(B, prompt, np.int32)
    if idle:
        lens[B // 2] = -1
    rows = {c: bf16_bits(n(nkv, max(prompt, 1), HD)) for c in ("k", "v")}
    embed = n(V, H)
    x = {"qg": n(B, nq, 2 * HD), "k_new": n(B, nkv, HD), "v_new": n(B, nkv, HD), "q_norm": 0.1 * n(HD), "k_norm": 0.1 * n(HD), "rot": 64,
         "len": lens, "pos": np.maximum(lens, 0), "out": n(B, nq, HD)}
    temperature = np.where(lens < 0, -1.0, rng.choice([0.0, 0.8, 1.3], B)).astype(np.float32)
    with Buffers(hip, X=embed[:B], Y=n(B, H), logits=n(B, V), temperature=temperature, top_k=np.full(B, 50, np.int32),
                 top_p=np.full(B, 0.9, np.float32), min_p=np.zeros(B, np.float32), u=rng.random(B, dtype=np.float32),
                 token=np.full(B, -7, np.int32), prob=np.full(B, -7, np.float32), end=np.maximum(lens, 0).astype(np.int32),
                 k_rows=rows["k"], v_rows=rows["v"], **{c: a for c, a in x.items() if c != "rot"}) as bufs:
        for c in ("k", "v"):
            bufs.put(c, rng.integers(0, 256, (B, nkv, cap, 128), dtype=np.uint8))
            bufs.put(c + "_scale", np.full((B, nkv, cap, 4, 2), np.nan, np.float16))
        wq, wk, wv = (Weights(bufs, name, r, H, G, z, rng, B) for name, r, G, z in
                      (("wq", nq * 2 * HD, 64, False), ("wk", nkv * HD, 32, True), ("wv", nkv * HD, 32, False)))
        wo, head = Weights(bufs, "wo", H, nq * HD, 128, True, rng, B), Weights(bufs, "head", V, H, 64, False, rng, B)

        # the prompt's rows, the same for all
        pyq35.check(lib.q35_kv_q4_store(kv_q4_args(bufs, B, nkv, max(prompt, 1), cap, True, shared=True, begin=False), None))
        hip.sync()
        for c in ("k", "v"):
            codes, scale = row_codes(bf16_to_f32(rows[c])[:, :prompt])
            got, sc = bufs.get(c), bufs.get(c + "_scale")
            for b in range(B):
                there = prompt if lens[b] >= 0 else 0
                assert np.array_equal(got[b, :, :there], codes[:, :there]) and same_rows(sc[b, :, :there], scale[:, :there])
                assert np.isnan(sc[b, :, there:].astype(np.float32)).all()

        attend, draw = attn_q4_args(bufs, dict(x), cap, ws="attn_ws"), sample_args(bufs, B, V, V, ws="sample_ws")

        def step(stream):
            wq.multiply("X", "qg", B, stream)
            wk.multiply("X", "k_new", B, stream)
            wv.multiply("X", "v_new", B, stream)
            pyq35.check(lib.q35_attn_q4(attend, stream))
            wo.multiply("out", "Y", B, stream, R="X")
            head.multiply("Y", "logits", B, stream)
            pyq35.check(lib.q35_sample(draw, stream))

        graph = Graph(hip, step)
        try:
            for i in range(steps):
                before = {c: bufs.get(c) for c in ("k", "v", "k_scale", "v_scale", "out", "token", "len", "pos")}
                graph.replay()
                got = {c: bufs.get(c) for c in ("X", "qg", "k_new", "v_new", "out", "k", "v", "k_scale", "v_scale", "Y", "logits", "token",
                                               "prob", "u", "temperature")}
                wq.check(got["X"], got["qg"].reshape(B, -1))
                wk.check(got["X"], got["k_new"].reshape(B, -1))
                wv.check(got["X"], got["v_new"].reshape(B, -1))
                check_attention({**x, **before, "qg": got["qg"], "k_new": got["k_new"], "v_new": got["v_new"]}, got)
                wo.check(got["out"].reshape(B, -1), got["Y"], got["X"])
                head.check(got["Y"], got["logits"])
                for b in range(B):
                    if lens[b] < 0:
                        assert got["token"][b] == -7 and got["prob"][b] == -7
                        continue
                    want, p, room = sample64(got["logits"][b], got["temperature"][b], 50, np.float32(0.9), np.float32(0), got["u"][b])
                    if room > V * 2.0 ** -49:  # nearer to a border than the weights' roundings: either
                        assert got["token"][b] == want and abs(got["prob"][b] - p) <= p * 2.0 ** -22
                # the same eagerly, on the state of before: the same bits
                for c in ("k", "v", "k_scale", "v_scale"):
                    bufs.set(c, before[c])
                step(None)
                hip.sync()
                for c in ("out", "k", "v", "logits", "token", "prob"):
                    assert np.array_equal(bufs.get(c), got[c]), f"step {i}: {c}"
                on = lens >= 0
                lens[on] += 1
                bufs.set("len", lens)
                bufs.set("pos", np.maximum(lens, 0))
                bufs.set("X", embed[np.maximum(got["token"], 0)])
                bufs.set("u", rng.random(B, dtype=np.float32))
        finally:
            graph.close()

        # read back
        ends = np.where(lens >= 0, prompt + steps, 0).astype(np.int32)
        bufs.set("end", ends)
        for c in ("k_rows", "v_rows"):
            bufs.put(c, np.full((B, nkv, cap, HD), -3.0, np.float32))
        pyq35.check(lib.q35_kv_q4_load(kv_q4_args(bufs, B, nkv, cap, cap, False, begin=False), None))
        hip.sync()
        for c in ("k", "v"):
            got, want = bufs.get(c + "_rows"), row_values(bufs.get(c), bufs.get(c + "_scale")).astype(np.float32)
            for b in range(B):
                assert np.array_equal(got[b, :, :ends[b]], want[b, :, :ends[b]]) and (got[b, :, ends[b]:] == -3.0).all()
