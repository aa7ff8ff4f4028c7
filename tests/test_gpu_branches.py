"""The operators for a batch of continuations as they are used together: answers forked from one
prompt's GDN state and attention cache, decoded step by step with their own caches cut back to a
budget by accumulated weight, against the same steps in float64."""
import numpy as np
import pytest

import pyq35
from batch_ref import (D, HD, Buffers, attn64, attn_args, cache_in, cache_out, evict_args, evict_rows, gdn64, gdn_args)
from helpers import REL_L2, bf16_bits, bf16_to_f32, rel_l2

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
def test_answers_of_one_prompt(bf16):
    hip = pyq35.Hip()
    rng = np.random.default_rng(11)
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
    rnd = (lambda v: bf16_to_f32(bf16_bits(v))) if bf16 else (lambda v: v)
    B, NQ, NKV, P, CAP, KEEP, SINK, RECENT, STEPS = 5, 8, 2, 150, 24, 16, 1, 4, 40
    KH, VH = 2, 4
    CONV, VD = (2 * KH + VH) * D, VH * D
    x = {"KH": KH, "VH": VH, "rot": 64, "q_norm": 0.1 * n(HD), "k_norm": 0.1 * n(HD), "conv_w": 0.5 * n(CONV, 4),
         "A_log": n(VH), "dt_bias": n(VH), "norm_w": 1 + 0.1 * n(D), "k_prefix": rnd(n(NKV, P, HD)),
         "v_prefix": rnd(n(NKV, P, HD)), "qg": n(B, NQ, 2 * HD), "k_new": n(B, NKV, HD), "v_new": n(B, NKV, HD),
         "qkv": n(B, CONV), "z": n(B, VD), "b": n(B, VH), "a": n(B, VH), "ring_in": n(4, CONV), "state_in": 0.1 * n(VH, D, D)}
    dev = {k: cache_in(v, bf16) if k in ("k_prefix", "v_prefix") else v for k, v in x.items() if k not in ("KH", "VH", "rot")}
    cache = np.zeros((B, NKV, CAP, HD), np.uint16 if bf16 else np.float32)
    dev.update(k_own=cache, v_own=cache, own_score=np.zeros((B, NKV, CAP), np.float32), out=np.zeros((B, NQ, HD), np.float32),
               own_pos=np.zeros((B, NKV, CAP), np.int32), own_len=np.zeros(B, np.int32), pos=np.full(B, P, np.int32),
               ring=np.zeros((B, 4, CONV), np.float32), state=np.zeros((B, VH, D, D), np.float32))
    lens, pos = np.zeros(B, np.int64), np.full(B, P)
    rings, states = [x["ring_in"]] * B, [x["state_in"]] * B
    K = np.zeros((B, NKV, CAP, HD), np.float32)
    V, SC, PO = K.copy(), np.zeros((B, NKV, CAP)), np.zeros((B, NKV, CAP), np.int64)
    with Buffers(hip, **dev) as bufs:
        bufs.put("mix", np.zeros((B, VD), np.float32))
        for step in range(STEPS):
            # sequence 3 ends half way: its place stays empty
            alive = [b for b in range(B) if not (b == 3 and step >= STEPS // 2)]
            for c in ("qg", "k_new", "v_new", "qkv", "z", "b", "a"):
                x[c] = n(*x[c].shape)
                bufs.set(c, x[c])
            place = np.array([lens[b] if b in alive else -1 for b in range(B)], np.int32)
            x["pos"] = np.array([pos[b] if b in alive else -1 for b in range(B)], np.int32)
            bufs.set("own_len", place)
            bufs.set("pos", x["pos"])
            g = gdn_args(bufs, x, B, B, fork=step == 0)
            g.out = bufs.p["mix"]
            pyq35.check(pyq35.lib.q35_gdn_batch(g, None))
            a = attn_args(bufs, x, bf16, CAP, P, P)
            pyq35.check(pyq35.lib.q35_attn_batch(a, None))
            hip.sync()
            mix, out, ko = bufs.get("mix"), bufs.get("out"), cache_out(bufs.get("k_own"))
            for b in alive:
                ref, rings[b], states[b] = gdn64(x, b, b, 1, int(pos[b]), rings[b], states[b])
                assert rel_l2(mix[b], ref[0]) < REL_L2, (step, b)
                at = int(lens[b])
                K[b, :, at], V[b, :, at], PO[b, :, at] = ko[b, :, at], rnd(x["v_new"][b]), pos[b]
                ref, w = attn64(x, b, np.concatenate([x["k_prefix"], K[b, :, :at + 1]], 1),
                                np.concatenate([x["v_prefix"], V[b, :, :at + 1]], 1))
                assert rel_l2(out[b], ref) < REL_L2, (step, b)
                w = w[:, P:].reshape(NKV, NQ // NKV, -1).sum(1)
                SC[b, :, at] = 0.0
                SC[b, :, :at + 1] += w
                lens[b] += 1
                pos[b] += 1
            if max(lens) < CAP and step % 7:
                continue
            # every head cuts its own cache; the chosen rows agree with the sums in 64 bits
            bufs.set("own_len", np.array([lens[b] if b in alive else -1 for b in range(B)], np.int32))
            bufs.set("pos", np.array(pos, np.int32))
            e = evict_args(bufs, B, NKV, CAP, KEEP, SINK, RECENT, bf16, len="own_len", next_pos="pos", score="own_score",
                           pos="own_pos", k="k_own", v="v_own", score_out="own_score", pos_out="own_pos", new_len="own_len")
            pyq35.check(pyq35.lib.q35_kv_evict(e, None))
            hip.sync()
            new, ko, vo, so, po = (bufs.get(c) for c in ("own_len", "k_own", "v_own", "own_score", "own_pos"))
            for b in alive:
                for h in range(NKV):
                    take = evict_rows(SC[b, h], PO[b, h], int(lens[b]), KEEP, SINK, RECENT, pos[b])
                    m = len(take)
                    for c in (K, V, SC, PO):
                        c[b, h, :m] = c[b, h][take]
                    assert np.array_equal(po[b, h, :m], PO[b, h, :m]), (step, b, h)
                    assert np.array_equal(cache_out(ko)[b, h, :m], K[b, h, :m])
                    assert np.array_equal(cache_out(vo)[b, h, :m], V[b, h, :m])
                    assert rel_l2(so[b, h, :m], SC[b, h, :m]) < REL_L2
                lens[b] = min(int(lens[b]), KEEP)
                assert new[b] == lens[b]
        for b in range(B):
            assert rel_l2(bufs.get("state")[b], states[b]) < REL_L2
