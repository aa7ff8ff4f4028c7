"""A long prompt's cache cut to a budget: the prompt is prefilled straight into own caches of a batch, a few
tokens are decoded over them while weights accumulate, every head then keeps the rows of most weight, and
decoding goes on over those, against the same steps in float64 on the caches as they lie. Bars as in
test_gpu_attn_batch.py."""
import numpy as np
import pytest

import pyq35
from batch_ref import EPS, HD, THETA, Buffers, attn64, attn_args, cache_in, cache_out, evict_args, evict_rows
from helpers import REL_L2, rel_l2

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
def test_prompt_in_own_caches(bf16):
    hip = pyq35.Hip()
    rng = np.random.default_rng(51)
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
    NQ, NKV, CAP, KEEP, SINK, RECENT = 8, 2, 160, 64, 4, 16
    lens = [150, 101]
    B = len(lens)
    x = {"rot": 64, "q_norm": 0.1 * n(HD), "k_norm": 0.1 * n(HD)}
    # (rows that nothing wrote yet are NaN, and the weights of a prompt start at 0)
    cache = cache_in(np.full((B, NKV, CAP, HD), np.nan, np.float32), bf16)
    with Buffers(hip, k_own=cache, v_own=cache, own_score=np.zeros((B, NKV, CAP), np.float32),
                 own_pos=np.tile(np.arange(CAP, dtype=np.int32), (B, NKV, 1)), own_len=np.array(lens, np.int32),
                 pos=np.array(lens, np.int32), out=n(B, NQ, HD), q_norm=x["q_norm"], k_norm=x["k_norm"], qg=n(B, NQ, 2 * HD),
                 k_new=n(B, NKV, HD), v_new=n(B, NKV, HD)) as bufs:
        for b, m in enumerate(lens):
            ld = (2 * NQ + 2 * NKV) * HD
            at = b * NKV * CAP * HD * (2 if bf16 else 4)
            with Buffers(hip, qkv=n(m, ld), out=np.zeros((m, NQ * HD), np.float32)) as one:
                p = pyq35.AttnPrefillArgs(n_tokens=m, pos0=0, q_heads=NQ, kv_heads=NKV, head_dim=HD, rotary_dim=64,
                                          kv_dtype=int(bf16), max_context=CAP, rope_theta=THETA, eps=EPS, qkv=one.p["qkv"],
                                          ld_qkv=ld, q_norm=bufs.p["q_norm"], k_norm=bufs.p["k_norm"],
                                          k_cache=bufs.p["k_own"] + at, v_cache=bufs.p["v_own"] + at, out=one.p["out"])
                p.workspace_bytes = pyq35.lib.q35_attn_prefill_workspace_bytes(p)
                one.put("ws", np.zeros(p.workspace_bytes, np.uint8))
                p.workspace = one.p["ws"]
                pyq35.check(pyq35.lib.q35_attn_prefill(p, None))
                hip.sync()
        score = np.zeros((B, NKV, CAP))
        pos = np.array(lens)
        for step in range(8):
            for c in ("qg", "k_new", "v_new"):
                x[c] = n(*bufs.shape[c][0])
                bufs.set(c, x[c])
            x["pos"] = pos
            bufs.set("own_len", np.array(lens))
            bufs.set("pos", pos)
            pyq35.check(pyq35.lib.q35_attn_batch(attn_args(bufs, x, bf16, CAP, 0, 0), None))
            hip.sync()
            K, V, out = cache_out(bufs.get("k_own")), cache_out(bufs.get("v_own")), bufs.get("out")
            for b in range(B):
                m = lens[b] + 1
                ref, w = attn64(x, b, K[b, :, :m], V[b, :, :m])
                assert rel_l2(out[b], ref) < REL_L2, (step, b)
                score[b, :, :m] += w.reshape(NKV, NQ // NKV, m).sum(1)
                assert rel_l2(bufs.get("own_score")[b, :, :m], score[b, :, :m]) < REL_L2, (step, b)
            lens = [m + 1 for m in lens]
            pos = pos + 1
            if step != 4:
                continue
            bufs.set("own_len", np.array(lens))
            bufs.set("pos", pos)
            place = bufs.get("own_pos")
            e = evict_args(bufs, B, NKV, CAP, KEEP, SINK, RECENT, bf16, len="own_len", next_pos="pos", score="own_score",
                           pos="own_pos", k="k_own", v="v_own", score_out="own_score", pos_out="own_pos", new_len="own_len")
            pyq35.check(pyq35.lib.q35_kv_evict(e, None))
            hip.sync()
            for b in range(B):
                for h in range(NKV):
                    take = evict_rows(score[b, h], place[b, h], lens[b], KEEP, SINK, RECENT, pos[b])
                    assert np.array_equal(bufs.get("own_pos")[b, h, :KEEP], place[b, h][take])
                    assert np.array_equal(cache_out(bufs.get("k_own"))[b, h, :KEEP], K[b, h][take])
                    assert np.array_equal(cache_out(bufs.get("v_own"))[b, h, :KEEP], V[b, h][take])
                    score[b, h, :KEEP], score[b, h, KEEP:] = score[b, h][take], 0.0
            lens = bufs.get("own_len").tolist()
            assert lens == [KEEP] * B
