"""q35_attn_batch gives what q35_attn_decode gives for each of its sequences alone: the prompt's rows
followed by the sequence's own in one cache, the new token at the position behind them.

Tolerance: either is held to REL_L2 against the definition, so they differ by at most twice that;
fp32 key rows by twice 8 * 2^-24 of the row's largest entry. bf16 rows are the same bits where no entry
lies that close to the middle of two bf16 values, which the inputs are checked for."""
import numpy as np
import pytest

import pyq35
from batch_ref import EPS, HD, THETA, Buffers, attn_args, cache_in, cache_out, rms64, rope64
from helpers import REL_L2, bf16_bits, rel_l2
from test_gpu_attn_batch import make, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return pyq35.Hip()


# of (query heads, prefix): with these no bf16 rounding of a new key can go either way
SEEDS = {(16, 700): 41, (8, 0): 42, (8, 333): 41, (2, 50): 41, (4, 90): 59}


def new_keys(x, b):
    return rope64(rms64(x["k_new"][b], x["k_norm"]), x["pos"][b], x["rot"])


def safe_to_round(x):
    """No entry of a new key within 16 * 2^-24 of itself (a rotated one: of its pair's length) of the middle
    of two bf16 values."""
    h = x["rot"] // 2
    for b in range(len(x["pos"])):
        k = new_keys(x, b)
        size = np.abs(k)
        size[:, :h] = size[:, h:2 * h] = np.hypot(k[:, :h], k[:, h:2 * h])
        err = 16 * 2.0 ** -24 * size
        if not np.array_equal(bf16_bits((k - err).astype(np.float32)), bf16_bits((k + err).astype(np.float32))):
            return False
    return True


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("nq,nkv,P,lens", [(16, 2, 700, [0, 5, 63, 40]), (8, 2, 0, [0, 1, 200]), (8, 2, 333, [31, 32]),
                                           (2, 1, 50, [7, 0]), (4, 4, 90, [3, 64, 12])])
def test_each_sequence_alone(hip, nq, nkv, P, lens, bf16):
    cap = max(lens) + 1
    x = make(nq, nkv, P, lens, cap, SEEDS[nq, P], bf16=bf16)
    assert not bf16 or safe_to_round(x)
    with upload(hip, x, bf16) as bufs:
        a = attn_args(bufs, x, bf16, cap, P, P)
        pyq35.check(pyq35.lib.q35_attn_batch(a, None))
        hip.sync()
        out, ko, vo = bufs.get("out"), cache_out(bufs.get("k_own")), cache_out(bufs.get("v_own"))
    for b, n in enumerate(lens):
        whole = {c: np.concatenate([x[c + "_prefix"], x[c + "_own"][b]], 1) for c in "kv"}
        with Buffers(hip, qg=x["qg"][b], kn=x["k_new"][b], vn=x["v_new"][b], qw=x["q_norm"], kw=x["k_norm"],
                     k=cache_in(whole["k"], bf16), v=cache_in(whole["v"], bf16), out=np.zeros((nq, HD), np.float32)) as one:
            d = pyq35.AttnDecodeArgs(q_heads=nq, kv_heads=nkv, head_dim=HD, rotary_dim=x["rot"], pos=P + n, kv_dtype=int(bf16),
                                     max_context=P + cap, rope_theta=THETA, eps=EPS, qg=one.p["qg"], k_new=one.p["kn"],
                                     v_new=one.p["vn"], q_norm=one.p["qw"], k_norm=one.p["kw"], k_cache=one.p["k"],
                                     v_cache=one.p["v"], out=one.p["out"])
            d.workspace_bytes = pyq35.lib.q35_attn_decode_workspace_bytes(d)
            one.put("ws", np.zeros(d.workspace_bytes, np.uint8))
            d.workspace = one.p["ws"]
            pyq35.check(pyq35.lib.q35_attn_decode(d, None))
            hip.sync()
            ref, kr, vr = one.get("out"), cache_out(one.get("k")), cache_out(one.get("v"))
        assert np.array_equal(vo[b], vr[:, P:], equal_nan=True)
        k, was = ko[b, :, n], kr[:, P + n]
        if bf16:
            assert np.array_equal(k, was)
        else:
            assert (np.abs(k - was) <= 16 * 2.0 ** -24 * np.abs(was).max(-1, keepdims=True)).all()
        for h in range(nq):
            assert rel_l2(out[b, h], ref[h]) < 2 * REL_L2, f"sequence {b} head {h}"
