"""How the batched attention is cut (csrc/plans.hpp, built with g++): CPU only. Pieces cover the prefix
and every own cache in whole tiles, none is empty, and their number stays within what the merge
holds in LDS and the grid in 31 bits, for any sizes and number of compute units."""
import ctypes as C
import os
import random
import subprocess

import pytest

import pyq35

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("plans") / "batch_plan.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "qwen3.5-cpu-cpp_amd", "csrc"), "-o", so,
                    os.path.join(ROOT, "tests", "cpp", "batch_plan.cpp")], check=True)
    return C.CDLL(so)


def plan(lib, B, grp, nkv, P, cap, bf16, cu=256):
    out = (C.c_int * 6)()
    lib.attn_batch_plan_c(B, grp, nkv, C.c_int64(P), C.c_int64(cap), int(bf16), cu, out)
    return list(out)


def test_pieces_cover_the_keys(lib):
    rng = random.Random(3)
    for _ in range(20000):
        B, grp, nkv = int(2 ** rng.uniform(0, 12)), rng.randint(1, 16), rng.choice([1, 2, 3, 4, 8])
        P = rng.choice([0, int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(20, 30))])
        cap, bf16 = int(2 ** rng.uniform(0, rng.choice([12, 30]))), rng.random() < 0.5
        cu = rng.choice([1, 8, 104, 256, 256, 256, 304])
        block, nblk, pieces, pkeys, own, okeys = plan(lib, B, grp, nkv, P, cap, bf16, cu)
        assert okeys % 32 == 0 and (own - 1) * okeys < cap <= own * okeys
        if P == 0:
            assert pieces == 0
        else:
            assert pkeys % 32 == 0 and (pieces - 1) * pkeys < P <= pieces * pkeys
            assert block in (16, 64, 128) and (nblk - 1) * block < B * grp <= nblk * block
            assert (block == 16) == (B * grp <= 16)
        # the merge keeps a factor per piece in LDS; the grid and its counts are 31-bit numbers
        assert (pieces + own) * 4 <= 32768
        assert (pieces * nkv + 7) // 8 * 8 * max(nblk, 1) + B * nkv * own < 2 ** 31


def test_workspace_holds_the_plan(lib):
    """The size a caller is asked for has room for every part of the plan (on 256 compute units, which
    is what is assumed where there is no GPU)."""
    rng = random.Random(4)
    for _ in range(500):
        B, grp, nkv = rng.randint(1, 70), rng.randint(1, 16), rng.choice([1, 2, 4])
        P, cap, bf16 = rng.randint(0, 40000), rng.randint(1, 5000), rng.random() < 0.5
        _, _, pieces, _, own, _ = plan(lib, B, grp, nkv, P, cap, bf16)
        a = pyq35.AttnBatchArgs(batch=B, q_heads=grp * nkv, kv_heads=nkv, head_dim=256, rotary_dim=64, kv_dtype=int(bf16),
                                prefix_len=P, prefix_capacity=P, own_capacity=cap)
        rows = B * grp * nkv
        plain = pyq35.lib.q35_attn_batch_workspace_bytes(a)
        assert plain >= rows * (pieces + own) * 258 * 4 + rows * 256 * (6 if bf16 else 4)
        a.own_score = 4096
        assert pyq35.lib.q35_attn_batch_workspace_bytes(a) - plain == rows * ((cap + 31) // 32 * 32) * 4
