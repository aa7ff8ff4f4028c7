"""The operators of a decode step held in 4 bits, and what their speed is judged on.

Products with 4-bit weights and group scales for one row to a batch of them (``q35_matmul_q4``),
attention of one token per sequence over a cache of 4-bit rows (``q35_attn_q4``), such a cache's rows
from and to an fp32 or bf16 cache (``q35_kv_q4_store``, ``q35_kv_q4_load``), and sampling with
temperature, top-k, top-p and min-p (``q35_sample``). ``run`` computes them in elementary torch
operations, or, with ``own`` set, through the library.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

HD = 256       # attention head dim
KG = 64        # dims of a cache row that share a step and a least value
ROT = 64       # rotary dims
THETA = 1e7
EPS = 1e-6
VOCAB = 151936
DEV = "cuda"


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through a square output projection: latency
        {"name": "q4 1 x 2048 x 2048", "kind": "mul", "rows": 1, "n": 2048, "k": 2048, "group": 64, "zeros": False,
         "residual": True},
        # one token through gate and up, zero points as converted checkpoints have them
        {"name": "q4 1 x 12288 x 2048 zeros", "kind": "mul", "rows": 1, "n": 12288, "k": 2048, "group": 128, "zeros": True,
         "residual": False},
        # one token's output head
        {"name": "q4 1 x head", "kind": "mul", "rows": 1, "n": VOCAB, "k": 2048, "group": 64, "zeros": False,
         "residual": False},
        # thirteen sequences through the down projection, small groups
        {"name": "q4 13 x 2048 x 6144", "kind": "mul", "rows": 13, "n": 2048, "k": 6144, "group": 32, "zeros": False,
         "residual": True},
        # a full batch through a GDN layer's fused input projection
        {"name": "q4 48 x 8224 x 2048 zeros", "kind": "mul", "rows": 48, "n": 8224, "k": 2048, "group": 64, "zeros": True,
         "residual": False},
        # one sequence of a short chat, small model's heads: latency
        {"name": "attn 1 of 700", "kind": "attn", "batch": 1, "q_heads": 8, "kv_heads": 2, "cap": 700, "full": True, "idle": 0},
        # one sequence at the longest context
        {"name": "attn 1 of 131072", "kind": "attn", "batch": 1, "q_heads": 16, "kv_heads": 2, "cap": 131072, "full": True,
         "idle": 0},
        # a padded batch, lengths spread from nothing to 8k: the largest
        {"name": "attn 40 of 8192", "kind": "attn", "batch": 40, "q_heads": 16, "kv_heads": 2, "cap": 8192, "full": False,
         "idle": 1},
        # a prompt's fp32 cache handed over after its prefill
        {"name": "store 1 of 8192", "kind": "store", "batch": 1, "kv_heads": 2, "cap": 8192, "bf16": False, "shared": False},
        # the caches of a few sequences opened again for the next prompts' prefill
        {"name": "load 5 of 4099 bf16", "kind": "load", "batch": 5, "kv_heads": 2, "cap": 4099, "bf16": True, "shared": False},
        # one sequence's next token
        {"name": "sample 1", "kind": "sample", "batch": 1, "vocab": VOCAB, "masked": False},
        # a batch with every sequence's own settings, some under a grammar that rules out most tokens
        {"name": "sample 48", "kind": "sample", "batch": 48, "vocab": VOCAB, "masked": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))


def draw(rng):
    kind = rng.choice(["mul", "mul", "attn", "attn", "store", "load", "sample", "sample"])
    if kind == "mul":
        rows, k = _log(rng, 1, 64), _log(rng, 32, 8192)
        most = min(VOCAB, 48 * 8224 * 2048 // (rows * k))
        return {"kind": kind, "rows": rows, "n": _log(rng, 16, most), "k": k, "group": rng.choice([32, 64, 64, 128]),
                "zeros": rng.random() < 0.4, "residual": rng.random() < 0.4}
    if kind == "attn":
        nq, nkv = rng.choice([(16, 2), (16, 2), (8, 2), (8, 2), (4, 1), (2, 1), (6, 3), (16, 1), (2, 2)])
        b = _log(rng, 1, 48)
        return {"kind": kind, "batch": b, "q_heads": nq, "kv_heads": nkv, "cap": _log(rng, 1, min(131072, 280000 // b)),
                "full": rng.random() < 0.4, "idle": rng.choice([0, 0, rng.randint(0, b - 1)])}
    if kind in ("store", "load"):
        b = _log(rng, 1, 24)
        return {"kind": kind, "batch": b, "kv_heads": rng.choice([1, 2, 2, 3]), "cap": _log(rng, 1, 24000 // b),
                "bf16": rng.random() < 0.5, "shared": kind == "store" and rng.random() < 0.3}
    b = _log(rng, 1, 48)
    return {"kind": kind, "batch": b, "vocab": _log(rng, 2, VOCAB), "masked": rng.random() < 0.3}


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 4242)
    return g


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    x = torch.empty(shape, dtype=torch.float32, device=DEV)
    x.normal_(0.0, std, generator=g)
    return x if dtype == torch.float32 else x.to(dtype)


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, dtype=torch.uint8, device=DEV, generator=g)


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _floats(a):
    return torch.tensor(np.asarray(a), dtype=torch.float32, device=DEV)


def _lengths(case, rng):
    cap, b = case["cap"], case["batch"]
    return rng.randint(cap - 1 - cap // 16, cap, b) if case.get("full", True) else rng.randint(0, cap, b)


def _cache(g, *shape):
    """Rows of 4-bit codes, and the (step, least) of their groups as normal values leave them."""
    step = 0.30 + 0.05 * _normal(g, *shape, HD // KG)
    return _bytes(g, *shape, HD // 2), torch.stack([step, -7.5 * step + 0.2 * _normal(g, *shape, HD // KG)], -1).half()


def prepare(case, seed):
    g, rng = _gen(seed), np.random.RandomState(int(seed) % (1 << 31))
    s = {"case": case, "workspace": torch.empty(0, dtype=torch.uint8, device=DEV)}
    if case["kind"] == "mul":
        M, N, K, G = (case[c] for c in ("rows", "n", "k", "group"))
        groups = (K + G - 1) // G
        zeros = torch.randint(5, 11, (N, groups), dtype=torch.uint8, device=DEV, generator=g) if case["zeros"] else None
        centre = torch.repeat_interleave(zeros, G, 1)[:, :K] if case["zeros"] else 8
        codes = torch.round(_normal(g, N, K, std=2.7) + centre).clamp_(0, 15).to(torch.uint8)
        if K % 2:
            codes = torch.cat([codes, codes.new_zeros(N, 1)], 1)
        s["codes"] = codes[:, 0::2] | codes[:, 1::2] << 4
        s["scales"], s["zeros"] = (0.0075 * torch.exp(_normal(g, N, groups, std=0.2))).half(), zeros
        s["x"] = _normal(g, M, K) * torch.exp(_normal(g, K, std=0.7))      # channels of unlike size
        s["r"] = _normal(g, M, N) if case["residual"] else None
        s["y"] = torch.zeros(M, N, device=DEV)
        if own:                                                            # laid out once, with the model
            q = _lib()
            s["packed"] = torch.empty(q.lib.q35_q4_packed_bytes(N, K, G, int(case["zeros"])), dtype=torch.uint8, device=DEV)
            q.check(q.lib.q35_q4_pack(s["codes"].data_ptr(), s["scales"].data_ptr(), zeros.data_ptr() if case["zeros"] else None,
                                      N, K, G, s["packed"].data_ptr(), torch.cuda.current_stream().cuda_stream))
    elif case["kind"] == "attn":
        B, NQ, NKV, cap = (case[c] for c in ("batch", "q_heads", "kv_heads", "cap"))
        s["k"], s["k_scale"] = _cache(g, B, NKV, cap)
        s["v"], s["v_scale"] = _cache(g, B, NKV, cap)
        n = _lengths(case, rng)
        pos = n + rng.randint(0, 1000, B)                                  # rows may have been evicted
        if case["idle"]:
            n[rng.permutation(B)[:case["idle"]]] = -1
        s["len"], s["pos"] = _ints(n), _ints(pos)
        s["qg"], s["k_new"], s["v_new"] = _normal(g, B, NQ, 2 * HD), _normal(g, B, NKV, HD), _normal(g, B, NKV, HD)
        s["q_norm"], s["k_norm"] = _normal(g, HD, std=0.1), _normal(g, HD, std=0.1)
        s["out"] = torch.zeros(B, NQ, HD, device=DEV)
    elif case["kind"] in ("store", "load"):
        B, NKV, cap = (case[c] for c in ("batch", "kv_heads", "cap"))
        kv = torch.bfloat16 if case["bf16"] else torch.float32
        src = 1 if case["shared"] else B
        store = case["kind"] == "store"
        for c in ("k", "v"):
            s[c], s[c + "_scale"] = _cache(g, B, NKV, cap)
            s[c + "_rows"] = _normal(g, src, NKV, cap, HD, dtype=kv) if store else torch.zeros(B, NKV, cap, HD, dtype=kv, device=DEV)
        end = np.full(B, cap) if B == 1 else rng.randint(0, cap + 1, B)
        s["begin"], s["end"] = _ints(np.where(rng.rand(B) < 0.7, 0, rng.randint(0, cap, B))), _ints(end)
        if B == 1:
            s["begin"].zero_()
    else:
        B, V = case["batch"], case["vocab"]
        # a head's logits: most tokens near one level, some few far above it
        x = _normal(g, B, V) * _floats(rng.uniform(1.0, 3.0, (B, 1)))
        x += 8.0 * torch.rand(B, V, device=DEV, generator=g).pow(2000)
        if case["masked"]:
            ruled = torch.rand(B, V, device=DEV, generator=g) < _floats(np.where(rng.rand(B, 1) < 0.3, 0.9, 0.0))
            ruled[:, 0] = False
            x = x.masked_fill(ruled, -math.inf)
        s["logits"] = x
        s["temperature"] = _floats(rng.choice([0.0, 0.6, 0.7, 1.0, 1.0, 1.3], B))
        s["top_k"] = _ints(rng.choice([0, 0, 20, 50, 1000], B))
        s["top_p"] = _floats(rng.choice([1.0, 0.95, 0.8], B))
        s["min_p"] = _floats(rng.choice([0.0, 0.0, 0.05], B))
        if B == 1:                                                         # the settings of a chat
            s["temperature"][:], s["top_k"][:], s["top_p"][:], s["min_p"][:] = 0.7, 20, 0.8, 0.0
        s["u"] = _floats(rng.rand(B).astype(np.float32).clip(0, 1 - 2.0 ** -24))
        s["token"], s["prob"] = torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B, device=DEV)
    return s


# ------------------------------------------------------------------------------ plain forms
def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _mul_plain(s):
    case = s["case"]
    K, G = case["k"], case["group"]
    c = _nibbles(s["codes"])[:, :K].float()
    zero = torch.repeat_interleave(s["zeros"].float(), G, 1)[:, :K] if case["zeros"] else 8.0
    w = (c - zero) * torch.repeat_interleave(s["scales"].float(), G, 1)[:, :K]
    y = torch.matmul(s["x"], w.t())
    s["y"].copy_(y + s["r"] if case["residual"] else y)
    return {"y": s["y"]}


def _values(codes, scale):
    """Cache rows as fp32: least + step * code."""
    sc = scale.float()
    return (_nibbles(codes).float().unflatten(-1, (HD // KG, KG)) * sc[..., :1] + sc[..., 1:]).flatten(-2)


def _codes(x):
    """Rows x (fp32 or bf16 values, or in 64 bits) as 4-bit codes and fp16 (step, least), from 64 bits:
    codes are compared as the whole numbers they are."""
    x = x.double().unflatten(-1, (HD // KG, KG))
    least = x.amin(-1).float().half()
    step = ((x.amax(-1) - least.double()) / 15.0).clamp(min=0.0).float().half()
    st = step.double()[..., None]
    n = torch.round((x - least.double()[..., None]) / torch.where(st == 0, torch.ones_like(st), st)).clamp(0, 15)
    n = torch.where(st == 0, torch.zeros_like(n), n).to(torch.uint8).flatten(-2)
    return n[..., 0::2] | n[..., 1::2] << 4, torch.stack([step, least], -1)


def _turned(x, w, pos, kind):
    """Normed rows x [B, n, HD] rotated at pos [B], computed in `kind`; angles in 64 bits."""
    x = x.to(kind)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w.to(kind))
    h = ROT // 2
    inv = THETA ** (-2.0 * torch.arange(h, device=DEV, dtype=torch.float64) / ROT)
    ang = pos.double()[:, None, None] * inv
    c, sn = torch.cos(ang).to(kind), torch.sin(ang).to(kind)
    a, b = x[..., :h], x[..., h:ROT]
    return torch.cat([a * c - b * sn, b * c + a * sn, x[..., ROT:]], -1)


def _attn_plain(s):
    case = s["case"]
    B, NQ, NKV, cap = (case[c] for c in ("batch", "q_heads", "kv_heads", "cap"))
    q = _turned(s["qg"][..., :HD], s["q_norm"], s["pos"], torch.float32).view(B, NKV, NQ // NKV, HD) * HD ** -0.5
    at, active = s["len"].long(), s["len"] >= 0
    lane, slot = torch.arange(B, device=DEV), at.clamp(min=0)
    # the new rows in 64 bits: a value next to the border of two codes is on one side of it
    for c, x in (("k", _turned(s["k_new"], s["k_norm"], s["pos"], torch.float64)), ("v", s["v_new"])):
        codes, scale = _codes(x)
        s[c][lane, :, slot] = torch.where(active[:, None, None], codes, s[c][lane, :, slot])
        s[c + "_scale"][lane, :, slot] = torch.where(active[:, None, None, None], scale, s[c + "_scale"][lane, :, slot])
    sc = torch.matmul(q, _values(s["k"], s["k_scale"]).transpose(-1, -2))          # [B][NKV][group][cap]
    sc = sc.masked_fill((torch.arange(cap, device=DEV) > at[:, None])[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, torch.zeros_like(m), m))
    o = torch.matmul(p, _values(s["v"], s["v_scale"])) / p.sum(-1, keepdim=True)
    y = o.reshape(B, NQ, HD) * torch.sigmoid(s["qg"][..., HD:])
    s["out"].copy_(torch.where(active[:, None, None], y, s["out"]))
    return {c: s[c] for c in ("out", "k", "v", "k_scale", "v_scale")}


def _within(s):
    row = torch.arange(s["case"]["cap"], device=DEV)
    return ((row >= s["begin"][:, None]) & (row < s["end"][:, None]))[:, None, :, None]


def _store_plain(s):
    on = _within(s)
    for c in ("k", "v"):
        codes, scale = _codes(s[c + "_rows"])
        s[c].copy_(torch.where(on, codes, s[c]))
        s[c + "_scale"].copy_(torch.where(on[..., None], scale, s[c + "_scale"]))
    return {c: s[c] for c in ("k", "v", "k_scale", "v_scale")}


def _load_plain(s):
    on = _within(s)
    for c in ("k", "v"):
        s[c + "_rows"].copy_(torch.where(on, _values(s[c], s[c + "_scale"]).to(s[c + "_rows"].dtype), s[c + "_rows"]))
    return {c: s[c] for c in ("k_rows", "v_rows")}


def _sample_plain(s):
    """In 64 bits: which candidates are left, and which of them is drawn, goes by sums next to borders."""
    x, order = torch.sort(s["logits"], dim=-1, descending=True, stable=True)       # ties: the lower id first
    t = s["temperature"].double()[:, None]
    z = (x.double() - x[:, :1].double()) / torch.where(t > 0, t, torch.ones_like(t))
    w = torch.exp(z)
    rank = torch.arange(x.shape[1], device=DEV)
    k = s["top_k"].long()[:, None]
    w = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    before = torch.cumsum(w, -1) - w
    total = w.sum(-1, keepdim=True)
    keep = ((before < s["top_p"].double()[:, None] * total) | (s["top_p"][:, None] >= 1)) & (w >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    keep &= (t > 0) | (rank == 0)
    w = torch.where(keep, w, torch.zeros_like(w))
    run_ = torch.cumsum(w, -1)
    mass = run_[:, -1:]
    at = (run_ <= s["u"].double()[:, None] * mass).sum(-1, keepdim=True)
    s["token"].copy_(torch.gather(order, 1, at)[:, 0])
    s["prob"].copy_((torch.gather(w, 1, at) / mass)[:, 0])
    return {"token": s["token"], "prob": s["prob"]}


# ------------------------------------------------------------------------------ the library
def _lib():
    if "pyq35" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.5-cpu-cpp_amd"))
    import pyq35
    return pyq35


def _workspace(s, need):
    if s["workspace"].numel() < need:   # kept with the state, as a program keeps one for all its calls
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    return s["workspace"].data_ptr()


def _mul_own(s):
    q, case = _lib(), s["case"]
    M, N, K, G = (case[c] for c in ("rows", "n", "k", "group"))
    need = q.lib.q35_matmul_q4_workspace_bytes(M, N, K, G)
    q.check(q.lib.q35_matmul_q4(s["x"].data_ptr(), K, s["packed"].data_ptr(), int(case["zeros"]), M, N, K, G,
                                s["r"].data_ptr() if case["residual"] else None, N, s["y"].data_ptr(), N,
                                _workspace(s, need), need, torch.cuda.current_stream().cuda_stream))
    return {"y": s["y"]}


def _attn_own(s):
    q, case = _lib(), s["case"]
    P = {n: s[n].data_ptr() for n in ("len", "pos", "qg", "k_new", "v_new", "q_norm", "k_norm", "k", "v", "k_scale",
                                      "v_scale", "out")}
    a = q.AttnQ4Args(batch=case["batch"], q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=HD, rotary_dim=ROT,
                     capacity=case["cap"], rope_theta=THETA, eps=EPS, **P)
    a.workspace_bytes = q.lib.q35_attn_q4_workspace_bytes(a)
    a.workspace = _workspace(s, a.workspace_bytes)
    q.check(q.lib.q35_attn_q4(a, torch.cuda.current_stream().cuda_stream))
    return {c: s[c] for c in ("out", "k", "v", "k_scale", "v_scale")}


def _kv_own(s):
    q, case = _lib(), s["case"]
    names = ("begin", "end", "k", "v", "k_scale", "v_scale", "k_rows", "v_rows")
    a = q.KvQ4Args(batch=case["batch"], kv_heads=case["kv_heads"], head_dim=HD, kv_dtype=int(case["bf16"]),
                   shared_rows=int(case["shared"]), rows_capacity=case["cap"], capacity=case["cap"],
                   **{n: s[n].data_ptr() for n in names})
    store = case["kind"] == "store"
    q.check((q.lib.q35_kv_q4_store if store else q.lib.q35_kv_q4_load)(a, torch.cuda.current_stream().cuda_stream))
    return {c: s[c] for c in (("k", "v", "k_scale", "v_scale") if store else ("k_rows", "v_rows"))}


def _sample_own(s):
    q, case = _lib(), s["case"]
    names = ("logits", "temperature", "top_k", "top_p", "min_p", "u", "token", "prob")
    a = q.SampleArgs(batch=case["batch"], vocab=case["vocab"], ld_logits=case["vocab"], **{n: s[n].data_ptr() for n in names})
    a.workspace_bytes = q.lib.q35_sample_workspace_bytes(a)
    a.workspace = _workspace(s, a.workspace_bytes)
    q.check(q.lib.q35_sample(a, torch.cuda.current_stream().cuda_stream))
    return {"token": s["token"], "prob": s["prob"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"mul": _mul_own, "attn": _attn_own, "store": _kv_own, "load": _kv_own, "sample": _sample_own}[kind](state)
    return {"mul": _mul_plain, "attn": _attn_plain, "store": _store_plain, "load": _load_plain,
            "sample": _sample_plain}[kind](state)


# ------------------------------------------------------------------------------ work
def work(case):
    if case["kind"] == "mul":
        M, N, K, G = (case[c] for c in ("rows", "n", "k", "group"))
        w = N * ((K + 1) // 2) + N * ((K + G - 1) // G) * (3 if case["zeros"] else 2)
        return {"bytes": w + 4.0 * M * (K + N * (2 if case["residual"] else 1)), "flops": 2.0 * M * N * K}
    if case["kind"] == "attn":
        B, NQ, NKV, cap = (case[c] for c in ("batch", "q_heads", "kv_heads", "cap"))
        B -= case["idle"]
        rows = B * (cap - 1 - cap // 32 if case["full"] else (cap - 1) / 2.0)
        return {"bytes": 2 * NKV * 144.0 * (rows + B) + 4.0 * B * HD * (3 * NQ + 2 * NKV), "flops": 4.0 * NQ * HD * (rows + B)}
    if case["kind"] in ("store", "load"):
        B, NKV, cap = (case[c] for c in ("batch", "kv_heads", "cap"))
        rows = cap if B == 1 else B * cap * (0.5 * 0.7 + 0.3 / 6)
        wide = rows if not case["shared"] else min(rows, cap)
        return {"bytes": 2.0 * NKV * (rows * 144 + wide * HD * (2 if case["bf16"] else 4)), "flops": 4.0 * NKV * rows * HD}
    return {"bytes": 4.0 * case["batch"] * case["vocab"], "flops": 4.0 * case["batch"] * case["vocab"]}


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"mul": _exact_mul, "attn": _exact_attn, "store": _exact_store, "load": _exact_load,
            "sample": _exact_sample}[case["kind"]](s)


def _exact_mul(s):
    """Column by column of groups: codes and scales are never multiplied out."""
    case, f = s["case"], torch.float64
    M, N, K, G = (case[c] for c in ("rows", "n", "k", "group"))
    y = s["r"].to(f) if case["residual"] else torch.zeros(M, N, dtype=f, device=DEV)
    for i, k0 in enumerate(range(0, K, G)):
        at = torch.arange(k0, min(k0 + G, K), device=DEV)
        c = torch.bitwise_right_shift(s["codes"][:, at // 2], (4 * (at % 2)).to(torch.uint8)) % 16
        x = s["x"][:, at].to(f)
        zero = s["zeros"][:, i].to(f) if case["zeros"] else torch.full((N,), 8.0, dtype=f, device=DEV)
        y += (x @ c.to(f).T.contiguous() - x.sum(1, keepdim=True) * zero) * s["scales"][:, i].to(f)
    return {"y": y}


def _row_values(codes, scale, f=torch.float64):
    at = torch.arange(HD, device=DEV)
    n = torch.bitwise_right_shift(codes[..., at // 2], (4 * (at % 2)).to(torch.uint8)) % 16
    return scale[..., at // KG, 1].to(f) + scale[..., at // KG, 0].to(f) * n.to(f)


def _row_codes(x):
    """Rows on the host, group by group, with numpy."""
    x = x.detach().double().cpu().numpy().reshape(-1, HD // KG, KG)
    lo, hi = x.min(-1), x.max(-1)
    least = lo.astype(np.float32).astype(np.float16)
    step = np.maximum((hi - least.astype(np.float64)) / 15.0, 0.0).astype(np.float32).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.rint((x - least[..., None].astype(np.float64)) / step[..., None].astype(np.float64))
    n = np.where(step[..., None] == 0, 0, np.clip(n, 0, 15)).astype(np.uint8).reshape(-1, HD)
    codes = n[:, ::2] + 16 * n[:, 1::2]
    return torch.from_numpy(codes).to(DEV), torch.from_numpy(np.stack([step, least], -1)).to(DEV)


def _exact_attn(s):
    """Sequence by sequence, over the rows that it attends."""
    case, f = s["case"], torch.float64
    G, h = case["q_heads"] // case["kv_heads"], ROT // 2
    res = {"out": s["out"].to(f)}

    def turned(x, w, pos):
        x = x.to(f)
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * (1 + w.to(f))
        z = torch.complex(x[:, :h].contiguous(), x[:, h:ROT].contiguous())
        ang = pos / THETA ** (2 * torch.arange(h, device=DEV, dtype=f) / ROT)
        z = z * torch.polar(torch.ones_like(ang), ang)
        return torch.cat([z.real, z.imag, x[:, ROT:]], 1)

    for b, (n, pos) in enumerate(zip(s["len"].tolist(), s["pos"].tolist())):
        if n < 0:
            continue
        q = turned(s["qg"][b, :, :HD], s["q_norm"], pos)
        s["k"][b, :, n], s["k_scale"][b, :, n] = _row_codes(turned(s["k_new"][b], s["k_norm"], pos))
        s["v"][b, :, n], s["v_scale"][b, :, n] = _row_codes(s["v_new"][b])
        for kv in range(case["kv_heads"]):
            K = _row_values(s["k"][b, kv, :n + 1], s["k_scale"][b, kv, :n + 1])
            V = _row_values(s["v"][b, kv, :n + 1], s["v_scale"][b, kv, :n + 1])
            res["out"][b, kv * G:(kv + 1) * G] = torch.softmax(q[kv * G:(kv + 1) * G] @ K.T.contiguous() / 16.0, -1) @ V
        res["out"][b] /= 1 + torch.exp(-s["qg"][b, :, HD:].to(f))
    # the caches as they are afterwards: codes are whole numbers, steps and least values fp16
    res.update({c: s[c] for c in ("k", "v")}, **{c: s[c].to(f) for c in ("k_scale", "v_scale")})
    return res


def _ranges(s):
    return [(b, i, max(i, e)) for b, (i, e) in enumerate(zip(s["begin"].tolist(), s["end"].tolist()))]


def _exact_store(s):
    """On the host, sequence by sequence."""
    for b, i, e in _ranges(s):
        for c in ("k", "v"):
            rows = s[c + "_rows"][0 if s["case"]["shared"] else b, :, i:e]
            if e > i:
                codes, scale = _row_codes(rows)
                s[c][b, :, i:e], s[c + "_scale"][b, :, i:e] = codes.view(rows.shape[0], e - i, -1), scale.view(rows.shape[0], e - i, -1, 2)
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"].double(), "v_scale": s["v_scale"].double()}


def _exact_load(s):
    res = {c: s[c].double() for c in ("k_rows", "v_rows")}
    for b, i, e in _ranges(s):
        for c in ("k", "v"):
            res[c + "_rows"][b, :, i:e] = _row_values(s[c][b, :, i:e], s[c + "_scale"][b, :, i:e])
    return res


def _exact_sample(s):
    """On the host, row by row, over a sorted list."""
    token, prob = [], []
    p = {n: s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p", "u")}
    for b, x in enumerate(s["logits"].double().cpu().numpy()):
        order = np.lexsort((np.arange(len(x)), -x))
        if p["temperature"][b] <= 0:
            token.append(int(order[0]))
            prob.append(1.0)
            continue
        if p["top_k"][b] > 0:
            order = order[:p["top_k"][b]]
        w = np.exp((x[order] - x[order[0]]) / p["temperature"][b])
        n = len(w)
        if p["top_p"][b] < 1:
            n = max(1, int(np.searchsorted(np.cumsum(w), p["top_p"][b] * w.sum(), side="left")) + 1)
        n = max(1, min(n, int((w >= p["min_p"][b]).sum())))
        c = np.cumsum(w[:n])
        at = int(np.searchsorted(c, p["u"][b] * c[-1], side="right"))
        token.append(int(order[at]))
        prob.append(w[at] / c[-1])
    return {"token": torch.tensor(token, dtype=torch.int32, device=DEV), "prob": torch.tensor(prob, dtype=torch.float64, device=DEV)}
