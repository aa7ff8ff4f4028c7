"""The operators of decoding a batch of continuations of one prompt, and what their speed is judged on.

Three operators: attention of one token per sequence over a shared prefix and each sequence's own
cache (``q35_attn_batch``), eviction of own-cache rows by accumulated attention weight
(``q35_kv_evict``), and the recurrent gated delta rule with a state per sequence
(``q35_gdn_batch``). ``run`` computes them in elementary torch operations, or, with ``own`` set,
through the library.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

D = 128        # GDN head dims
HD = 256       # attention head dim
ROT = 64       # rotary dims
THETA = 1e7
EPS = 1e-6
DEV = "cuda"


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # two answers of a short chat prompt sampled side by side, small model's heads: latency
        {"name": "attn 2 after 700", "kind": "attn", "batch": 2, "q_heads": 8, "kv_heads": 2, "prefix": 700,
         "own": 64, "bf16": False, "scores": False, "idle": 0},
        # best-of-16 over an 8k document, bf16 caches
        {"name": "attn 16 after 8k bf16", "kind": "attn", "batch": 16, "q_heads": 16, "kv_heads": 2, "prefix": 8192,
         "own": 512, "bf16": True, "scores": False, "idle": 0},
        # a padded batch of the small model over an odd prompt length, fp32 caches
        {"name": "attn 13 after 5003", "kind": "attn", "batch": 13, "q_heads": 8, "kv_heads": 2, "prefix": 5003,
         "own": 300, "bf16": False, "scores": False, "idle": 2},
        # many branches of one long context: the largest
        {"name": "attn 48 after 30k", "kind": "attn", "batch": 48, "q_heads": 16, "kv_heads": 2, "prefix": 30001,
         "own": 1000, "bf16": False, "scores": False, "idle": 0},
        # independent sequences in bounded caches, weights accumulated for the next eviction
        {"name": "attn 24 bounded bf16", "kind": "attn", "batch": 24, "q_heads": 8, "kv_heads": 2, "prefix": 0,
         "own": 2304, "bf16": True, "scores": True, "idle": 1},
        # one sequence's cache a little over its budget
        {"name": "evict 1 of 1152", "kind": "evict", "batch": 1, "kv_heads": 2, "cap": 1152, "keep": 1024, "bf16": False},
        # a batch of bounded caches brought back to their budget
        {"name": "evict 24 of 2304 bf16", "kind": "evict", "batch": 24, "kv_heads": 2, "cap": 2304, "keep": 2048,
         "bf16": True},
        # a long prompt's cache cut to a quarter
        {"name": "evict 1 of 131072", "kind": "evict", "batch": 1, "kv_heads": 2, "cap": 131072, "keep": 32768,
         "bf16": False},
        # one token of a few answers sampled side by side: latency
        {"name": "gdn 3 x 1", "kind": "gdn", "batch": 3, "k_heads": 16, "v_heads": 16, "most": 1, "fork": False,
         "norm": True},
        # one token of a full batch
        {"name": "gdn 64 x 1", "kind": "gdn", "batch": 64, "k_heads": 16, "v_heads": 16, "most": 1, "fork": False,
         "norm": True},
        # drafted tokens verified: 0 to 8 a sequence, v-heads sharing k-heads
        {"name": "gdn 20 x 0..8", "kind": "gdn", "batch": 20, "k_heads": 8, "v_heads": 16, "most": 8, "fork": False,
         "norm": True},
        # the first token of 32 answers: every one starts from the prompt's state
        {"name": "gdn fork 32", "kind": "gdn", "batch": 32, "k_heads": 16, "v_heads": 16, "most": 1, "fork": True,
         "norm": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "evict", "gdn"])
    bf16 = rng.random() < 0.5
    if kind == "attn":
        nq, nkv = rng.choice([(16, 2), (16, 2), (8, 2), (8, 2), (4, 1), (2, 1), (6, 3), (16, 1)])
        b = _log(rng, 1, 48)
        prefix = 0 if rng.random() < 0.2 else _log(rng, 1, min(30000, 700000 // b))
        return {"kind": kind, "batch": b, "q_heads": nq, "kv_heads": nkv, "prefix": prefix,
                "own": _log(rng, 1, 2304 if b <= 24 else 1000), "bf16": bf16, "scores": rng.random() < 0.4,
                "idle": rng.choice([0, 0, rng.randint(0, b - 1)])}
    if kind == "evict":
        b = _log(rng, 1, 32)
        cap = _log(rng, 2, 131072 // b)
        return {"kind": kind, "batch": b, "kv_heads": rng.choice([1, 2, 2, 3]), "cap": cap,
                "keep": rng.choice([rng.randint(1, cap), max(1, cap * 7 // 8)]), "bf16": bf16}
    kh = rng.choice([2, 4, 8, 16, 16])
    vh = kh * (1 if kh == 16 else rng.choice([1, 2]))
    return {"kind": kind, "batch": _log(rng, 1, 64), "k_heads": kh, "v_heads": vh,
            "most": rng.choice([1, 1, rng.randint(2, 12)]), "fork": rng.random() < 0.3, "norm": rng.random() < 0.8}


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 777)
    return g


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    x = torch.empty(shape, dtype=torch.float32, device=DEV)
    x.normal_(0.0, std, generator=g)
    return x if dtype == torch.float32 else x.to(dtype)


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g, rng = _gen(seed), np.random.RandomState(int(seed) % (1 << 31))
    s = {"case": case}
    if case["kind"] == "attn":
        B, NQ, NKV, P, cap = (case[k] for k in ("batch", "q_heads", "kv_heads", "prefix", "own"))
        kv = torch.bfloat16 if case["bf16"] else torch.float32
        s["k_prefix"], s["v_prefix"] = (_normal(g, NKV, P, HD, dtype=kv) for _ in range(2))
        s["k_own"], s["v_own"] = (_normal(g, B, NKV, cap, HD, dtype=kv) for _ in range(2))
        n = rng.randint(0, cap, B)
        if case["idle"]:
            n[rng.permutation(B)[:case["idle"]]] = -1
        s["own_len"], s["pos"] = _ints(n), _ints(P + np.maximum(n, 0))
        s["qg"], s["k_new"], s["v_new"] = _normal(g, B, NQ, 2 * HD), _normal(g, B, NKV, HD), _normal(g, B, NKV, HD)
        s["q_norm"], s["k_norm"] = _normal(g, HD, std=0.1), _normal(g, HD, std=0.1)
        s["out"] = torch.zeros(B, NQ, HD, device=DEV)
        if case["scores"]:
            s["score"] = _normal(g, B, NKV, cap).abs_()
            s["own_pos"] = torch.arange(cap, dtype=torch.int32, device=DEV).repeat(B, NKV, 1) + P
        s["workspace"] = torch.empty(0, dtype=torch.uint8, device=DEV)
    elif case["kind"] == "evict":
        B, NKV, cap, keep = (case[k] for k in ("batch", "kv_heads", "cap", "keep"))
        kv = torch.bfloat16 if case["bf16"] else torch.float32
        s["k"], s["v"] = (_normal(g, B, NKV, cap, HD, dtype=kv) for _ in range(2))
        n = np.where(rng.rand(B) < 0.75, cap, rng.randint(0, cap + 1, B))
        s["len"], s["next_pos"] = _ints(n), _ints(np.full(B, cap + 11))
        # what attention leaves: few rows with much weight, ties at nothing
        score = torch.exp(2.0 * _normal(g, B, NKV, cap))
        s["score"] = torch.where(torch.rand(B, NKV, cap, device=DEV, generator=g) < 0.1, torch.zeros_like(score), score)
        # an earlier eviction has left the rows out of order
        s["pos"] = torch.rand(B, NKV, cap, device=DEV, generator=g).argsort(-1).to(torch.int32)
        s["score_out"], s["pos_out"] = torch.zeros_like(score), torch.zeros_like(s["pos"])
        s["new_len"] = torch.zeros_like(s["len"])
        s["workspace"] = torch.empty(0, dtype=torch.uint8, device=DEV)
    else:
        B, KH, VH, most = (case[k] for k in ("batch", "k_heads", "v_heads", "most"))
        conv, VD = (2 * KH + VH) * D, VH * D
        n = np.ones(B, np.int64) if most == 1 else rng.randint(0, most + 1, B)
        rows = B * most                             # a padded buffer: the sequences' rows lie at its front
        s["row0"] = _ints(np.concatenate([[0], np.cumsum(n)])) if most > 1 else None
        s["rows"] = rows
        p = _normal(g, rows, conv + VD + 2 * VH)   # the projection's rows, as one product leaves them
        s["proj"] = p
        s["pos"] = _ints(np.full(B, 1037) if case["fork"] else rng.randint(0, 100000, B))
        s["conv_w"], s["A_log"], s["dt_bias"] = _normal(g, conv, 4, std=0.5), _normal(g, VH), _normal(g, VH)
        s["norm_w"] = 1.0 + _normal(g, D, std=0.1)
        s["ring"], s["state"] = _normal(g, B, 4, conv), _normal(g, B, VH, D, D, std=0.1)
        if case["fork"]:
            s["ring_in"], s["state_in"] = _normal(g, 4, conv), _normal(g, VH, D, D, std=0.1)
        s["out"] = torch.zeros(rows, VD, device=DEV)
    return s


# ------------------------------------------------------------------------------ plain forms
def _rope(x, pos, one):
    """Rotates the first ROT dims of x [..., n, HD] at pos (one per leading index)."""
    h = ROT // 2
    inv = THETA ** (-2.0 * torch.arange(h, device=DEV, dtype=torch.float64) / ROT)
    ang = pos.double()[:, None, None] * inv
    c, s = torch.cos(ang).to(one), torch.sin(ang).to(one)
    a, b = x[..., :h], x[..., h:ROT]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., ROT:]], -1)


def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)


def _attn_plain(s):
    case = s["case"]
    B, NQ, NKV, P, cap = (case[k] for k in ("batch", "q_heads", "kv_heads", "prefix", "own"))
    G = NQ // NKV
    q = _rope(_rms(s["qg"][..., :HD], s["q_norm"]), s["pos"], torch.float32).view(B, NKV, G, HD) * HD ** -0.5
    k = _rope(_rms(s["k_new"], s["k_norm"]), s["pos"], torch.float32)
    slot = torch.arange(cap, device=DEV)
    at, active = s["own_len"].long(), s["own_len"] >= 0
    fresh = (slot == at[:, None])[:, None, :]                             # the appended slot
    s["k_own"].copy_(torch.where(fresh[..., None], k[:, :, None].to(s["k_own"].dtype), s["k_own"]))
    s["v_own"].copy_(torch.where(fresh[..., None], s["v_new"][:, :, None].to(s["v_own"].dtype), s["v_own"]))
    so = torch.matmul(q, s["k_own"].float().transpose(-1, -2))             # [B][NKV][G][cap]
    so = so.masked_fill((slot > at[:, None])[:, None, None, :], -math.inf)
    m = so.amax(-1, keepdim=True)
    if P:
        qp = q.transpose(0, 1).reshape(NKV, B * G, HD)
        sp = torch.matmul(qp, s["k_prefix"].float().transpose(-1, -2))     # [NKV][B G][P]
        mp = sp.amax(-1, keepdim=True).view(NKV, B, G, 1).transpose(0, 1)
        m = torch.maximum(m, mp)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    po = torch.exp(so - m)
    l = po.sum(-1, keepdim=True)
    o = torch.matmul(po, s["v_own"].float())
    if P:
        pp = torch.exp(sp - m.transpose(0, 1).reshape(NKV, B * G, 1))
        l = l + pp.sum(-1, keepdim=True).view(NKV, B, G, 1).transpose(0, 1)
        o = o + torch.matmul(pp, s["v_prefix"].float()).view(NKV, B, G, HD).transpose(0, 1)
    y = (o / l).reshape(B, NQ, HD) * torch.sigmoid(s["qg"][..., HD:])
    s["out"].copy_(torch.where(active[:, None, None], y, s["out"]))
    r = {"out": s["out"], "k_own": s["k_own"], "v_own": s["v_own"]}
    if case["scores"]:
        w = torch.where(active[:, None, None], (po / l).sum(2), torch.zeros_like(s["score"]))
        s["score"].copy_(torch.where(fresh, w, s["score"] + w))
        s["own_pos"].copy_(torch.where(fresh, s["pos"][:, None, None], s["own_pos"]))
        r.update(score=s["score"], own_pos=s["own_pos"])
    return r


def _sinks(keep):
    """Rows kept whatever their weight: the first and the latest positions."""
    return min(4, keep // 2), min(64, keep // 4)


def _evict_plain(s):
    case = s["case"]
    cap, keep = case["cap"], case["keep"]
    n_sink, n_recent = _sinks(keep)
    slot = torch.arange(cap, device=DEV)
    n = s["len"].long()[:, None, None]
    live = slot < n
    held = (s["pos"] < n_sink) | (s["pos"] >= (s["next_pos"][:, None, None] - n_recent))
    key = torch.where(live, torch.where(held, math.inf, s["score"]), -1.0)
    rank = torch.argsort(torch.argsort(key, dim=-1, descending=True, stable=True), dim=-1)
    kept = live & ((rank < keep) | (n <= keep))
    low = slot < keep
    hole, src = low & live & ~kept, ~low & kept
    nth_hole = torch.cumsum(hole, -1) - 1
    first = torch.argsort((~src).to(torch.uint8), dim=-1, stable=True)     # the survivors to move, in order
    take = torch.where(hole, torch.gather(first, -1, nth_hole.clamp(min=0)), slot)
    rows = take[..., :keep, None].expand(-1, -1, -1, HD)
    s["k"][:, :, :keep] = torch.gather(s["k"], 2, rows)
    s["v"][:, :, :keep] = torch.gather(s["v"], 2, rows)
    new_len = torch.where(s["len"] > keep, keep, s["len"])
    left = slot < new_len[:, None, None]
    s["score_out"].copy_(torch.where(left, torch.gather(s["score"], -1, take), s["score_out"]))
    s["pos_out"].copy_(torch.where(left, torch.gather(s["pos"], -1, take), s["pos_out"]))
    s["new_len"].copy_(new_len)
    return {n: s[n] for n in ("k", "v", "score_out", "pos_out", "new_len")}


def _gdn_plain(s):
    case = s["case"]
    B, KH, VH, most = (case[k] for k in ("batch", "k_heads", "v_heads", "most"))
    conv, VD = (2 * KH + VH) * D, VH * D
    p, lanes = s["proj"], torch.arange(B, device=DEV)
    state = s["state_in"].expand(B, VH, D, D) if case["fork"] else s["state"]
    ring = s["ring_in"].expand(B, 4, conv) if case["fork"] else s["ring"]
    first = lanes if s["row0"] is None else s["row0"][:-1].long()
    n = torch.ones_like(lanes) if s["row0"] is None else s["row0"][1:].long() - first
    pos = s["pos"].long()
    order = torch.stack([(pos + i) % 4 for i in (1, 2, 3)], 1)
    win = torch.gather(ring, 1, order[..., None].expand(-1, -1, conv))     # the three inputs before, oldest first
    decay_w, wt = -torch.exp(s["A_log"]), s["conv_w"].t()
    out = torch.cat([s["out"], s["out"][:1]])     # and a row for the sequences that have no more tokens
    for t in range(most):
        on = n > t
        x = p[torch.where(on, first + t, 0)]
        seen = torch.cat([win, x[:, None, :conv]], 1)
        y = torch.nn.functional.silu((seen * wt).sum(1))
        qk = y[:, :2 * KH * D].view(B, 2, KH, D)
        qk = qk * torch.rsqrt((qk * qk).sum(-1, keepdim=True) + 1e-6)
        qk = qk.repeat_interleave(VH // KH, dim=2)
        q, k, v = qk[:, 0] * D ** -0.5, qk[:, 1], y[:, 2 * KH * D:].view(B, VH, D)
        beta = torch.sigmoid(x[:, conv + VD:conv + VD + VH])
        decay = torch.exp(decay_w * torch.nn.functional.softplus(x[:, conv + VD + VH:] + s["dt_bias"]))
        S = state * decay[..., None, None]
        d = (v - (S * k[..., None]).sum(-2)) * beta[..., None]
        S = S + k[..., None] * d[..., None, :]
        o = (S * q[..., None]).sum(-2)
        if case["norm"]:
            z = x[:, conv:conv + VD].view(B, VH, D)
            o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_w"] * torch.nn.functional.silu(z)
        out[torch.where(on, first + t, s["rows"])] = o.reshape(B, VD)
        state = torch.where(on[:, None, None, None], S, state)   # sequences with fewer tokens stand still
        win = torch.where(on[:, None, None], seen[:, 1:], win)
    s["out"].copy_(out[:-1])
    s["state"].copy_(state)
    if case["fork"]:
        s["ring"].copy_(s["ring_in"].expand(B, 4, conv))
    last = (pos + n)[:, None] + torch.tensor([-3, -2, -1], device=DEV)
    s["ring"].scatter_(1, (last % 4)[..., None].expand(-1, -1, conv), win)
    s["ring"].copy_(_oldest(s, n, pos, ring, conv))
    return {"out": s["out"], "state": s["state"], "ring": s["ring"]}


def _oldest(s, n, pos, ring, conv):
    """The ring with its fourth slot, the input of position pos + n - 4, set too."""
    row = (s["row0"][1:].long() if s["row0"] is not None else torch.arange(1, n.numel() + 1, device=DEV)) - 4
    slot = (pos + n) % 4
    new = s["proj"][row.clamp(min=0)][:, :conv]
    kept = torch.gather(ring, 1, slot[:, None, None].expand(-1, 1, conv))[:, 0]
    return s["ring"].scatter(1, slot[:, None, None].expand(-1, 1, conv), torch.where((n >= 4)[:, None], new, kept)[:, None])


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


def _attn_own(s):
    q, case = _lib(), s["case"]
    P = {n: s[n].data_ptr() for n in ("own_len", "pos", "qg", "k_new", "v_new", "q_norm", "k_norm", "k_prefix",
                                      "v_prefix", "k_own", "v_own", "out")}
    if case["scores"]:
        P["own_score"], P["own_pos"] = s["score"].data_ptr(), s["own_pos"].data_ptr()
    a = q.AttnBatchArgs(batch=case["batch"], q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=HD,
                        rotary_dim=ROT, kv_dtype=int(case["bf16"]), prefix_len=case["prefix"],
                        prefix_capacity=case["prefix"], own_capacity=case["own"], rope_theta=THETA, eps=EPS, **P)
    a.workspace_bytes = q.lib.q35_attn_batch_workspace_bytes(a)
    a.workspace = _workspace(s, a.workspace_bytes)
    q.check(q.lib.q35_attn_batch(a, torch.cuda.current_stream().cuda_stream))
    r = {"out": s["out"], "k_own": s["k_own"], "v_own": s["v_own"]}
    if case["scores"]:
        r.update(score=s["score"], own_pos=s["own_pos"])
    return r


def _evict_own(s):
    q, case = _lib(), s["case"]
    n_sink, n_recent = _sinks(case["keep"])
    a = q.KvEvictArgs(batch=case["batch"], kv_heads=case["kv_heads"], head_dim=HD, kv_dtype=int(case["bf16"]),
                      keep=case["keep"], n_sink=n_sink, n_recent=n_recent, capacity=case["cap"],
                      **{n: s[n].data_ptr() for n in ("len", "next_pos", "score", "pos", "k", "v", "score_out",
                                                      "pos_out", "new_len")})
    a.workspace_bytes = q.lib.q35_kv_evict_workspace_bytes(a)
    a.workspace = _workspace(s, a.workspace_bytes)
    q.check(q.lib.q35_kv_evict(a, torch.cuda.current_stream().cuda_stream))
    return {n: s[n] for n in ("k", "v", "score_out", "pos_out", "new_len")}


def _gdn_own(s):
    q, case = _lib(), s["case"]
    KH, VH = case["k_heads"], case["v_heads"]
    conv, VD = (2 * KH + VH) * D, VH * D
    base, ld = s["proj"].data_ptr(), s["proj"].shape[1]
    P = {n: s[n].data_ptr() for n in ("pos", "conv_w", "A_log", "dt_bias", "state", "out")}
    if s["row0"] is not None:
        P["row0"] = s["row0"].data_ptr()
    if case["norm"]:
        P["norm_w"] = s["norm_w"].data_ptr()
    if case["fork"]:
        P["state_in"], P["conv_ring_in"] = s["state_in"].data_ptr(), s["ring_in"].data_ptr()
    a = q.GdnBatchArgs(batch=case["batch"], rows=s["rows"], k_heads=KH, v_heads=VH, head_dim_k=D, head_dim_v=D,
                       conv_kernel=4, eps=EPS, qkv=base, z=base + 4 * conv, b=base + 4 * (conv + VD),
                       a=base + 4 * (conv + VD + VH), ld_qkv=ld, ld_z=ld, ld_ba=ld, conv_ring=s["ring"].data_ptr(),
                       stride_ring=4 * conv, stride_state=VH * D * D, **P)
    q.check(q.lib.q35_gdn_batch(a, torch.cuda.current_stream().cuda_stream))
    return {"out": s["out"], "state": s["state"], "ring": s["ring"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return (_attn_own if kind == "attn" else _evict_own if kind == "evict" else _gdn_own)(state)
    return (_attn_plain if kind == "attn" else _evict_plain if kind == "evict" else _gdn_plain)(state)


# ------------------------------------------------------------------------------ work
def work(case):
    e = 2 if case.get("bf16") else 4
    if case["kind"] == "attn":
        B, NQ, NKV, P = (case[k] for k in ("batch", "q_heads", "kv_heads", "prefix"))
        B -= case["idle"]
        rows = B * (case["own"] - 1) / 2.0           # own lengths are spread evenly over [0, own)
        b = 2 * NKV * HD * e * (P + rows) + 2 * NKV * HD * (4 + e) * B + 4 * B * NQ * HD * 3
        if case["scores"]:
            b += 8 * NKV * (rows + B)
        return {"bytes": b, "flops": 4.0 * NQ * HD * (B * (P + 1) + rows)}
    if case["kind"] == "evict":
        B, NKV, cap, keep = (case[k] for k in ("batch", "kv_heads", "cap", "keep"))
        over = 0.75 + 0.25 * (cap - keep) / (cap + 1.0)   # sequences beyond their budget
        n = 0.75 * cap + 0.25 * (cap + keep) / 2.0 * (cap - keep) / (cap + 1.0)
        moved = over * keep * (1.0 - keep / max(cap, 1.0))
        return {"bytes": B * NKV * (8 * n + 8 * min(keep, cap) + moved * 4 * HD * e), "flops": B * NKV * n}
    B, KH, VH = (case[k] for k in ("batch", "k_heads", "v_heads"))
    conv, VD = (2 * KH + VH) * D, VH * D
    rows = B if case["most"] == 1 else B * case["most"] / 2.0
    states = B + (1 if case["fork"] else B)
    return {"bytes": 4.0 * (states * VH * D * D + rows * (conv + 2 * VD + 2 * VH) + (3 * B + min(rows, 4 * B)) * conv + 4 * conv),
            "flops": rows * VH * D * D * 8.0}


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attn(s) if case["kind"] == "attn" else _exact_evict(s) if case["kind"] == "evict" else _exact_gdn(s)


def _exact_attn(s):
    """Sequence by sequence, over the rows that it attends."""
    case, f = s["case"], torch.float64
    NQ, NKV, P = case["q_heads"], case["kv_heads"], case["prefix"]
    G, h = NQ // NKV, ROT // 2
    res = {"out": s["out"].to(f), "k_own": s["k_own"].to(f), "v_own": s["v_own"].to(f)}
    if case["scores"]:
        res["score"], res["own_pos"] = s["score"].to(f), None
    kp, vp = s["k_prefix"].to(f), s["v_prefix"].to(f)

    def turned(x, w, pos):
        x = x.to(f)
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * (1 + w.to(f))
        z = torch.complex(x[:, :h].contiguous(), x[:, h:ROT].contiguous())
        ang = pos / THETA ** (2 * torch.arange(h, device=DEV, dtype=f) / ROT)
        z = z * torch.polar(torch.ones_like(ang), ang)
        return torch.cat([z.real, z.imag, x[:, ROT:]], 1)

    for b, (n, pos) in enumerate(zip(s["own_len"].tolist(), s["pos"].tolist())):
        if n < 0:
            continue
        q, k = turned(s["qg"][b, :, :HD], s["q_norm"], pos), turned(s["k_new"][b], s["k_norm"], pos)
        res["k_own"][b, :, n], res["v_own"][b, :, n] = k, s["v_new"][b].to(f)
        # the cache's rows as attention reads them: rounded to its type
        ko = torch.cat([s["k_own"][b, :, :n].to(f), k.to(s["k_own"].dtype).to(f)[:, None]], 1)
        vo = torch.cat([s["v_own"][b, :, :n].to(f), s["v_new"][b].to(s["v_own"].dtype).to(f)[:, None]], 1)
        for kv in range(NKV):
            K, V = torch.cat([kp[kv], ko[kv]]), torch.cat([vp[kv], vo[kv]])
            p = torch.softmax(q[kv * G:(kv + 1) * G] @ K.T / 16.0, -1)
            res["out"][b, kv * G:(kv + 1) * G] = p @ V
            if case["scores"]:
                w = p[:, P:].sum(0)
                res["score"][b, kv, :n] += w[:n]
                res["score"][b, kv, n] = w[n]
        res["out"][b] /= 1 + torch.exp(-s["qg"][b, :, HD:].to(f))
    return res


def _exact_evict(s):
    """On the host, cache by cache: whole numbers and copies, so every value is exact."""
    case = s["case"]
    keep = case["keep"]
    n_sink, n_recent = _sinks(keep)
    score, pos = s["score"].cpu().numpy(), s["pos"].cpu().numpy()
    k, v = s["k"].double(), s["v"].double()
    so, po, nl = s["score_out"].double(), s["pos_out"].clone(), s["len"].clone()
    for b, (n, nxt) in enumerate(zip(s["len"].tolist(), s["next_pos"].tolist())):
        for h in range(case["kv_heads"]):
            at = np.arange(min(n, keep))
            if n > keep:
                held = (pos[b, h, :n] < n_sink) | (pos[b, h, :n] >= nxt - n_recent)
                best = np.lexsort((np.arange(n), -score[b, h, :n].astype(np.float64), ~held))[:keep]
                at[np.setdiff1d(np.arange(keep), best)] = np.sort(best[best >= keep])
                i = torch.from_numpy(at).to(DEV)
                k[b, h, :keep], v[b, h, :keep] = k[b, h][i], v[b, h][i]
                nl[b] = keep
            so[b, h, :len(at)] = torch.from_numpy(score[b, h][at]).to(DEV).double()
            po[b, h, :len(at)] = torch.from_numpy(pos[b, h][at]).to(DEV)
    return {"k": k, "v": v, "score_out": so, "pos_out": po, "new_len": nl}


def _exact_gdn(s):
    """Sequence by sequence, token by token, with matrix products; the ring as a list of inputs."""
    case, f = s["case"], torch.float64
    KH, VH = case["k_heads"], case["v_heads"]
    conv, VD = (2 * KH + VH) * D, VH * D
    p, out = s["proj"].to(f), s["out"].to(f)
    state, ring = s["state"].to(f), s["ring"].to(f)
    w = s["conv_w"].to(f)
    ends = list(range(case["batch"] + 1)) if s["row0"] is None else s["row0"].tolist()
    for b, pos in enumerate(s["pos"].tolist()):
        S = (s["state_in"] if case["fork"] else s["state"][b]).to(f)
        if case["fork"]:
            ring[b] = s["ring_in"].to(f)
        for r in range(ends[b], ends[b + 1]):
            ring[b, pos % 4] = p[r, :conv]
            x = sum(w[:, i] * ring[b, (pos + 1 + i) % 4] for i in range(4))
            x = x / (1 + torch.exp(-x))
            q, k = (x[i * KH * D:(i + 1) * KH * D].view(KH, D) for i in (0, 1))
            q, k = (u / (u.pow(2).sum(1, keepdim=True) + 1e-6).sqrt() for u in (q, k))
            q, k = (u.repeat_interleave(VH // KH, 0)[:, :, None] for u in (q / D ** 0.5, k))
            v = x[2 * KH * D:].view(VH, 1, D)
            beta = 1 / (1 + torch.exp(-p[r, conv + VD:conv + VD + VH]))
            gate = torch.exp(-torch.exp(s["A_log"].to(f)) * torch.log1p(torch.exp(p[r, conv + VD + VH:] + s["dt_bias"].to(f))))
            S = S * gate[:, None, None]
            S = S + torch.bmm(k, (v - torch.bmm(k.transpose(1, 2), S)) * beta[:, None, None])
            o = torch.bmm(q.transpose(1, 2), S)[:, 0]
            if case["norm"]:
                z = p[r, conv:conv + VD].view(VH, D)
                o = o / (o.pow(2).mean(1, keepdim=True) + EPS).sqrt() * s["norm_w"].to(f) * z / (1 + torch.exp(-z))
            out[r] = o.reshape(VD)
            pos += 1
        state[b] = S
    return {"out": out, "state": state, "ring": ring}
