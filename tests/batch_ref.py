"""Float64 definitions of the operators for a batch of continuations, device buffers for their
calls, and captured graphs (test infrastructure)."""
from __future__ import annotations

import ctypes as C

import numpy as np

import pyq35
from helpers import bf16_bits, bf16_to_f32

HD, D = 256, 128
THETA, EPS = 1e7, 1e-6


# ------------------------------------------------------------------------------ definitions
def rope64(x, pos, rot, theta=THETA):
    """Rotates the first `rot` dims of the rows x [n][HD] to position pos."""
    h = rot // 2
    y = np.array(x, np.float64)
    if h:
        ang = float(pos) * float(theta) ** (-2.0 * np.arange(h) / rot)
        c, s = np.cos(ang), np.sin(ang)
        a, b = y[:, :h].copy(), y[:, h:rot].copy()
        y[:, :h], y[:, h:rot] = a * c - b * s, b * c + a * s
    return y


def rms64(x, w, eps=EPS):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + np.asarray(w, np.float64))


def attn64(x, b, rows_k, rows_v):
    """Sequence b over the given key and value rows [NKV][T][HD] (its new row among them):
    (out [NQ][HD], weights [NQ][T])."""
    NQ, NKV = x["qg"].shape[1], x["k_new"].shape[1]
    G = NQ // NKV
    q = rope64(rms64(x["qg"][b, :, :HD], x["q_norm"]), x["pos"][b], x["rot"])
    out, wts = np.zeros((NQ, HD)), np.zeros((NQ, rows_k.shape[1]))
    for h in range(NQ):
        s = np.asarray(rows_k[h // G], np.float64) @ q[h] / 16.0
        p = np.exp(s - s.max())
        p /= p.sum()
        wts[h] = p
        out[h] = (p @ np.asarray(rows_v[h // G], np.float64)) / (1.0 + np.exp(-x["qg"][b, h, HD:].astype(np.float64)))
    return out, wts


def evict_rows(score, pos, n, keep, n_sink, n_recent, next_pos):
    """Slots the first min(n, keep) rows come from after the eviction of one cache."""
    if n <= keep:
        return np.arange(max(n, 0))
    held = (pos[:n] < n_sink) | (pos[:n].astype(np.int64) >= int(next_pos) - n_recent)
    s = score[:n].astype(np.float64)
    nan = np.isnan(s)
    # protected rows are equal among themselves, whatever their weight
    order = sorted(range(n), key=lambda t: (0, 0, 0, t) if held[t] else (1, nan[t], 0.0 if nan[t] else -s[t], t))
    kept = np.zeros(n, bool)
    kept[order[:keep]] = True
    take = np.arange(keep)
    take[~kept[:keep]] = np.nonzero(kept[keep:])[0] + keep
    return take


def gdn64(x, b, first, n, pos, ring, state):
    """n tokens of one sequence from row `first`: (out [n][VD], ring, state) in float64."""
    KH, VH = x["KH"], x["VH"]
    KD, VD = KH * D, VH * D
    CONV = 2 * KD + VD
    ring, S = np.array(ring, np.float64), np.array(state, np.float64)
    out = np.zeros((n, VD))
    sig = lambda u: 1.0 / (1.0 + np.exp(-u))  # noqa: E731
    for t in range(n):
        r, p = first + t, pos + t
        ring[p % 4] = x["qkv"][r, :CONV]
        y = sum(x["conv_w"][:, i].astype(np.float64) * ring[(p + 1 + i) % 4] for i in range(4))
        y = y * sig(y)
        q, k, v = y[:KD].reshape(KH, D), y[KD:2 * KD].reshape(KH, D), y[2 * KD:].reshape(VH, D)
        q = q / np.sqrt((q * q).sum(-1, keepdims=True) + 1e-6) / np.sqrt(D)
        k = k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6)
        for h in range(VH):
            kh = h // (VH // KH)
            u = float(x["a"][r, h]) + float(x["dt_bias"][h])
            g = -np.exp(float(x["A_log"][h])) * (u if u > 30 else np.log1p(np.exp(u)))
            S[h] *= np.exp(g)
            d = (v[h] - k[kh] @ S[h]) * sig(float(x["b"][r, h]))
            S[h] += np.outer(k[kh], d)
            o = q[kh] @ S[h]
            if x.get("norm_w") is not None:
                z = x["z"][r, h * D:(h + 1) * D].astype(np.float64)
                o = o / np.sqrt((o * o).mean() + EPS) * x["norm_w"] * z * sig(z)
            out[t, h * D:(h + 1) * D] = o
    return out, ring, S


# ------------------------------------------------------------------------------ device side
class Buffers:
    """Named device copies of host arrays, freed together."""

    def __init__(self, hip, **arrays):
        self.hip, self.p, self.shape = hip, {}, {}
        for n, a in arrays.items():
            if a is not None:
                self.put(n, a)

    def put(self, name, a):
        a = np.ascontiguousarray(a)
        self.p[name], self.shape[name] = self.hip.upload(a), (a.shape, a.dtype)

    def get(self, name):
        shape, dt = self.shape[name]
        return self.hip.download(self.p[name], shape, dt)

    def set(self, name, a):
        self.hip.copy_in(self.p[name], np.ascontiguousarray(a, self.shape[name][1]))

    def __enter__(self):
        return self

    def __exit__(self, *e):
        self.hip.sync()
        for p in self.p.values():
            self.hip.free(p)


def cache_in(x, bf16):
    return bf16_bits(x) if bf16 else np.ascontiguousarray(x, np.float32)


def cache_out(x):
    return bf16_to_f32(x) if x.dtype == np.uint16 else x


def attn_args(bufs, x, bf16, cap, prefix_len, prefix_cap, scores=True, ws="ws"):
    B, NQ = x["qg"].shape[:2]
    a = pyq35.AttnBatchArgs(batch=B, q_heads=NQ, kv_heads=x["k_new"].shape[1], head_dim=HD, rotary_dim=x["rot"],
                            kv_dtype=int(bf16), prefix_len=prefix_len, prefix_capacity=prefix_cap, own_capacity=cap,
                            rope_theta=THETA, eps=EPS)
    for n in ("own_len", "pos", "qg", "k_new", "v_new", "q_norm", "k_norm", "k_own", "v_own", "out") + (
            ("k_prefix", "v_prefix") if prefix_cap else ()) + (("own_score", "own_pos") if scores else ()):
        setattr(a, n, bufs.p[n])
    a.workspace_bytes = pyq35.lib.q35_attn_batch_workspace_bytes(a)
    assert a.workspace_bytes > 0
    if ws not in bufs.p:
        bufs.put(ws, np.full(a.workspace_bytes, 0xFF, np.uint8))   # NaN wherever it is read before it is written
    a.workspace = bufs.p[ws]
    return a


def evict_args(bufs, B, NKV, cap, keep, n_sink, n_recent, bf16, **names):
    a = pyq35.KvEvictArgs(batch=B, kv_heads=NKV, head_dim=HD, kv_dtype=int(bf16), keep=keep, n_sink=n_sink,
                          n_recent=n_recent, capacity=cap)
    for n in ("len", "next_pos", "score", "pos", "k", "v", "score_out", "pos_out", "new_len"):
        setattr(a, n, bufs.p[names.get(n, n)])
    a.workspace_bytes = pyq35.lib.q35_kv_evict_workspace_bytes(a)
    assert a.workspace_bytes > 0
    if "ws_evict" not in bufs.p:
        bufs.put("ws_evict", np.full(a.workspace_bytes, 0x7F, np.uint8))
    a.workspace = bufs.p["ws_evict"]
    return a


def gdn_args(bufs, x, B, rows, fork=False):
    KH, VH = x["KH"], x["VH"]
    CONV = (2 * KH + VH) * D
    a = pyq35.GdnBatchArgs(batch=B, rows=rows, k_heads=KH, v_heads=VH, head_dim_k=D, head_dim_v=D, conv_kernel=4, eps=EPS,
                           ld_qkv=x["qkv"].shape[1], ld_z=x["z"].shape[1], ld_ba=x["b"].shape[1],
                           conv_ring=bufs.p["ring"], stride_ring=4 * CONV, stride_state=VH * D * D)
    for n in ("row0", "pos", "qkv", "z", "b", "a", "conv_w", "A_log", "dt_bias", "norm_w", "state", "out"):
        if n in bufs.p:
            setattr(a, n, bufs.p[n])
    if fork:
        a.conv_ring_in, a.state_in = bufs.p["ring_in"], bufs.p["state_in"]
    return a


class Graph:
    """What `calls(stream)` launches, captured once and replayed."""

    def __init__(self, hip, calls):
        rt, P = hip.rt, C.c_void_p
        self.hip, self.stream, g, self.exec = hip, P(), P(), P()
        hip._ck(rt.hipStreamCreate(C.byref(self.stream)), "hipStreamCreate")
        hip._ck(rt.hipStreamBeginCapture(self.stream, C.c_int(1)), "hipStreamBeginCapture")
        try:
            calls(self.stream)
        finally:
            e = rt.hipStreamEndCapture(self.stream, C.byref(g))
        hip._ck(e, "hipStreamEndCapture")
        hip._ck(rt.hipGraphInstantiate(C.byref(self.exec), g, None, None, C.c_size_t(0)), "hipGraphInstantiate")
        hip._ck(rt.hipGraphDestroy(g), "hipGraphDestroy")

    def replay(self):
        self.hip._ck(self.hip.rt.hipGraphLaunch(self.exec, self.stream), "hipGraphLaunch")
        self.hip.stream_sync(self.stream.value)

    def close(self):
        self.hip._ck(self.hip.rt.hipGraphExecDestroy(self.exec), "hipGraphExecDestroy")
        self.hip._ck(self.hip.rt.hipStreamDestroy(self.stream), "hipStreamDestroy")
