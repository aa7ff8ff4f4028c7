"""Definitions of the operators of a decode step held in 4 bits, in float64 and whole numbers, and
arguments for their calls (test infrastructure)."""
from __future__ import annotations

import numpy as np

import pyq35
from batch_ref import EPS, HD, THETA, rms64, rope64

KG = 64  # values of a cache row that share a step and a least value


# ------------------------------------------------------------------------------ 4-bit weights
def nibbles(b):
    """Bytes [..., n] as codes [..., 2 n], the low four bits first."""
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def bytes_of(c):
    """Codes [N][K] as bytes [N][(K + 1) / 2]."""
    if c.shape[-1] % 2:
        c = np.concatenate([c, np.zeros_like(c[..., :1])], -1)
    return (c[..., ::2] | c[..., 1::2] << 4).astype(np.uint8)


def weights64(codes, scales, zeros, K, G):
    """The values of 4-bit weights [N][K]."""
    c = nibbles(codes)[:, :K].astype(np.float64)
    g = np.arange(K) // G
    z = 8.0 if zeros is None else (zeros[:, g] & 15).astype(np.float64)
    return (c - z) * scales.view(np.float16)[:, g].astype(np.float64)


def quantize_weights(W, K, G, asym):
    """Codes, scale bits and zeros of fp32 values W [N][K], step by step as the header has it."""
    N, groups = W.shape[0], (K + G - 1) // G
    pad = np.zeros((N, groups * G), np.float32)
    pad[:, :K] = W
    x = pad.reshape(N, groups, G)
    with np.errstate(all="ignore"):
        lo, hi = np.minimum(np.nanmin(x, -1), 0), np.maximum(np.nanmax(x, -1), 0)
        raw = (hi - lo) / np.float32(15) if asym else np.where(hi > -lo, hi, lo) * np.float32(-0.125)
        bad = ~np.isfinite(x).all(-1)
        s16 = np.where(bad, np.float16(np.nan), raw.astype(np.float32).astype(np.float16))
        s = s16.astype(np.float32)
        none = bad | (s == 0)
        zero = np.where(none | (not asym), np.float32(8), np.clip(np.rint(-lo / s), 0, 15)).astype(np.float32)
        c = np.where(none[..., None], zero[..., None], np.clip(np.rint(x / s[..., None]) + zero[..., None], 0, 15))
    c = np.nan_to_num(c).astype(np.uint8).reshape(N, -1)[:, :K]
    return bytes_of(c), s16.view(np.uint16), zero.astype(np.uint8)


# ------------------------------------------------------------------------------ 4-bit cache rows
def row_codes(x):
    """Rows x [..., 256] as codes [..., 128] bytes and (step, least) [..., 4, 2] fp16."""
    x = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], HD // KG, KG)
    with np.errstate(all="ignore"):
        least = x.min(-1).astype(np.float32).astype(np.float16)
        step = np.maximum((x.max(-1) - least.astype(np.float64)) / 15.0, 0.0).astype(np.float32).astype(np.float16)
        bad = ~(np.isfinite(x).all(-1) & np.isfinite(least) & np.isfinite(step))
        n = np.rint((x - least[..., None].astype(np.float64)) / step[..., None].astype(np.float64))
        n = np.where(bad[..., None] | (step[..., None] == 0), 0, np.clip(n, 0, 15)).astype(np.uint8)
    sc = np.stack([step, least], -1)
    sc[bad] = np.float16(np.nan)
    n = n.reshape(*n.shape[:-2], HD)
    return (n[..., ::2] | n[..., 1::2] << 4).astype(np.uint8), sc


def row_values(codes, scale):
    """What 4-bit rows stand for, in float64."""
    sc = scale.astype(np.float64)
    n = nibbles(codes).astype(np.float64).reshape(*codes.shape[:-1], HD // KG, KG)
    return (sc[..., 1:] + sc[..., :1] * n).reshape(*codes.shape[:-1], HD)


def same_rows(a, b):
    """Bitwise, but any NaN for another."""
    x, y = a.view(np.uint16), b.view(np.uint16)
    return ((x == y) | (np.isnan(a.astype(np.float32)) & np.isnan(b.astype(np.float32)))).all()


def attn_q4_args(bufs, x, cap, ws="ws"):
    B, NQ = x["qg"].shape[:2]
    a = pyq35.AttnQ4Args(batch=B, q_heads=NQ, kv_heads=x["k_new"].shape[1], head_dim=HD, rotary_dim=x["rot"], capacity=cap,
                         rope_theta=THETA, eps=EPS)
    for n in ("len", "pos", "qg", "k_new", "v_new", "q_norm", "k_norm", "k", "v", "k_scale", "v_scale", "out"):
        setattr(a, n, bufs.p[n])
    a.workspace_bytes = pyq35.lib.q35_attn_q4_workspace_bytes(a)
    assert a.workspace_bytes > 0
    if ws not in bufs.p:
        bufs.put(ws, np.full(a.workspace_bytes, 0xFF, np.uint8))   # NaN wherever it is read before it is written
    a.workspace = bufs.p[ws]
    return a


def kv_q4_args(bufs, B, NKV, rows_cap, cap, bf16, shared=False, begin=True):
    a = pyq35.KvQ4Args(batch=B, kv_heads=NKV, head_dim=HD, kv_dtype=int(bf16), shared_rows=int(shared), rows_capacity=rows_cap,
                       capacity=cap)
    for n in ("end", "k_rows", "v_rows", "k", "v", "k_scale", "v_scale") + (("begin",) if begin else ()):
        setattr(a, n, bufs.p[n])
    return a


# ------------------------------------------------------------------------------ sampling
def sample64(x, t, k, p, m, u):
    """(token, prob, room) of one row: room is how far the nearest border is, relative to the weight."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    order = np.lexsort((np.arange(len(x)), -x))
    top = x[order[0]]
    if top == -np.inf:
        return -1, 0.0, np.inf
    if t == 0:
        return int(order[0]), 1.0, np.inf
    if k > 0:
        order = order[:k]
    with np.errstate(all="ignore"):
        d = np.where(x[order] == top, 0.0, x[order] - top)
        w = np.where(x[order] == -np.inf, 0.0, np.exp(np.where(d == 0, 0.0, d / t)))
    w = np.where((top == np.inf) & (x[order] != np.inf), 0.0, w)
    n, room = len(w), np.inf
    if p < 1:
        before = np.cumsum(w) - w
        n = max(1, int((before < float(p) * w.sum()).sum()))
        room = min(room, np.abs(before[1:] - float(p) * w.sum()).min(initial=np.inf) / w.sum())
    if m > 0:
        n = max(1, min(n, int((w >= float(m)).sum())))
        room = min(room, np.abs(w[1:] - float(m)).min(initial=np.inf))
    c = np.cumsum(w[:n])
    goal = min(max(float(u), 0.0), 1 - 2.0 ** -53) * c[-1]
    at = min(int(np.searchsorted(c, goal, side="right")), n - 1)
    room = min(room, np.abs(c[:-1] - goal).min(initial=np.inf) / c[-1])
    return int(order[at]), w[at] / c[-1], room


def sample_args(bufs, B, V, ld, ws="ws"):
    a = pyq35.SampleArgs(batch=B, vocab=V, ld_logits=ld)
    for n in ("logits", "temperature", "top_k", "top_p", "min_p", "u", "token", "prob"):
        if n in bufs.p:
            setattr(a, n, bufs.p[n])
    a.workspace_bytes = pyq35.lib.q35_sample_workspace_bytes(a)
    assert a.workspace_bytes > 0
    if ws not in bufs.p:
        bufs.put(ws, np.full(a.workspace_bytes, 0xFF, np.uint8))
    a.workspace = bufs.p[ws]
    return a


def turned(x, b, rows, w):
    return rope64(rms64(rows, w), x["pos"][b], x["rot"])


