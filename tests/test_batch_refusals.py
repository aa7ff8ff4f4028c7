"""What the operators for a batch of continuations refuse: every check comes before any GPU work,
so it runs without one. (Lengths that only the device knows are covered by the GPU tests.)"""
import pytest

import pyq35

ARG, RANGE, UNSUPPORTED = -1, -6, -7
BASE = 1 << 20


def ptrs(names):
    """Distinct aligned addresses, never read."""
    return {n: BASE * (i + 1) * 4096 for i, n in enumerate(names)}


def attn(**over):
    p = ptrs(("own_len", "pos", "qg", "k_new", "v_new", "q_norm", "k_norm", "k_prefix", "v_prefix", "k_own", "v_own", "out",
              "workspace"))
    a = dict(batch=3, q_heads=8, kv_heads=2, head_dim=256, rotary_dim=64, kv_dtype=0, prefix_len=100, prefix_capacity=128,
             own_capacity=64, rope_theta=1e7, eps=1e-6, workspace_bytes=1 << 40, **p)
    a.update(over)
    return pyq35.AttnBatchArgs(**a)


def evict(**over):
    p = ptrs(("len", "next_pos", "score", "pos", "k", "v", "score_out", "pos_out", "new_len", "workspace"))
    a = dict(batch=3, kv_heads=2, head_dim=256, kv_dtype=0, keep=50, n_sink=4, n_recent=8, capacity=64,
             workspace_bytes=1 << 40, **p)
    a.update(over)
    return pyq35.KvEvictArgs(**a)


def gdn(**over):
    p = ptrs(("row0", "pos", "qkv", "z", "b", "a", "conv_w", "A_log", "dt_bias", "norm_w", "conv_ring", "state", "out"))
    a = dict(batch=3, rows=9, k_heads=2, v_heads=4, head_dim_k=128, head_dim_v=128, conv_kernel=4, eps=1e-6, ld_qkv=1024,
             ld_z=512, ld_ba=4, stride_ring=4096, stride_state=65536, **p)
    a.update(over)
    return pyq35.GdnBatchArgs(**a)


def status(fn, a):
    st = fn(a, None)
    if st:
        assert pyq35.lib.q35_last_error()
    return st


@pytest.mark.parametrize("over,want", [
    (dict(head_dim=128), UNSUPPORTED), (dict(batch=0), ARG), (dict(batch=-1), ARG), (dict(batch=65536), UNSUPPORTED),
    (dict(q_heads=0), ARG), (dict(kv_heads=0), ARG), (dict(q_heads=7), ARG), (dict(q_heads=34), UNSUPPORTED),
    (dict(rotary_dim=-2), ARG), (dict(rotary_dim=258), ARG), (dict(rotary_dim=63), ARG), (dict(kv_dtype=2), ARG),
    (dict(prefix_len=-1), RANGE), (dict(prefix_len=129), RANGE), (dict(own_capacity=0), RANGE),
    (dict(own_capacity=1 << 31), RANGE), (dict(prefix_capacity=1 << 31), RANGE),
    (dict(batch=65535, own_capacity=1 << 24, own_score=BASE), UNSUPPORTED),
    (dict(own_len=None), ARG), (dict(pos=None), ARG), (dict(qg=None), ARG), (dict(k_new=None), ARG), (dict(v_new=None), ARG),
    (dict(q_norm=None), ARG), (dict(k_norm=None), ARG), (dict(k_prefix=None), ARG), (dict(v_prefix=None), ARG),
    (dict(k_own=None), ARG), (dict(v_own=None), ARG), (dict(out=None), ARG), (dict(workspace=None), ARG),
    (dict(k_own=BASE + 8), ARG), (dict(qg=BASE + 4), ARG), (dict(k_prefix=BASE + 2), ARG), (dict(workspace=BASE + 8), ARG),
    (dict(workspace_bytes=1000), ARG)])
def test_attn_batch(over, want):
    assert status(pyq35.lib.q35_attn_batch, attn(**over)) == want


def test_attn_batch_workspace():
    size = lambda **o: pyq35.lib.q35_attn_batch_workspace_bytes(attn(**o))  # noqa: E731
    need = size()
    assert need > 0 and size(batch=0) == 0 and size(prefix_len=200) == 0
    assert status(pyq35.lib.q35_attn_batch, attn(workspace_bytes=need - 1)) == ARG
    assert size(own_score=BASE) >= need + 3 * 8 * 64 * 4          # the raw scores of the own rows
    assert size(prefix_len=0) < need and size(kv_dtype=1) > 0
    # sizes beyond 32 bits
    assert size(batch=4096, own_capacity=1 << 20, own_score=BASE) > 4096 * 8 * (1 << 20) * 4


@pytest.mark.parametrize("over,want", [
    (dict(head_dim=64), UNSUPPORTED), (dict(batch=0), ARG), (dict(kv_heads=0), ARG), (dict(batch=65536), UNSUPPORTED),
    (dict(kv_dtype=-1), ARG), (dict(capacity=0), RANGE), (dict(capacity=1 << 31), RANGE), (dict(keep=0), ARG), (dict(keep=-3), ARG),
    (dict(n_sink=-1), ARG), (dict(n_recent=-1), ARG), (dict(keep=11), ARG), (dict(n_sink=2147483647, n_recent=2147483647), ARG),
    (dict(len=None), ARG), (dict(next_pos=None), ARG), (dict(score=None), ARG), (dict(pos=None), ARG), (dict(k=None), ARG),
    (dict(v=None), ARG), (dict(score_out=None), ARG), (dict(pos_out=None), ARG), (dict(new_len=None), ARG),
    (dict(workspace=None), ARG), (dict(k=BASE + 8), ARG), (dict(workspace=BASE + 4), ARG), (dict(workspace_bytes=8), ARG),
    (dict(score=BASE * 4096, score_out=BASE * 4096 + 4), ARG), (dict(pos=BASE * 4096, pos_out=BASE * 4096 + 1024), ARG),
    (dict(k=BASE * 4096, v=BASE * 4096), ARG), (dict(len=BASE * 4096, new_len=BASE * 4096 + 4), ARG)])
def test_kv_evict(over, want):
    assert status(pyq35.lib.q35_kv_evict, evict(**over)) == want


def test_kv_evict_workspace():
    size = lambda **o: pyq35.lib.q35_kv_evict_workspace_bytes(evict(**o))  # noqa: E731
    assert size() > 0 and size(keep=100) > 0 and size(keep=0) == 0
    assert status(pyq35.lib.q35_kv_evict, evict(workspace_bytes=size() - 1)) == ARG


IN = dict(conv_ring_in=BASE * 1 << 20, state_in=BASE * 1 << 21)


@pytest.mark.parametrize("over,want", [
    (dict(head_dim_k=64), UNSUPPORTED), (dict(head_dim_v=256), UNSUPPORTED), (dict(conv_kernel=3), UNSUPPORTED),
    (dict(batch=0), ARG), (dict(rows=0), ARG), (dict(k_heads=0), ARG), (dict(v_heads=3), ARG), (dict(batch=65536), UNSUPPORTED),
    (dict(row0=None, rows=2), ARG), (dict(pos=None), ARG), (dict(qkv=None), ARG), (dict(b=None), ARG), (dict(a=None), ARG),
    (dict(conv_w=None), ARG), (dict(A_log=None), ARG), (dict(dt_bias=None), ARG), (dict(conv_ring=None), ARG),
    (dict(state=None), ARG), (dict(out=None), ARG), (dict(z=None), ARG), (dict(ld_qkv=1023), ARG), (dict(ld_z=511), ARG),
    (dict(ld_ba=3), ARG), (dict(stride_ring=4095), ARG), (dict(stride_state=65532), ARG), (dict(stride_state=65538), ARG),
    (dict(state=BASE + 4), ARG), (dict(conv_w=BASE + 8), ARG),
    (dict(state_in=BASE << 20), ARG), (dict(conv_ring_in=BASE << 20), ARG),
    (dict(**IN, stride_state_in=65532), ARG), (dict(**IN, stride_ring_in=4), ARG), (dict(**IN, stride_state_in=65538), ARG),
    # what is read overlaps what is written: the prompt's state is one of the branches', or half of one
    (dict(conv_ring_in=BASE << 20, state_in=BASE * 12 * 4096), ARG),
    (dict(conv_ring_in=BASE << 20, state_in=BASE * 12 * 4096 + 3 * 65536 * 4 - 16), ARG),
    (dict(conv_ring_in=BASE * 11 * 4096 + 4096 * 4, state_in=BASE << 21), ARG)])
def test_gdn_batch(over, want):
    assert status(pyq35.lib.q35_gdn_batch, gdn(**over)) == want


def test_null_args():
    for fn in (pyq35.lib.q35_attn_batch, pyq35.lib.q35_kv_evict, pyq35.lib.q35_gdn_batch):
        assert status(fn, None) == ARG
    assert pyq35.lib.q35_attn_batch_workspace_bytes(None) == 0 and pyq35.lib.q35_kv_evict_workspace_bytes(None) == 0
