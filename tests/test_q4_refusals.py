"""What the operators of a decode step held in 4 bits refuse: every check comes before any GPU work,
so it runs without one. (Lengths and settings that only the device knows are covered by the GPU tests.)"""
import pytest

import pyq35

ARG, RANGE, UNSUPPORTED = -1, -6, -7
BASE = 1 << 20
lib = pyq35.lib


def ptrs(names):
    """Distinct aligned addresses far apart, never read."""
    return {n: (i + 1) << 44 for i, n in enumerate(names)}


def status(fn, *a):
    st = fn(*a)
    if st:
        assert lib.q35_last_error()
    return st


MUL = ("X", "ldx", "packed", "zeros", "M", "N", "K", "group", "R", "ldr", "Y", "ldy", "workspace", "workspace_bytes")


def mul(**over):
    a = dict(ldx=200, zeros=0, M=3, N=100, K=200, group=64, R=None, ldr=0, ldy=100, workspace_bytes=1 << 40,
             **ptrs(("X", "packed", "Y", "workspace")))
    a.update(over)
    return status(lib.q35_matmul_q4, *(a[n] for n in MUL), None)


@pytest.mark.parametrize("over,want", [
    (dict(M=0), ARG), (dict(M=-1), ARG), (dict(M=4097), UNSUPPORTED), (dict(N=0), ARG), (dict(K=0), ARG), (dict(N=-5), ARG),
    (dict(group=16), UNSUPPORTED), (dict(group=0), UNSUPPORTED), (dict(group=256), UNSUPPORTED), (dict(zeros=2), ARG),
    (dict(zeros=-1), ARG), (dict(N=1 << 24, K=512, ldx=512, ldy=1 << 24), UNSUPPORTED), (dict(N=2147483647, K=2147483647), UNSUPPORTED),
    (dict(X=None), ARG), (dict(packed=None), ARG), (dict(Y=None), ARG), (dict(workspace=None), ARG), (dict(ldx=199), ARG),
    (dict(ldy=99), ARG), (dict(R=BASE, ldr=99), ARG), (dict(ldx=1 << 41), ARG), (dict(ldy=(1 << 63) - 1), ARG),
    (dict(packed=BASE + 8), ARG), (dict(workspace=BASE + 8), ARG), (dict(X=BASE + 2), ARG), (dict(Y=BASE + 1), ARG),
    (dict(X=BASE, Y=BASE + 400), ARG), (dict(packed=BASE, Y=BASE + 400), ARG), (dict(R=BASE, ldr=100, Y=BASE + 400), ARG),
    (dict(R=BASE, ldr=101, Y=BASE), ARG), (dict(workspace_bytes=0), ARG)])
def test_matmul(over, want):
    assert mul(**over) == want


def test_sizes():
    f = lib.q35_q4_packed_bytes
    assert f(16, 256, 64, 0) == 2048 + 128 and f(16, 256, 64, 1) == 2048 + 256 and f(17, 257, 32, 0) == 4 * (2048 + 256)
    assert f(1, 1, 128, 0) == 2048 + 64
    assert f(0, 256, 64, 0) == 0 and f(16, 256, 48, 0) == 0 and f(1 << 30, 256, 64, 0) == 0
    assert f(1 << 24, 256, 64, 0) == (1 << 20) * 2176                # beyond 32 bits of bytes
    w = lib.q35_matmul_q4_workspace_bytes
    assert w(1, 16, 256, 64) > 0 and w(0, 16, 256, 64) == 0 and w(4097, 16, 256, 64) == 0 and w(1, 16, 256, 31) == 0


@pytest.mark.parametrize("over,want", [
    (dict(N=0), ARG), (dict(K=-1), ARG), (dict(group=100), UNSUPPORTED), (dict(w_dtype=2), ARG), (dict(W=None), ARG),
    (dict(codes=None), ARG), (dict(scales=None), ARG), (dict(scales=BASE + 1), ARG), (dict(W=BASE + 1), ARG),
    (dict(W=BASE, codes=BASE + 8), ARG), (dict(codes=BASE, zeros=BASE + 3), ARG), (dict(N=1 << 28, K=1), UNSUPPORTED)])
def test_quantize(over, want):
    a = dict(w_dtype=0, N=10, K=100, group=32, zeros=None, **ptrs(("W", "codes", "scales")))
    a.update(over)
    assert status(lib.q35_q4_quantize, *(a[n] for n in ("W", "w_dtype", "N", "K", "group", "codes", "scales", "zeros")), None) == want


@pytest.mark.parametrize("over,want", [
    (dict(N=0), ARG), (dict(K=0), ARG), (dict(group=8), UNSUPPORTED), (dict(codes=None), ARG), (dict(scales=None), ARG),
    (dict(packed=None), ARG), (dict(packed=BASE + 8), ARG), (dict(codes=BASE + 16, packed=BASE), ARG),
    (dict(zeros=BASE + 16, packed=BASE), ARG)])
def test_pack(over, want):
    a = dict(N=10, K=100, group=32, zeros=None, **ptrs(("codes", "scales", "packed")))
    a.update(over)
    assert status(lib.q35_q4_pack, *(a[n] for n in ("codes", "scales", "zeros", "N", "K", "group", "packed")), None) == want


ATTN = ("len", "pos", "qg", "k_new", "v_new", "q_norm", "k_norm", "k", "v", "k_scale", "v_scale", "out", "workspace")


def attn(**over):
    a = dict(batch=3, q_heads=8, kv_heads=2, head_dim=256, rotary_dim=64, capacity=100, rope_theta=1e7, eps=1e-6,
             workspace_bytes=1 << 50, **ptrs(ATTN))
    a.update(over)
    return pyq35.AttnQ4Args(**a)


@pytest.mark.parametrize("over,want", [
    (dict(head_dim=128), UNSUPPORTED), (dict(batch=0), ARG), (dict(batch=-1), ARG), (dict(batch=65536), UNSUPPORTED),
    (dict(q_heads=0), ARG), (dict(kv_heads=0), ARG), (dict(q_heads=7), ARG), (dict(q_heads=34), UNSUPPORTED),
    (dict(batch=65535, q_heads=128, kv_heads=8), UNSUPPORTED), (dict(rotary_dim=-2), ARG), (dict(rotary_dim=258), ARG),
    (dict(rotary_dim=63), ARG), (dict(capacity=0), RANGE), (dict(capacity=1 << 31), RANGE), (dict(k=BASE, v=BASE + 128), ARG),
    (dict(k=BASE, v_scale=BASE + 128), ARG), (dict(workspace_bytes=100), ARG)] + [
    (dict([(n, None)]), ARG) for n in ATTN] + [(dict([(n, BASE + 8)]), ARG) for n in ATTN if n not in ("len", "pos")])
def test_attn(over, want):
    assert status(lib.q35_attn_q4, attn(**over), None) == want


def test_attn_null():
    assert status(lib.q35_attn_q4, None, None) == ARG and lib.q35_attn_q4_workspace_bytes(None) == 0
    need = lib.q35_attn_q4_workspace_bytes(attn())
    assert need > 0 and status(lib.q35_attn_q4, attn(workspace_bytes=need - 1), None) == ARG
    # the size depends on the sizes alone
    assert need == lib.q35_attn_q4_workspace_bytes(pyq35.AttnQ4Args(batch=3, q_heads=8, kv_heads=2, head_dim=256, rotary_dim=64,
                                                                    capacity=100))


KV = ("begin", "end", "k_rows", "v_rows", "k", "v", "k_scale", "v_scale")


def kv(**over):
    a = dict(batch=3, kv_heads=2, head_dim=256, kv_dtype=0, rows_capacity=100, capacity=80, **ptrs(KV))
    a.update(over)
    return pyq35.KvQ4Args(**a)


@pytest.mark.parametrize("fn", ["store", "load"])
@pytest.mark.parametrize("over,want", [
    (dict(head_dim=64), UNSUPPORTED), (dict(batch=0), ARG), (dict(kv_heads=-1), ARG), (dict(batch=65536), UNSUPPORTED),
    (dict(batch=65535, kv_heads=65535), UNSUPPORTED), (dict(kv_dtype=2), ARG), (dict(shared_rows=2), ARG), (dict(capacity=0), RANGE),
    (dict(rows_capacity=0), RANGE), (dict(capacity=1 << 31), RANGE), (dict(k=BASE, v=BASE + 64), None), (dict(k_rows=BASE, k=BASE), ARG),
    (dict(k_scale=BASE, v=BASE + 16), None)] + [(dict([(n, None)]), ARG) for n in KV[1:]] + [
    (dict([(n, BASE + 8)]), ARG) for n in KV[2:]])
def test_kv(fn, over, want):
    call = getattr(lib, f"q35_kv_q4_{fn}")
    if want is None:                       # arrays that only one direction writes
        if fn == "load":
            return
        want = ARG
    assert status(call, kv(**over), None) == want


def test_kv_shared():
    assert status(lib.q35_kv_q4_load, kv(shared_rows=1), None) == ARG
    assert status(lib.q35_kv_q4_load, kv(k_rows=BASE, v_rows=BASE + 1024), None) == ARG
    assert status(lib.q35_kv_q4_store, None, None) == ARG


SAMPLE = ("logits", "temperature", "top_k", "top_p", "min_p", "u", "token", "prob", "workspace")


def sample(**over):
    a = dict(batch=3, vocab=1000, ld_logits=1000, workspace_bytes=1 << 50, **ptrs(SAMPLE))
    a.update(over)
    return pyq35.SampleArgs(**a)


@pytest.mark.parametrize("over,want", [
    (dict(batch=0), ARG), (dict(vocab=0), ARG), (dict(batch=65536), UNSUPPORTED), (dict(vocab=(1 << 22) + 1), UNSUPPORTED),
    (dict(ld_logits=999), ARG), (dict(ld_logits=1 << 41), ARG), (dict(workspace=BASE + 4), ARG), (dict(logits=BASE + 2), ARG),
    (dict(workspace_bytes=0), ARG)] + [(dict([(n, None)]), ARG) for n in ("logits", "temperature", "u", "token", "workspace")])
def test_sample(over, want):
    assert status(lib.q35_sample, sample(**over), None) == want


def test_sample_null():
    assert status(lib.q35_sample, None, None) == ARG and lib.q35_sample_workspace_bytes(None) == 0
    need = lib.q35_sample_workspace_bytes(sample())
    assert need > 0 and status(lib.q35_sample, sample(workspace_bytes=need - 1), None) == ARG


@pytest.mark.parametrize("out", ["k", "v", "k_scale", "v_scale", "out", "workspace"])
@pytest.mark.parametrize("other", [n for n in ATTN])
def test_attn_overlap(out, other):
    """What is written shares a byte with another array's end, or ends where that begins."""
    if out == other:
        return
    sizes = {"len": 12, "pos": 12, "qg": 3 * 8 * 2048, "k_new": 3 * 2 * 1024, "v_new": 3 * 2 * 1024, "q_norm": 1024, "k_norm": 1024,
             "k": 600 * 128, "v": 600 * 128, "k_scale": 600 * 16, "v_scale": 600 * 16, "out": 3 * 8 * 1024}
    if other != "workspace":
        at = (sizes[other] - 1) // 16 * 16
        assert status(lib.q35_attn_q4, attn(**{other: BASE, out: BASE + at}), None) == ARG
    if out != "workspace":
        at = sizes[out] - 16
        assert status(lib.q35_attn_q4, attn(**{out: BASE, other: BASE + at}), None) == ARG


@pytest.mark.parametrize("out", ["token", "prob", "workspace"])
@pytest.mark.parametrize("other", SAMPLE)
def test_sample_overlap(out, other):
    if out == other:
        return
    if other != "workspace":
        last = {"logits": 3000}.get(other, 3) * 4 - 4
        at = last // 16 * 16 if out == "workspace" else last
        assert status(lib.q35_sample, sample(**{other: BASE, out: BASE + at}), None) == ARG
    if out != "workspace":
        assert status(lib.q35_sample, sample(**{out: BASE, other: BASE}), None) == ARG
