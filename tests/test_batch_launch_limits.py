"""Batches whose launches would exceed the 2^32 threads of a grid's dimension are refused before the
first launch, which appends the new rows. CPU only; every call here is one that has to be refused."""
import pytest

import pyq35
from test_batch_refusals import BASE, UNSUPPORTED, attn, status


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("over", [
    dict(batch=65535, q_heads=256, kv_heads=16, own_capacity=8),                  # output rows
    dict(batch=32768, q_heads=256, kv_heads=256, own_capacity=1, prefix_len=0),   # one row more than there may be
    dict(batch=4096, own_capacity=1 << 20, own_score=BASE)])                      # pieces of the scores
def test_merge(over, bf16):
    assert status(pyq35.lib.q35_attn_batch, attn(kv_dtype=bf16, workspace_bytes=1 << 50, **over)) == UNSUPPORTED


def test_pieces():
    """Fewer output rows than the limit, but with the prefix's pieces more workgroups of 512 threads."""
    a = attn(batch=32768, q_heads=255, kv_heads=255, own_capacity=1, workspace_bytes=1 << 50)
    assert status(pyq35.lib.q35_attn_batch, a) == UNSUPPORTED
