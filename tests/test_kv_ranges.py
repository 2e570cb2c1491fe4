"""Integers that do not fit the C ABI's fields are refused; their low bits
would mean something else (a window of 2^32 + 5 positions: one of 5)."""
import pytest
import torch

from inferq_b200.kv import KvBatch, KvCache
from inferq_b200.model import State


@pytest.mark.parametrize("args,kw", [((2**32 + 2, 64, 4), {}), ((2, 2**32 + 64, 4), {}), ((2, 64, 2**64 + 4), {}),
                                     ((2, 64, 4), {"page_tokens": 2**32 + 64})])
def test_caches(args, kw):
    with pytest.raises(ValueError, match="out of range"):
        KvCache(*args, **kw)


def test_states():
    for args, kw in (((2**64 + 16,), {}), ((16,), {"window": 2**32 + 5}), ((16,), {"window": 4, "sinks": 2**32})):
        with pytest.raises(ValueError, match="out of range"):
            State(None, *args, kv="i8", **kw)


@pytest.mark.gpu
def test_calls(cuda):
    cache = KvCache(1, 64, 4)
    table, position = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="out of range"):
        KvBatch(table, position, max_rows=2**32)
    q = torch.ones(1, 8, 64, device="cuda")
    for kw in ({"window": 2**32 + 5}, {"window": 4, "sinks": 2**32}, {"chunk": 2**32 + 64}):
        for _ in range(2):
            with pytest.raises(ValueError, match="out of range"):
                cache.attend(q, KvBatch(table, position), **kw)
