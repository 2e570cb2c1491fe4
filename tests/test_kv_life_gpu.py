"""What a cache and a batch keep, and for how long."""
import pytest
import torch

from test_kv_gpu import Sequences, close

pytestmark = pytest.mark.gpu


def test_calls_of_ever_new_arguments_keep_no_more_and_more(cuda):
    s = Sequences([(9, 600)], heads=8, hd=64, kv_heads=1)
    b = s.batch(0)
    whole = s.all
    q = s.q.cuda()
    for i in range(300):
        s.cache.attend(q[: 1 + i % 9], b, scale=0.1 + 0.001 * i)
        s.cache.read(whole, rows=i)
    assert len(s.cache._attn) <= 64 and len(b._of_rows) <= 64 and len(whole._of_rows) <= 64
    close(s.cache.attend(q, b, scale=0.1), *s.want(scale=0.1), s.dt)
    s.cache.status()
