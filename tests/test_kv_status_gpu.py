"""iq_kv_status reports everything that calls on a cache met, from whichever
stream: two kinds at once, and what arrives while another report is taken."""
import random

import pytest
import torch

from inferq_b200 import _lib
from inferq_b200.kv import KvBatch
from test_kv_gpu import Sequences

pytestmark = pytest.mark.gpu


def told(cache, stream):
    try:
        cache.status(stream=stream)
        return ""
    except _lib.IqError as e:
        return str(e)


def test_no_report_is_lost_between_two(cuda, monkeypatch):
    s = Sequences([(1, 40)], heads=8, hd=64, kv_heads=1)
    q, k, b = s.q.cuda(), s.k[:1].cuda(), s.batch()
    bad = KvBatch(torch.full_like(s.table, 2 ** 30), s.position)
    a, other = torch.cuda.Stream(), torch.cuda.Stream()

    def gives_up():
        monkeypatch.setenv("IQ_KV_TEST_TIMEOUT", "1")
        s.cache.attend(q, b)
        monkeypatch.delenv("IQ_KV_TEST_TIMEOUT")
        torch.cuda.synchronize()

    gives_up()
    s.cache.append(k, k, bad)
    both = told(s.cache, 0)
    assert "gave up" in both and "pool" in both
    assert not told(s.cache, 0)
    r = random.Random(0)
    for _ in range(60):  # a bad page of the other stream somewhere around the report of the wait
        gives_up()
        with torch.cuda.stream(other):
            torch.cuda._sleep(r.randrange(1000, 150000))
            s.cache.append(k, k, bad)
        first = told(s.cache, a.cuda_stream)
        assert "gave up" in first
        torch.cuda.synchronize()
        assert ("pool" in first) != ("pool" in told(s.cache, a.cuda_stream))


def test_many_reports_at_once(cuda):
    from concurrent.futures import ThreadPoolExecutor

    s = Sequences([(1, 40)], heads=8, hd=64, kv_heads=1)
    streams = [torch.cuda.Stream() for _ in range(8)]
    with ThreadPoolExecutor(8) as pool:
        assert not any(pool.map(lambda i: told(s.cache, streams[i % 8].cuda_stream), range(400)))
        bad = KvBatch(torch.full_like(s.table, -1), s.position)
        s.cache.append(s.k[:1].cuda(), s.k[:1].cuda(), bad)
        torch.cuda.synchronize()
        got = list(pool.map(lambda i: told(s.cache, streams[i % 8].cuda_stream), range(400)))
    assert sum("pool" in g for g in got) == 1
