"""What a cache and a batch keep, and for how long."""
import os
import subprocess
import sys

import pytest
import torch

from inferq_b200.kv import KvBatch, KvCache
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


def test_a_call_on_a_stream_given_by_handle_holds_its_tensors(cuda):
    """Keys, queries and the batch are let go while the stream is still busy with earlier work, and their memory is
    asked for again."""
    s = Sequences([(300, 0)], heads=8, hd=64, kv_heads=1)
    k, v = s.cache.read(s.all, rows=300)
    want = s.cache.attend(s.q.cuda(), s.batch())
    side = torch.cuda.Stream()
    for _ in range(3):
        s.cache.append(torch.zeros_like(k), torch.zeros_like(v), s.all)
        out = torch.empty_like(want)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        q, table, position = s.q.cuda(), s.table.clone(), s.position.clone()
        a, b = k.clone(), v.clone()
        torch.cuda.current_stream().synchronize()
        s.cache.append(a, b, KvBatch(table, position), stream=side.cuda_stream)
        s.cache.attend(q, KvBatch(table, position), out=out, stream=side.cuda_stream)
        shapes = [x.shape for x in (q, a, b, table, position)]
        types = [x.dtype for x in (q, a, b, table, position)]
        del q, a, b, table, position
        for _ in range(3):
            again = [torch.full(shape, 1, dtype=dt, device="cuda") for shape, dt in zip(shapes, types)]
        torch.cuda.synchronize()
        del again
        assert torch.equal(s.cache.read(s.all, rows=300)[0], k)
        assert torch.equal(out, want)
    s.cache.status()


def test_a_cache_let_go_under_capture_is_freed_later(cuda):
    s, lone = Sequences([(2, 60)], heads=8, hd=64, kv_heads=1), KvCache(1, 64, 1000)
    q, b = s.q.cuda(), s.batch()
    want = s.cache.attend(q, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        del lone
        out = s.cache.attend(q, b)
    graph.replay()
    assert torch.equal(out, want)
    free = torch.cuda.mem_get_info()[0]
    del graph, out
    KvCache(1, 64, 1)
    assert torch.cuda.mem_get_info()[0] >= free + 1000 * 64 * 64 * 2
    s.cache.status()


CHILD = r"""
import builtins
import sys
import torch
from inferq_b200.kv import KvCache
cache, builtins.kept, sys.kept = (KvCache(1, 64, 4) for _ in range(3))
cache.cycle = cache, torch
print(cache.nbytes)
"""


def test_a_cache_may_outlive_the_program(cuda):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and not r.stderr, r.stderr
