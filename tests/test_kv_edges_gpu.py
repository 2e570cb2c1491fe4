"""Calls on the paged cache that its documentation allows at its edges: places
past 32 bits, outputs over the queries, streams given by handle, block tables
and row lists that a caller got wrong."""
import pytest
import torch

from inferq_b200 import _lib
from inferq_b200.kv import KvBatch, KvCache
from test_kv_gpu import Sequences, close, held

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("fmt,page,pages", [("i8", 64, 140000), ("f16", 128, 36000)])
def test_pages_past_32_bits(cuda, fmt, page, pages):
    """4.6 GB of keys and as many values: what the last pages hold and what
    attention over them gives is, bit for bit, that of the first ones."""
    cache = KvCache(2, 256, pages, page_tokens=page, format=fmt)
    assert cache.nbytes > 2 << 32
    n = 5 * page + 3
    k, v = (torch.randn(n, 2, 256, device="cuda") for _ in range(2))
    low = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    got = []
    for table in (low, pages - 1 - low):
        cache.append(k, v, KvBatch(table, ints(0)))
        held_k, held_v = cache.read(KvBatch(table, ints(0)), rows=n)
        rows = [held_k, held_v]
        for r in (1, 4, 70):
            for dt in (torch.float32, torch.bfloat16):
                q = torch.randn(r, 16, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(r)).to(dt)
                rows.append(cache.attend(q, KvBatch(table, ints(n - r))))
        got.append(rows)
    assert torch.equal(got[0][0].cpu().double(), held(k, fmt)) or torch.allclose(got[0][0].cpu().double(), held(k, fmt), rtol=2.0 ** -23, atol=0)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    cache.status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "f16"])
@pytest.mark.parametrize("rows,chunk", [(1, 0), (1, 1024), (1, 64), (6, 0), (6, 128), (75, 0), (75, 1024)])
def test_outputs_over_the_queries(cuda, fmt, dtype, rows, chunk):
    s = Sequences([(rows, 600 - rows), (rows, 333)], fmt=fmt, dtype=dtype)
    q = s.q.cuda()
    want = s.cache.attend(q, s.batch(), chunk=chunk)
    assert s.cache.attend(q, s.batch(), chunk=chunk, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("rows", [1, 5, 70])
def test_scores_scaled_below_zero(cuda, rows):
    s = Sequences([(rows, 200)], fmt="f16", hd=128)
    want, most = s.want(scale=-0.07)
    close(s.cache.attend(s.q.cuda(), s.batch(), scale=-0.07), want, most, s.dt)


def test_results_of_a_stream_given_by_handle(cuda):
    s = Sequences([(3, 900), (3, 1200)])
    q, b = s.q.cuda(), s.batch()
    want, kept = s.cache.attend(q, b), s.cache.read(b, rows=s.rows)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        out = s.cache.attend(q, b, stream=side.cuda_stream)
        k, v = s.cache.read(b, rows=s.rows, stream=side.cuda_stream)
        side.synchronize()
        twice = out + out, k + k, v + v  # work of the current stream, the tensors freed before it ran
        del out, k, v
        assert all(torch.equal(t, w + w) for t, w in zip(twice, (want, *kept)))
    out = s.cache.attend(q, b, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("starts", [(4, 2, 6), (0, 9, 6), (-3, 2, 6), (0, 2**31 - 1, 6), (6, 6, 6), (-2**31, 2**31 - 1, 2**31 - 1),
                                    (2**31 - 1, -2**31, 6)])
@pytest.mark.parametrize("max_rows", [1, 3, 70])
@pytest.mark.parametrize("heads", [16, 14])
def test_row_lists_that_do_not_ascend_touch_nothing_else(cuda, starts, max_rows, heads):
    """Which rows such a list names is undefined; the rows around the call's stay as they were."""
    s = Sequences([(3, 100), (3, 200)], heads=heads)
    b = KvBatch(s.table, s.position, ints(*starts), max_rows=max_rows)
    around = torch.full((s.rows + 400, heads, 256), 7.0, device="cuda")
    out = around[200:200 + s.rows]
    s.cache.attend(s.q.cuda(), b, out=out)
    kv = torch.full((2, s.rows + 400, 2, 256), 7.0, device="cuda")
    s.cache.read(b, rows=s.rows, out=(kv[0, 200:200 + s.rows], kv[1, 200:200 + s.rows]))
    torch.cuda.synchronize()
    assert (around[:200] == 7).all() and (around[200 + s.rows:] == 7).all()
    assert (kv[:, :200] == 7).all() and (kv[:, 200 + s.rows:] == 7).all()


def test_one_place_for_keys_and_values_is_refused(cuda):
    s = Sequences([(2, 10)])
    k = torch.zeros(2, 2, 256, device="cuda")
    with pytest.raises(_lib.IqError, match="one place"):
        s.cache.read(s.batch(), rows=2, out=(k, k))
    with pytest.raises(_lib.IqError, match="too large"):
        s.cache.attend(s.q.cuda(), s.batch(), scale=3e38)


@pytest.mark.parametrize("rows", [1, 5, 70])
@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("f16", "bf16")])
def test_windows_first_tokens_and_splits_past_any_table(cuda, rows, fmt, dtype):
    """Up to the types' ends: all of them mean the whole context, padding before it included."""
    most = 2**31 - 1
    s = Sequences([(rows, 300), (rows, -2 if rows > 1 else 9), (rows, 128)], fmt=fmt, dtype=dtype)
    q, b = s.q.cuda(), s.batch()
    want = s.cache.attend(q, b, chunk=1024)
    for window, sinks in ((most, 0), (most, most), (1, most), (most, 1), (5, most - 63)):
        for chunk in (1024, most - 63):
            got = s.cache.attend(q, b, window=window, sinks=sinks, chunk=chunk)
            assert torch.equal(got, want), (window, sinks, chunk)
        close(s.cache.attend(q, b, window=window, sinks=sinks), *s.want(), s.dt)
    for chunk in (64, most - 63):
        close(s.cache.attend(q, b, window=7, sinks=0, chunk=chunk), *s.want(window=7), s.dt)
    s.cache.status()


@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (8, 2, 64), (16, 2, 256)])
@pytest.mark.parametrize("fmt,dtype", [("f16", "f16"), ("i8", "f32"), ("i8", "bf16")])
def test_cold_and_warm_calls_agree(cuda, heads, kv_heads, hd, fmt, dtype):
    """Bit for bit, whatever order copies and warps happen to run in: caches emptied before every call."""
    s = Sequences([(300, 3000), (41, 700), (90, 60)], heads=heads, kv_heads=kv_heads, hd=hd, fmt=fmt, dtype=dtype)
    q, b = s.q.cuda(), s.batch()
    flush = torch.empty(200 << 20, dtype=torch.uint8, device="cuda")
    for kw in ({}, {"window": 1023, "sinks": 5}, {"chunk": 512}):
        want = s.cache.attend(q, b, **kw)
        for i in range(15):
            flush.fill_(i)
            assert torch.equal(s.cache.attend(q, b, **kw), want), (kw, i)
    s.cache.status()


@pytest.mark.parametrize("rows", [1, 4, 70])
@pytest.mark.parametrize("fmt", ["i8", "f16"])
def test_a_bad_page_id_is_the_matter_of_the_rows_that_see_it(cuda, fmt, rows):
    s = Sequences([(rows, 30), (rows, 300)], fmt=fmt, page=64)
    q, b = s.q.cuda(), s.batch()
    want = s.cache.attend(q, b)
    s.table[1, 3] = 2**31 - 1
    got = s.cache.attend(q, b)
    with pytest.raises(_lib.IqError, match="pool"):
        s.cache.status()
    assert torch.equal(got[:rows], want[:rows])
    s.table[1, 3] = -7
    s.cache.attend(q, b)
    with pytest.raises(_lib.IqError, match="pool"):
        s.cache.status()
    s.cache.status()
