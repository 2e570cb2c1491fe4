"""The paged key/value cache and the attention over it, against their
definitions in 64 bits on the CPU.

Tolerances.  With V the largest visible |value| of a row, an output element is
off by at most
  * the output type's rounding, eps / 2 of it;
  * 16-bit types: the weights' rounding to f16, 2^-11 of each, so 2^-11 V; 32
    bits: two parts, 2^-22 V;
  * what the f32 scores and sums carry: a score of D products in D / 16
    matrix instructions (twice that with two parts), each rounding (or cutting
    off) at most 2^-22 of the sum of magnitudes S = sum |q k| scale (below 30
    for these inputs), moves a weight by at most 2^-22 * D / 8 * S: 2^-22 * 32 *
    30 < 2^-12; the value sums over T / 16 instructions (T < 1500) at most
    2^-22 * 94 < 2^-15.  Together below 2^-11.8 V.
Such errors have no common direction, so over all outputs of a case the root
mean square stays far lower: 32 bits are held to 2^-17 of the outputs' own,
16 bits to 2^-11 (weights, keys of 2^-12) plus the type's eps / 2.
"""
import math

import numpy as np
import pytest
import torch

from inferq_b200 import _lib
from inferq_b200.kv import KvBatch, KvCache

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def held(x, fmt):
    """The values that the cache stands for, in 64 bits (NaN for a vector that is not finite)."""
    x = x.detach().cpu().double()
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "i8":
        scale = (top.float() / 127).double()
        v = torch.where(top > 0, torch.round(127 * x / top) * scale, 0.0)
    else:
        e = torch.where(top > 0, torch.frexp(top).exponent.double() - 15, 0.0)
        scale = torch.exp2(e.clamp(min=-126))
        v = (x / scale).float().half().double() * scale
    return torch.where(torch.isfinite(x).all(-1, keepdim=True), v, float("nan"))


class Sequences:
    """A cache with sequences of `lens` = [(new rows, position of the first new row)], pages in random order; every token
    up to the last new row is written."""

    def __init__(self, lens, *, heads=16, kv_heads=2, hd=256, fmt="i8", dtype="f32", page=64, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.hd, self.fmt, self.dt, self.page = lens, heads, kv_heads, hd, fmt, DT[dtype], page
        self.ctx = [max(0, p + n) for n, p in lens]
        counts = [-(-c // page) for c in self.ctx]
        cols = max(max(counts), 1)
        pages = sum(counts) + 2
        order = torch.randperm(pages, generator=g)
        table, at = torch.full((len(lens), cols), pages - 1), 0
        for s, n in enumerate(counts):
            table[s, :n] = order[at:at + n]
            at += n
        self.table = table.to(torch.int32).cuda()
        self.position = torch.tensor([p for _, p in lens], dtype=torch.int32).cuda()
        starts = np.cumsum([0] + [n for n, _ in lens])
        self.rows = int(starts[-1])
        self.row_start = torch.tensor(starts, dtype=torch.int32).cuda()
        every = np.cumsum([0] + self.ctx)
        self.k = (torch.randn(int(every[-1]), kv_heads, hd, generator=g) * spread).to(self.dt)
        self.v = (torch.randn(int(every[-1]), kv_heads, hd, generator=g) *
                  torch.exp(0.7 * torch.randn(int(every[-1]), 1, 1, generator=g))).to(self.dt)
        self.q = (1.2 * torch.randn(self.rows, heads, hd, generator=g)).to(self.dt)
        self.begin = every
        self.starts = starts
        self.cache = KvCache(kv_heads, hd, pages, page_tokens=page, format=fmt)
        self.all = KvBatch(self.table, torch.zeros_like(self.position), torch.tensor(every, dtype=torch.int32).cuda(),
                           max_rows=max(self.ctx))
        if every[-1]:
            self.cache.append(self.k.cuda(), self.v.cuda(), self.all)

    def batch(self, max_rows=None):
        m = max((n for n, _ in self.lens), default=0)
        return KvBatch(self.table, self.position, self.row_start, max_rows=m if max_rows is None else max_rows)

    def want(self, window=0, sinks=0, scale=None):
        """(outputs, largest visible |value| of each row and head) in 64 bits."""
        out = torch.zeros(self.rows, self.heads, self.hd, dtype=torch.float64)
        most = torch.zeros(self.rows, self.heads, 1, dtype=torch.float64)
        group = self.heads // self.kv_heads
        for (n, p), b, c, r in zip(self.lens, self.begin, self.ctx, self.starts):
            k, v = held(self.k[b:b + c], self.fmt), held(self.v[b:b + c], self.fmt)
            for i in range(n):
                t = torch.arange(c)
                seen = t <= p + i
                if window:
                    seen &= (t > p + i - window) | (t < sinks)
                if not seen.any():
                    continue
                ks, vs = k[seen], v[seen]
                for h in range(self.heads):
                    s = ks[:, h // group] @ self.q[r + i, h].double() * (scale or 1 / math.sqrt(self.hd))
                    out[r + i, h] = torch.softmax(s, 0) @ vs[:, h // group]
                    most[r + i, h] = vs[:, h // group].abs().max()
        return out, most


def close(got, want, most, dt, note=""):
    got, eps = got.detach().cpu().double(), torch.finfo(dt).eps
    off = (got - want).abs()
    part = 2.0 ** -22 if dt == torch.float32 else 2.0 ** -11
    bound = want.abs() * eps / 2 + most * (part + 2.0 ** -11.8)
    worst = (off - bound).max() if off.numel() else torch.tensor(-1.0)
    assert worst <= 0, (note, float(worst), float(off.max()))
    rms = want.square().mean().sqrt()
    limit = 2.0 ** -17 if dt == torch.float32 else 2.0 ** -11 + eps / 2
    assert not off.numel() or off.square().mean().sqrt() <= limit * rms, (note, float(off.square().mean().sqrt() / rms))


# ------------------------------------------------------------ write and read back
@pytest.mark.parametrize("fmt", ["i8", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kv_heads,hd,page", [(2, 256, 64), (1, 64, 16), (3, 128, 256), (5, 64, 32), (2, 128, 128)])
def test_rows_read_back_as_their_definition(cuda, fmt, dtype, kv_heads, hd, page):
    s = Sequences([(3, 0), (0, 5), (130, 61), (1, 15)], heads=kv_heads, kv_heads=kv_heads, hd=hd, fmt=fmt, dtype=dtype, page=page)
    n = int(s.begin[-1])
    k, v = s.cache.read(s.all, rows=n)
    for got, x in ((k, s.k), (v, s.v)):
        assert torch.equal(got.cpu(), held(x, fmt).float())  # f32: the product of code and scale, rounded once
    for dt in (torch.float16, torch.bfloat16):
        k2, _ = s.cache.read(s.all, rows=n, dtype=dt)
        assert torch.equal(k2, k.to(dt))
    s.cache.status()


@pytest.mark.parametrize("fmt", ["i8", "f16"])
def test_borders_extremes_and_non_finite_vectors(cuda, fmt):
    hd, kvh = 128, 1
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, kvh, hd, generator=g)
    x[0] = 0
    x[1] *= 1e-44          # below f32's normals
    x[2] *= 1e-30
    x[3] *= 3e37           # amax near the largest
    x[4, 0, 5] = float("inf")
    x[5, 0, 9] = float("nan")
    x[6] = -x[6].abs()
    # exact ties between two codes: (n + 1/2) / 127 of the maximum, and their neighbours
    x[7, 0] = torch.arange(hd) + 0.5
    x[7, 0, 127] = 127.0
    x[8] = torch.nextafter(x[7], torch.tensor(0.0))
    x[9] = torch.nextafter(x[7], torch.tensor(1e9))
    x[8, 0, 127] = x[9, 0, 127] = 127.0
    x[10] = torch.exp2(torch.randint(-60, 60, (1, hd), generator=g).float())
    if fmt == "i8":
        x[11] = x[10] * 1.9999999
    cache = KvCache(kvh, hd, 4, page_tokens=16, format=fmt)
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32).cuda()
    b = KvBatch(table, torch.zeros(1, dtype=torch.int32).cuda())
    cache.append(x.cuda(), (-x).cuda(), b)
    k, v = cache.read(b, rows=64)
    want = held(x, fmt)
    if fmt == "i8":  # the scale of a vector below the normals is rounded to its grid: codes are what is held
        want[1] = torch.round(127 * x[1].double() / x[1].double().abs().max()) * (x[1].abs().max() / 127).double()
    assert torch.equal(torch.nan_to_num(k.cpu(), nan=7.0), torch.nan_to_num(want.float(), nan=7.0))
    assert torch.equal(torch.nan_to_num(v.cpu(), nan=7.0), torch.nan_to_num(-want.float(), nan=-7.0).where(~want.isnan(), torch.tensor(7.0)))
    # what is read back in f32 is written again to the same values
    again = KvCache(kvh, hd, 4, page_tokens=16, format=fmt)
    again.append(k, v, b)
    k2, v2 = again.read(b, rows=64)
    assert torch.equal(torch.nan_to_num(k2, nan=7.0), torch.nan_to_num(k, nan=7.0))
    assert torch.equal(torch.nan_to_num(v2, nan=7.0), torch.nan_to_num(v, nan=7.0))


@pytest.mark.parametrize("fmt", ["i8", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_offsets_and_rows_behind_the_last_sequence(cuda, fmt, dtype):
    dt, hd, kvh = DT[dtype], 64, 2
    big = torch.randn(40, 3 * kvh * hd + 5, device="cuda").to(dt)
    views = [big[:, 1:1 + kvh * hd].unflatten(1, (kvh, hd)),                       # off any 16-byte border
             big[:, 8:8 + 2 * kvh * hd].unflatten(1, (kvh, 2 * hd))[:, :, :hd],    # heads with something between
             torch.randn(kvh, 40, hd, device="cuda").to(dt).transpose(0, 1)]       # heads outermost
    table = torch.tensor([[1, 0], [3, 2]], dtype=torch.int32).cuda()
    b = KvBatch(table, torch.tensor([0, -2], dtype=torch.int32).cuda(), torch.tensor([0, 17, 30], dtype=torch.int32).cuda())
    for x in views:
        cache = KvCache(kvh, hd, 4, page_tokens=32, format=fmt)
        cache.append(x, x, b)
        for out in (torch.full((40, kvh, hd), 5.0, device="cuda"), torch.full((kvh, 40, hd), 5.0, device="cuda").transpose(0, 1),
                    torch.full((40, 2 * kvh * hd + 1), 5.0, device="cuda")[:, 1:].unflatten(1, (kvh, 2 * hd))[:, :, :hd]):
            k, v = cache.read(b, rows=40, out=(out, torch.full_like(out, 5.0)))
            want = held(x, fmt).float()
            want[17:19] = 0   # padding: negative positions
            want[30:] = 5     # behind the last sequence: as they were
            assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
        cache.status()


def test_no_rows_and_no_sequences(cuda):
    cache = KvCache(2, 64, 2)
    none = torch.zeros(0, 2, 64, device="cuda")
    t, p = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    b = KvBatch(t, p)
    cache.append(none, none, b)
    assert cache.attend(none, b).shape == (0, 2, 64) and cache.read(b, rows=0)[0].shape == (0, 2, 64)
    empty = KvBatch(t[:0], p[:0], torch.zeros(1, dtype=torch.int32, device="cuda"))
    x = torch.ones(3, 2, 64, device="cuda")
    cache.append(x, x, empty)
    out = torch.full_like(x, 2.0)
    assert torch.equal(cache.attend(x, empty, out=out), torch.full_like(x, 2.0))
    cache.status()


def test_what_only_the_device_sees_is_reported_and_skipped(cuda):
    cache = KvCache(1, 64, 4, page_tokens=16, format="i8")
    x = torch.randn(20, 1, 64, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    for table, why in (([[0, 4]], "pool"), ([[0, -1]], "pool"), ([[0]], "table"), ([[0, 2 ** 31 - 1]], "pool")):
        b = KvBatch(torch.tensor(table, dtype=torch.int32).cuda(), zero)
        cache.append(x, x, b)
        with pytest.raises(_lib.IqError) as e:
            cache.status()
        assert e.value.code == -1 and why in str(e.value)
        k, _ = cache.read(b, rows=20)
        assert torch.equal(k[:16].cpu(), held(x[:16], "i8").float()) and not k[16:].any()
        with pytest.raises(_lib.IqError):
            cache.status()
        cache.attend(x, b)
        with pytest.raises(_lib.IqError):
            cache.status()
        cache.status()  # reported once


# ------------------------------------------------------------------- attention
GEOMETRIES = [(16, 2, 256, 64), (8, 2, 64, 16), (7, 1, 128, 32), (4, 4, 64, 128), (6, 2, 256, 256), (24, 1, 128, 64)]


@pytest.mark.parametrize("fmt", ["i8", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,hd,page", GEOMETRIES)
def test_single_tokens_and_short_rows(cuda, fmt, dtype, heads, kv_heads, hd, page):
    s = Sequences([(1, 0), (1, 63), (1, 64), (1, 700), (1, 15), (1, 128)], heads=heads, kv_heads=kv_heads, hd=hd, fmt=fmt,
                  dtype=dtype, page=page, seed=hd + heads)
    want, most = s.want()
    for chunk in (0, 64, 256):
        close(s.cache.attend(s.q.cuda(), s.batch(), chunk=chunk), want, most, s.dt, chunk)
    s = Sequences([(3, 0), (0, 7), (8, 60), (1, 299), (5, 1000)], heads=heads, kv_heads=kv_heads, hd=hd, fmt=fmt, dtype=dtype,
                  page=page, seed=hd)
    want, most = s.want()
    for max_rows in (0, 1, 2, 3, 8):  # a hint: each kernel is right for any rows
        close(s.cache.attend(s.q.cuda(), s.batch(max_rows)), want, most, s.dt, max_rows)
    s.cache.status()


@pytest.mark.parametrize("fmt,dtype,heads,kv_heads,hd,page", [
    ("i8", "f32", 16, 2, 256, 64), ("f16", "f32", 16, 2, 256, 16), ("i8", "bf16", 16, 2, 256, 32), ("f16", "f16", 16, 2, 256, 128),
    ("i8", "f16", 8, 2, 64, 16), ("f16", "bf16", 8, 2, 64, 64), ("i8", "bf16", 7, 1, 128, 32), ("f16", "f32", 6, 3, 128, 256),
    ("i8", "f32", 5, 5, 64, 64), ("f16", "bf16", 20, 1, 128, 16), ("f16", "f32", 12, 4, 64, 32), ("i8", "f32", 4, 1, 128, 128),
])
def test_chunks_of_rows(cuda, fmt, dtype, heads, kv_heads, hd, page):
    lens = [(64, 0), (130, 77), (1, 400), (0, 3), (17, 1003), (129, 0)]
    s = Sequences(lens, heads=heads, kv_heads=kv_heads, hd=hd, fmt=fmt, dtype=dtype, page=page, seed=heads * hd)
    want, most = s.want()
    for chunk in (0, 128, 1 << 12):
        close(s.cache.attend(s.q.cuda(), s.batch(), chunk=chunk), want, most, s.dt, chunk)
    s.cache.status()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (64, 0), (65, 64), (200, 63), (300, 500), (127, 129), (5000, 4)])
@pytest.mark.parametrize("fmt,dtype,heads,hd", [("i8", "f32", 16, 256), ("f16", "bf16", 14, 64)])
def test_windows_and_first_tokens(cuda, window, sinks, fmt, dtype, heads, hd):
    for lens in ([(1, 0), (1, 511), (4, 620), (3, 62)], [(150, 0), (70, 517), (1, 5)]):
        s = Sequences(lens, heads=heads, hd=hd, fmt=fmt, dtype=dtype, page=32, seed=window)
        want, most = s.want(window, sinks)
        for chunk in (0, 64, 192):
            close(s.cache.attend(s.q.cuda(), s.batch(), window=window, sinks=sinks, chunk=chunk), want, most, s.dt, chunk)
        s.cache.status()


@pytest.mark.parametrize("fmt", ["i8", "f16"])
def test_rows_that_see_nothing_are_zeros(cuda, fmt):
    s = Sequences([(5, -3), (2, -2), (100, -40)], fmt=fmt)
    want, most = s.want()
    for chunk in (0, 64):
        for mr in (0, 2):
            got = s.cache.attend(s.q.cuda(), s.batch(mr), chunk=chunk)
            close(got, want, most, s.dt)
            assert not got[:3].any() and not got[5:7].any() and not got[7:47].any()
    s.cache.status()


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("fmt", ["i8", "f16"])
def test_scales_of_any_magnitude(cuda, fmt, rows):
    """Weights are rounded relative to the largest value scale met so far: keys, values and queries over many binades."""
    s = Sequences([(rows, 333)], heads=8, kv_heads=1, hd=64, fmt=fmt, dtype="f32")
    n = s.k.shape[0]
    factor = torch.exp2(torch.linspace(-40, 30, n).round())[:, None, None]
    for f in (factor, factor.flip(0), torch.full_like(factor, 2.0 ** -90), torch.full_like(factor, 2.0 ** 60)):
        s.v = torch.randn(n, 1, 64, generator=torch.Generator().manual_seed(1)) * f
        s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
        want, most = s.want()
        close(s.cache.attend(s.q.cuda(), s.batch()), want, most, s.dt)
    s.v = torch.randn(n, 1, 64, generator=torch.Generator().manual_seed(1))
    s.k, s.q = s.k * 2.0 ** 50, s.q * 2.0 ** -50
    s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
    want, most = s.want()
    close(s.cache.attend(s.q.cuda(), s.batch()), want, most, s.dt)


@pytest.mark.parametrize("rows", [2, 70])
@pytest.mark.parametrize("fmt", ["i8", "f16"])
def test_nan_and_infinity_stay_with_the_rows_that_see_them(cuda, fmt, rows):
    s = Sequences([(rows, 200), (rows, 90)], fmt=fmt, heads=8, kv_heads=1, hd=64)
    clean = s.cache.attend(s.q.cuda(), s.batch())
    bad = 200 + rows - 1  # the last token of the first sequence: its last row sees it, no other
    for where, value in ((s.v, float("nan")), (s.v, float("inf")), (s.k, float("nan")), (s.k, float("-inf"))):
        keep = where[bad].clone()
        where[bad, 0, 3] = value
        s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
        got = s.cache.attend(s.q.cuda(), s.batch())
        assert got[rows - 1].isnan().all()
        rest = [i for i in range(2 * rows) if i != rows - 1]
        assert torch.equal(got[rest], clean[rest])
        # a window hides it from everyone: tokens behind the window, NaN or not, weigh nothing
        where[bad] = keep
        where[3, 0, 0] = value
        s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
        got = s.cache.attend(s.q.cuda(), s.batch(), window=50, sinks=2)
        assert got[:rows].isfinite().all()
        where[3, 0, 0] = 0.25
        s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
        clean = s.cache.attend(s.q.cuda(), s.batch())
    q = s.q.clone()
    q[0, 0, 0], q[1, 2, 5] = float("nan"), float("inf")
    got = s.cache.attend(q.cuda(), s.batch())
    assert got[0, 0].isnan().all() and got[1, 2].isnan().any()
    ok = torch.ones(2 * rows, 8, dtype=torch.bool)
    ok[0, 0] = ok[1, 2] = False
    assert torch.equal(got.cpu()[ok], clean.cpu()[ok])


def test_a_short_row_group_is_the_same_alone_and_in_any_batch(cuda):
    """With a chunk given, a row of at most 64 query rows a KV head depends on its own context only, bit for bit."""
    for fmt, dtype, window, sinks in (("i8", "f32", 0, 0), ("f16", "bf16", 0, 0), ("i8", "f32", 333, 70)):
        s = Sequences([(8, 700), (5, 250), (1, 64), (8, 1018)], fmt=fmt, dtype=dtype, page=32)
        q = s.q.cuda()
        all_ = s.cache.attend(q, s.batch(8), chunk=256, window=window, sinks=sinks)
        for seq, (n, p) in enumerate(s.lens):
            r = int(s.starts[seq])
            for k in range(1, n + 1):  # the first k rows alone, and each row alone
                b = KvBatch(s.table[seq:seq + 1], s.position[seq:seq + 1])
                assert torch.equal(s.cache.attend(q[r:r + k], b, chunk=256, window=window, sinks=sinks), all_[r:r + k])
                one = KvBatch(s.table[seq:seq + 1], s.position[seq:seq + 1] + (k - 1))
                assert torch.equal(s.cache.attend(q[r + k - 1:r + k], one, chunk=256, window=window, sinks=sinks),
                                   all_[r + k - 1:r + k])


def test_growing_sequences_with_shared_pages_as_a_server_runs_them(cuda):
    """Two sequences share a prompt's pages; a chunked prefill, then single tokens, then four rows at a time: every step
    appends and attends, and all of it equals the definition over the whole history."""
    page, hd, heads, kvh = 16, 64, 8, 2
    g = torch.Generator().manual_seed(5)
    cache = KvCache(kvh, hd, 40, page_tokens=page, format="i8")
    prompt = 3 * page
    tables = torch.zeros(2, 12, dtype=torch.int32)
    tables[0] = torch.arange(12)
    tables[1, :3], tables[1, 3:] = tables[0, :3], torch.arange(20, 29)
    tables = tables.cuda()
    hist = [[torch.empty(0, kvh, hd)] * 2 for _ in range(2)]

    def step(lens):  # [(sequence's new rows)] at the sequences' ends
        pos = torch.tensor([len(h[0]) for h in hist], dtype=torch.int32)
        rs = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32)
        n = int(rs[-1])
        k, v, q = torch.randn(n, kvh, hd, generator=g), torch.randn(n, kvh, hd, generator=g), torch.randn(n, heads, hd, generator=g)
        b = KvBatch(tables, pos.cuda(), rs.cuda(), max_rows=max(lens))
        cache.append(k.cuda(), v.cuda(), b)
        out = cache.attend(q.cuda(), b).cpu().double()
        for s in range(2):
            a, e = int(rs[s]), int(rs[s + 1])
            hist[s] = [torch.cat([hist[s][0], k[a:e]]), torch.cat([hist[s][1], v[a:e]])]
            hk, hv = held(hist[s][0], "i8"), held(hist[s][1], "i8")
            for i in range(a, e):
                t = int(pos[s]) + i - a + 1
                for h in range(heads):
                    w = torch.softmax(hk[:t, h // 4] @ q[i, h].double() / 8, 0)
                    assert ((w @ hv[:t, h // 4]) - out[i, h]).abs().max() < 2.0 ** -11.8 * float(hv[:t].abs().max())

    # the prompt enters once, for sequence 0; sequence 1 takes over its pages
    step([prompt, 0])
    hist[1] = list(hist[0])
    step([21, 33])
    for _ in range(3):
        step([1, 1])
    step([4, 2])
    step([0, 4])
    cache.status()


# --------------------------------------------------- streams, graphs, refusals
def test_another_stream_and_two_calls_at_once(cuda):
    s = Sequences([(1, 900), (1, 1200), (1, 30)])
    q = s.q.cuda()
    want = s.cache.attend(q, s.batch())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for rep in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(s.cache.attend(q, s.batch()))
    raw = torch.cuda.Stream()
    outs.append(s.cache.attend(q, s.batch(), stream=raw.cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_captured_steps_replay_with_new_positions_and_tables(cuda):
    s = Sequences([(1, 500), (1, 90)], page=32)
    q, k, v = s.q.cuda(), torch.randn(2, 2, 256, device="cuda"), torch.randn(2, 2, 256, device="cuda")
    b = s.batch()

    def step():
        s.cache.append(k, v, b)
        return s.cache.attend(q, b), s.cache.attend(q, b, window=100, sinks=4)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same call: each has its workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for i in range(3):
        s.position += -7 if i else 0
        k.normal_()
        q.normal_()
        want = step()
        for gr, out in graphs:
            out[0].zero_()
            gr.replay()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    s.table.copy_(s.table.flip(0))
    s.position.copy_(torch.tensor([60, 90], dtype=torch.int32))
    want = step()
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1][0], want[0])
    s.cache.status()


def test_refusals(cuda):
    s = Sequences([(2, 100)])
    q, b = s.q.cuda(), s.batch()
    for kw, text in (({"window": -1}, "negative"), ({"sinks": -1, "window": 4}, "negative"), ({"chunk": 100}, "multiple of 64"),
                     ({"chunk": -64}, "multiple of 64"), ({"scale": float("nan")}, "finite"), ({"scale": float("inf")}, "finite")):
        with pytest.raises(_lib.IqError, match=text):
            s.cache.attend(q, b, **kw)
    with pytest.raises(_lib.IqError, match="query heads"):
        s.cache.attend(q[:, :3], b)
    with pytest.raises(_lib.IqError, match="on one another"):
        s.cache.attend(q, b, out=torch.empty(2, 1, 256, device="cuda").expand(2, 16, 256))
    for bad in (q.double(), q[:, :, :128], q.cpu(), q.transpose(1, 2)):
        with pytest.raises(ValueError):
            s.cache.attend(bad, b)
    k = torch.zeros(2, 2, 256, device="cuda")
    with pytest.raises(ValueError):
        s.cache.append(k, k.half(), b)
    with pytest.raises(ValueError):
        s.cache.append(k[:, :1], k[:, :1], b)
    with pytest.raises(_lib.IqError, match="on one another"):
        s.cache.read(b, rows=2, out=(k[:1].expand(2, 2, 256), k))
    t, p = s.table, s.position
    for args in ((t.long(), p), (t, p.long()), (t[0], p), (t, torch.cat([p, p])), (torch.cat([t, t]), torch.cat([p, p])),
                 (t, p, s.row_start[:1]), (t.expand(1, -1).t(), p)):
        with pytest.raises(ValueError):
            KvBatch(*args)
    with pytest.raises(_lib.IqError) as e:  # more than the GPU has
        KvCache(256, 256, 1 << 28)
    assert e.value.code == -3
    # a scale of one's own and a score scale below zero are fine
    for scale in (0.3, -0.1):
        want, most = s.want(scale=scale)
        close(s.cache.attend(q, b, scale=scale), want, most, s.dt)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_every_short_quotient_is_rounded_right(cuda, dtype):
    """Codes of 16-bit rows come from f32 quotients alone near a border: every significand of bf16 (a fourth of f16's)
    over every one of the maximum's, in the binades that reach a code."""
    dt, bits = DT[dtype], 8 if dtype == "bf16" else 11
    m = torch.arange(1 << (bits - 1), 1 << bits).double() / (1 << (bits - 1))
    x = torch.cat([m[::1 if bits == 8 else 4] * 2.0 ** -e for e in range(1, 9)]).to(dt)
    hd = 64
    x = x[: len(x) // 63 * 63].view(-1, 63)
    for top in m[::1 if bits == 8 else 37]:
        rows = torch.cat([torch.full((len(x), 1), float(top)).to(dt), x], 1).view(-1, 1, hd)
        n = rows.shape[0]
        cache = KvCache(1, hd, -(-n // 64), format="i8")
        b = KvBatch(torch.arange(-(-n // 64), dtype=torch.int32, device="cuda").view(1, -1), torch.zeros(1, dtype=torch.int32, device="cuda"))
        cache.append(rows.cuda(), rows.cuda(), b)
        k, _ = cache.read(b, rows=n)
        assert torch.equal(k.cpu(), held(rows, "i8").float())
