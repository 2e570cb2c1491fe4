"""A row's attention depends on the tokens that it sees and on no others,
whatever finite values those hold: rows behind it in the same call, tokens
before its window.  Weights enter the matrix instructions as f16 over an
exponent above the value scales; here one hidden value is up to 2^100 times
the others', and scores are spread over some 15 nats, so that weights of every
size down to f16's smallest are met.

Tolerances are those of test_kv_gpu with the scores' part in proportion: a
score's error is 2^-22 of S = sum |q k| scale an instruction, at most |q| |k|
scale for S (there taken as 30)."""
import numpy as np
import pytest
import torch

from inferq_b200 import image, synth
from inferq_b200.kv import KvBatch
from inferq_b200.model import Model, State
from test_kv_gpu import Sequences

pytestmark = pytest.mark.gpu

KINDS = [("i8", "f32", 16, 256), ("f16", "f32", 8, 64), ("f16", "bf16", 16, 256), ("i8", "bf16", 8, 128)]


def near(s, got, want, most, note=None):
    got, eps = got.detach().cpu().double(), torch.finfo(s.dt).eps
    size = s.q.double().norm(dim=-1).max() * s.k.double().norm(dim=-1).max() / s.hd ** 0.5
    off = (got - want).abs()
    part = 2.0 ** -22 if s.dt == torch.float32 else 2.0 ** -11
    bound = want.abs() * eps / 2 + most * (part + 2.0 ** -22 * s.hd / 8 * size + 2.0 ** -15)
    assert (off <= bound).all(), (note, float((off - bound).max()), float(off.max()))
    limit = 2.0 ** -17 * size / 30 if s.dt == torch.float32 else 2.0 ** -11 + eps / 2
    rms = want.square().mean().sqrt()
    assert off.square().mean().sqrt() <= limit * rms, (note, float(off.square().mean().sqrt() / rms))


def rewrite(s, factors):
    """The same sequences with the values of some tokens multiplied."""
    s.v = s.v.clone()
    for token, f in factors.items():
        s.v[token] = (s.v[token].float() * f).to(s.dt)
    s.cache.append(s.k.cuda(), s.v.cuda(), s.all)


@pytest.mark.parametrize("binades", [1, 3, 12, 45, 100])
@pytest.mark.parametrize("fmt,dtype,heads,hd", KINDS)
def test_short_rows_are_the_same_whatever_stands_behind_them(cuda, fmt, dtype, heads, hd, binades):
    """Each of eight rows holds larger values than the one before it; alone and
    together, bit for bit, with the split's second chunk beginning among them."""
    for position in (257, 250, 3):
        s = Sequences([(8, position)], heads=heads, hd=hd, fmt=fmt, dtype=dtype, spread=5.0, seed=binades)
        rewrite(s, {position + i: 2.0 ** round(binades * i / 7) for i in range(8)})
        q = s.q.cuda()
        together = s.cache.attend(q, s.batch(), chunk=256)
        want, most = s.want()
        for i in range(8):
            alone = s.cache.attend(q[i:i + 1], KvBatch(s.table, s.position + i), chunk=256)
            assert torch.equal(alone[0], together[i]), (position, i)
            near(s, together[i], want[i], most[i], (position, i))
    s.cache.status()


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("binades", [1, 12, 45, 100])
@pytest.mark.parametrize("fmt,dtype,heads,hd", KINDS)
def test_short_rows_are_the_same_whatever_their_window_hides(cuda, fmt, dtype, heads, hd, binades, rows):
    s = Sequences([(rows, 300)], heads=heads, hd=hd, fmt=fmt, dtype=dtype, spread=5.0, seed=binades)
    kw = {"window": 50, "sinks": 3}
    for chunk in (64, 256):
        s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
        before = s.cache.attend(s.q.cuda(), s.batch(), chunk=chunk, **kw)
        keep = s.v
        rewrite(s, {t: 2.0 ** binades for t in (3, 4, 249, 250)})  # tiles that are read, tokens that no row sees
        got = s.cache.attend(s.q.cuda(), s.batch(), chunk=chunk, **kw)
        assert torch.equal(got, before)
        near(s, got, *s.want(50, 3))
        s.v = keep


CHUNKS = [("i8", "f32", 16, 256), ("f16", "f32", 16, 64), ("f16", "f32", 16, 128), ("f16", "bf16", 16, 256), ("i8", "bf16", 16, 128),
          ("i8", "f32", 16, 64), ("f16", "bf16", 32, 64)]


@pytest.mark.parametrize("binades", [1, 12, 45, 100])
@pytest.mark.parametrize("fmt,dtype,heads,hd", CHUNKS)
def test_chunks_are_the_same_whatever_stands_behind_their_rows(cuda, fmt, dtype, heads, hd, binades):
    """Row r's successor holds the large value: rows up to r keep their bits."""
    s = Sequences([(70, 190)], heads=heads, hd=hd, fmt=fmt, dtype=dtype, spread=5.0, seed=binades)
    q, b = s.q.cuda(), s.batch()
    want, most = s.want()
    before = s.cache.attend(q, b)
    keep = s.v
    for r in (0, 5, 14, 40, 68):
        rewrite(s, {190 + r + 1: 2.0 ** binades})
        got = s.cache.attend(q, b)
        assert torch.equal(got[:r + 1], before[:r + 1]), r
        near(s, got[:r + 1], want[:r + 1], most[:r + 1], r)
        s.v = keep
    s.cache.status()


@pytest.mark.parametrize("binades", [1, 12, 45, 100])
@pytest.mark.parametrize("fmt,dtype,heads,hd", CHUNKS)
def test_chunks_are_the_same_whatever_their_window_hides(cuda, fmt, dtype, heads, hd, binades):
    """Token t leaves the window of the rows from t + window on."""
    s = Sequences([(70, 190)], heads=heads, hd=hd, fmt=fmt, dtype=dtype, spread=5.0, seed=binades)
    q, b, kw = s.q.cuda(), s.batch(), {"window": 33, "sinks": 3}
    want, most = s.want(**kw)
    before = s.cache.attend(q, b, **kw)
    keep = s.v
    for token in (3, 64, 157, 170, 215):
        rewrite(s, {token: 2.0 ** binades})
        got = s.cache.attend(q, b, **kw)
        first = max(0, token + 33 - 190)  # rows from here on do not see it
        assert torch.equal(got[first:], before[first:]), token
        near(s, got[first:], want[first:], most[first:], token)
        rows = max(0, token - 190)  # nor do the rows before it
        assert torch.equal(got[:rows], before[:rows]), token
        s.v = keep


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_verify_rows_equal_sequential_rows_bitwise_where_scores_spread(cuda, kv):
    """The queries' norm weighs eight times as much: scores lie some 10 nats
    apart, behind a split's border (position 256) where few tokens share the
    exponent of a chunk."""
    cfg = synth.tiny()
    tensors = list(synth.generate(cfg, seed=11))
    for t in tensors:
        if "attn_q_norm" in t.name:
            t.data *= 8
    m = Model(cfg, tensors)
    for seed in range(6):
        base = image.synthetic(cfg, 250 + seed, seed=seed)
        a, b = State(m, 512, kv=kv), State(m, 512, kv=kv)
        a.import_image(base)
        b.import_image(base)
        toks = np.random.default_rng(seed).integers(0, cfg.vocab_size, 8)
        for rep in range(3):
            _, la, ha = a.forward(toks, logits=True, hidden=True)
            for i, t in enumerate(toks):
                _, lb, hb = b.forward([t], logits=True, hidden=True)
                assert np.array_equal(la[i].view(np.uint32), lb[0].view(np.uint32)), (seed, rep, i)
                assert np.array_equal(ha[i].view(np.uint32), hb[0].view(np.uint32)), (seed, rep, i)
