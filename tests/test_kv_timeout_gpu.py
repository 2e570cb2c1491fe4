"""Attention over the paged cache whose bounded device waits run out: the call
is reported, touches nothing but its outputs, and the next one is right.

With IQ_KV_TEST_TIMEOUT (looked up at every launch) the first CTA never
requests its first copy and waits a millisecond for it.  No GPU fault, trap or
hang is involved: every copy that is requested lands long before, every role
winds down (matrix instructions drained, tensor memory freed) and returns."""
import numpy as np
import pytest
import torch

from inferq_b200 import _lib, image, synth
from inferq_b200.model import Model, State
from test_kv_gpu import Sequences

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("f16", "f32"), ("i8", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("hd,heads", [(64, 8), (128, 8), (256, 16)])
@pytest.mark.parametrize("rows,ctx,kw", [
    (1, 40, {}), (1, 900, {"chunk": 256}), (8, 900, {"chunk": 256}),             # the split kernel: one tile, more than the stages
    (70, 70, {}), (70, 1500, {}), (70, 1500, {"window": 300, "sinks": 3}),       # the tensor-core kernel: likewise
])
def test_attend_reports_a_wait_that_ran_out(cuda, monkeypatch, rows, ctx, kw, hd, heads, fmt, dtype):
    s = Sequences([(rows, ctx - rows)], heads=heads, hd=hd, fmt=fmt, dtype=dtype)
    q, b = s.q.cuda(), s.batch()
    want = s.cache.attend(q, b, **kw)
    around = torch.full((rows + 64, heads, hd), 7.0, device="cuda", dtype=s.dt)
    monkeypatch.setenv("IQ_KV_TEST_TIMEOUT", "1")
    s.cache.attend(q, b, out=around[32:32 + rows], **kw)
    monkeypatch.delenv("IQ_KV_TEST_TIMEOUT")
    with pytest.raises(_lib.IqError, match="gave up") as e:
        s.cache.status()
    assert e.value.code == -6
    assert (around[:32] == 7).all() and (around[32 + rows:] == 7).all()
    assert torch.equal(s.cache.attend(q, b, **kw), want)
    s.cache.status()


def fails(monkeypatch, f):
    monkeypatch.setenv("IQ_KV_TEST_TIMEOUT", "1")
    with pytest.raises(_lib.IqError, match="gave up") as e:
        f()
    assert e.value.code == -6
    monkeypatch.delenv("IQ_KV_TEST_TIMEOUT")


def same(x, y):
    return np.array_equal(np.asarray(x).view(np.uint32), np.asarray(y).view(np.uint32))


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_mtp_calls_of_a_state_can_be_made_again(cuda, monkeypatch, kv):
    cfg = synth.mini_35b()
    m = Model(cfg, list(synth.generate(cfg, seed=1)))
    hid = np.random.default_rng(0).standard_normal((9, cfg.hidden_size)).astype(np.float32)
    a, b = State(m, 256, kv=kv), State(m, 256, kv=kv)
    for s in (a, b):
        s.import_image(image.synthetic(cfg, 40, seed=1))
    fails(monkeypatch, lambda: a.mtp_sync(30, hid[0], [1, 2, 3], hid[:3]))
    assert a.mtp_position == 30
    for s in (a, b):
        s.mtp_sync(30, hid[0], [1, 2, 3], hid[:3])
    fails(monkeypatch, lambda: a.mtp_draft(5, hid[4], 3, cfg.vocab_size))
    assert a.mtp_position == 33
    x, y = (s.mtp_draft(5, hid[4], 3, cfg.vocab_size) for s in (a, b))
    assert all(same(u, v) for u, v in zip(x[:3], y[:3]))


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_failed_passes_are_counted_and_an_image_makes_the_state_good_again(cuda, monkeypatch, kv):
    cfg = synth.tiny()
    m = Model(cfg, list(synth.generate(cfg, seed=1)))
    base = image.synthetic(cfg, 40, seed=1)
    a, b = State(m, 1024, kv=kv), State(m, 1024, kv=kv)
    toks = np.random.default_rng(1).integers(0, cfg.vocab_size, 100)
    # (one pass each: a second one would be captured with the copy left out)
    for call in (lambda s: s.verify(toks[:4]), lambda s: s.forward(toks[:4]), lambda s: s.forward(toks)):
        for s in (a, b):
            s.import_image(base)
        fails(monkeypatch, lambda: call(a))
        assert a.position > 40
        a.import_image(base)
        for s in (a, b):
            call(s)
        assert a.position == b.position
        la, lb = (s.forward(toks[:2], logits=True)[1] for s in (a, b))
        assert same(la, lb)
