"""States with a paged KV cache (iq_state_create_kv: f16 or i8 vectors, a
window with always-visible first tokens) against states with f32 rows and
against themselves.

What a paged state changes is the values that attention reads, and the sums'
order.  So the cache of the first attention layer (whose inputs do not depend
on any cache) holds exactly the quantised rows of the f32 state (as values: the
code 0 has no sign), and from one
and the same image a row's logits differ by rounding only: the row's own key
and value are quantised, one of some 300 that it sees.  Such a difference can
flip a quantised activation, which moves logits by 0.01 to 0.15 on these
random weights (the oracle's own rounding variants do); its median is held to
that range's lower part.
"""
import numpy as np
import pytest
import torch

from inferq_b200 import _lib, image, synth
from inferq_b200.model import Model, State
from test_kv_gpu import held

pytestmark = pytest.mark.gpu

CASES = {"tiny": synth.tiny, "mini_35b": synth.mini_35b}
KINDS = [("f16", 0, 0), ("i8", 0, 0), ("i8", 20, 3)]


@pytest.fixture(scope="module", params=list(CASES))
def model(request, cuda):
    cfg = CASES[request.param]()
    return cfg, Model(cfg, list(synth.generate(cfg, seed=11)))


def _same(a, b):
    return np.array_equal(np.ascontiguousarray(a, np.float32).view(np.uint32), np.ascontiguousarray(b, np.float32).view(np.uint32))


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_the_cache_holds_the_quantised_rows(model, kv):
    cfg, m = model
    prompt = np.random.default_rng(1).integers(0, cfg.vocab_size, 29)
    full, st = State(m, 256), State(m, 256, kv=kv)
    full.forward(prompt)
    st.forward(prompt)
    a, b = image.parse(full.export_image(), cfg), image.parse(st.export_image(), cfg)
    first = next(l for l in range(cfg.num_hidden_layers) if cfg.layer_is_full(l))
    for l in range(first):
        assert _same(a["layers"][l]["recurrent"], b["layers"][l]["recurrent"])
    for k in ("keys", "values"):
        assert np.array_equal(held(torch.from_numpy(a["layers"][first][k].copy()), kv).float().numpy(), b["layers"][first][k])
    assert st.kv_bytes < full.kv_bytes * (0.55 if kv == "f16" else 0.3) * 320 / 264  # whole pages: 5 x 64 of 264 positions


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_a_row_from_the_same_image_gives_the_same_logits(model, kv):
    cfg, m = model
    off = []
    for seed in range(9):
        im = image.synthetic(cfg, 300, seed=seed)
        full, st = State(m, 512), State(m, 512, kv=kv)
        st.import_image(im)
        full.import_image(st.export_image())  # the same values in both
        tok = [int(np.random.default_rng(seed).integers(0, cfg.vocab_size))]
        _, x, _ = full.forward(tok, logits=True)
        _, y, _ = st.forward(tok, logits=True)
        off.append(np.abs(x - y).max())
    assert np.median(off) <= 5e-2, off


@pytest.mark.parametrize("kv,window,sinks", KINDS)
@pytest.mark.parametrize("k", [2, 3, 4, 8])
def test_verify_rows_equal_sequential_rows_bitwise(model, kv, window, sinks, k):
    cfg, m = model
    rng = np.random.default_rng(k)
    base = image.synthetic(cfg, 250, seed=k)  # 256 lies among the rows: a split's and pages' border
    a, b = (State(m, 512, kv=kv, window=window, sinks=sinks) for _ in range(2))
    a.import_image(base)
    b.import_image(base)
    toks = rng.integers(0, cfg.vocab_size, k)
    for rep in range(3):  # eager, captured, replayed
        _, la, ha = a.forward(toks, logits=True, hidden=True)
        for i, t in enumerate(toks):
            _, lb, hb = b.forward([t], logits=True, hidden=True)
            assert _same(la[i], lb[0]) and _same(ha[i], hb[0]), (rep, i)


@pytest.mark.parametrize("kv,window,sinks", KINDS)
def test_rejected_drafts_leave_the_state_as_it_was(model, kv, window, sinks):
    cfg, m = model
    prompt = np.random.default_rng(2).integers(0, cfg.vocab_size, 21)
    a, b = (State(m, 256, kv=kv, window=window, sinks=sinks) for _ in range(2))
    am, _, _ = a.forward(prompt)
    b.forward(prompt)
    seed = int(am[-1])
    plain = [seed]
    for _ in range(12):
        plain.append(int(b.forward([plain[-1]])[0][0]))
    out = [seed]
    rng = np.random.default_rng(3)
    while len(out) < 10:
        right = plain[len(out):len(out) + int(rng.integers(0, 3))]
        draft = right + [(plain[len(out) + len(right)] + 1) % cfg.vocab_size]  # then a wrong one
        (acc, auth, com), _, _ = a.verify([out[-1]] + draft)
        assert acc == len(right) and com == acc + 1
        out += right + [auth]
    assert out == plain[:len(out)]


def test_images_go_round_and_between_formats(model):
    cfg, m = model
    im = image.synthetic(cfg, 97, seed=5)
    st = State(m, 256, kv="i8")
    st.import_image(im)
    once = st.export_image()
    again = State(m, 256, kv="i8")
    again.import_image(once)
    assert np.array_equal(once, again.export_image())  # nothing is lost a second time
    a, b = image.parse(im, cfg), image.parse(once, cfg)
    for l in range(cfg.num_hidden_layers):
        if cfg.layer_is_full(l):
            for k in ("keys", "values"):
                assert np.array_equal(held(torch.from_numpy(a["layers"][l][k].copy()), "i8").float().numpy(), b["layers"][l][k])
        else:
            assert _same(a["layers"][l]["recurrent"], b["layers"][l]["recurrent"])
    toks = np.random.default_rng(6).integers(0, cfg.vocab_size, 5)
    assert _same(st.forward(toks, logits=True)[1], again.forward(toks, logits=True)[1])


def test_a_window_as_long_as_the_context_changes_nothing(model):
    cfg, m = model
    toks = np.random.default_rng(7).integers(0, cfg.vocab_size, 40)
    a, b, c = State(m, 128, kv="i8"), State(m, 128, kv="i8", window=64, sinks=2), State(m, 128, kv="i8", window=8, sinks=2)
    x, y, z = (s.forward(toks, logits=True)[1] for s in (a, b, c))
    assert _same(x, y)
    assert _same(x[:8], z[:8]) and not _same(x[-1], z[-1])


@pytest.mark.parametrize("kv,window,sinks", KINDS)
def test_the_wide_pass_fills_the_cache_and_the_state_goes_on(cuda, kv, window, sinks):
    cfg = synth.tiny()
    m = Model(cfg, list(synth.generate(cfg, seed=11)))
    prompt = np.random.default_rng(8).integers(0, cfg.vocab_size, 700)  # chunks of 512 and 188 rows
    states = [State(m, 1024, kv=k, window=w, sinks=s) for k, w, s in ((kv, window, sinks), ("f32", 0, 0)) * 2]
    wide, wide32, st, st32 = states
    for s in (wide, wide32):
        s.forward(prompt)
    for s in (st, st32):
        for r in range(0, 700, 56):  # below 64 rows: passes of 8
            s.forward(prompt[r:r + 56])
    assert all(s.position == 700 for s in states)
    a, a32, b, b32 = (image.parse(s.export_image(), cfg) for s in states)
    first = next(l for l in range(cfg.num_hidden_layers) if cfg.layer_is_full(l))
    # the layers before the first attention layer are those of the f32 state's pass, wide or not
    for got, want in ((a, a32), (b, b32)):
        for k in ("keys", "values"):
            assert np.array_equal(held(torch.from_numpy(want["layers"][first][k].copy()), kv).float().numpy(), got["layers"][first][k])
    toks = np.random.default_rng(9).integers(0, cfg.vocab_size, 4)
    other = State(m, 1024, kv=kv, window=window, sinks=sinks)
    other.import_image(wide.export_image())
    (acc, auth, com), lg, _ = wide.verify(toks, logits=True)
    for i in range(com):
        assert _same(lg[i], other.forward([toks[i]], logits=True)[1][0])


@pytest.mark.parametrize("kv,window,sinks", KINDS)
def test_mtp_catch_up_in_pieces_equals_one_catch_up(cuda, kv, window, sinks):
    cfg = synth.mini_35b()
    m = Model(cfg, list(synth.generate(cfg, seed=11)))
    prompt = np.random.default_rng(4).integers(0, cfg.vocab_size, 31)
    a, b = (State(m, 256, kv=kv, window=window, sinks=sinks) for _ in range(2))
    am, _, hid = a.forward(prompt, hidden=True)
    b.forward(prompt)
    a.mtp_sync(0, None, prompt, hid)
    b.mtp_sync(0, None, prompt[:4], hid[:4])
    b.mtp_sync(4, hid[3], prompt[4:23], hid[4:23])
    b.mtp_sync(23, hid[22], prompt[23:], hid[23:])
    for _ in range(3):
        da = a.mtp_draft(int(am[-1]), hid[-1], 3, cfg.vocab_size)
        db = b.mtp_draft(int(am[-1]), hid[-1], 3, cfg.vocab_size)
        for x, y in zip(da[:3], db[:3]):
            assert np.array_equal(np.asarray(x).view(np.uint32), np.asarray(y).view(np.uint32))
        for s in (a, b):
            s.mtp_sync(31, hid[-1], [int(am[-1])], hid[-1:])
    assert a.mtp_position == b.mtp_position == 32


def test_refusals(model):
    cfg, m = model
    with pytest.raises(ValueError, match="KV cache format"):
        State(m, 64, kv="q4")
    for kw, code in (({"kv": "i8", "window": -1}, -1), ({"kv": "i8", "window": 4, "sinks": -1}, -1), ({"window": 8}, -4)):
        with pytest.raises(_lib.IqError) as e:
            State(m, 64, **kw)
        assert e.value.code == code
    st = State(m, 16, kv="i8")
    st.forward([1] * 16)
    with pytest.raises(_lib.IqError, match="exceeds"):
        st.forward([1])
