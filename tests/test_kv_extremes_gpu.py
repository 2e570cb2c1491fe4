"""Attention over keys, values and queries near the ends of f32's range, whose
scores and results are ordinary numbers: against the definition in 64 bits,
with the tolerances of test_kv_gpu."""
import pytest
import torch

from test_kv_gpu import Sequences, close

pytestmark = pytest.mark.gpu


def run(s, **kw):
    s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
    got = s.cache.attend(s.q.cuda(), s.batch(), **kw)
    want, most = s.want()
    return got, want, most


@pytest.mark.parametrize("rows,chunk", [(1, 0), (1, 128), (3, 0), (8, 128), (70, 0), (70, 640)])
@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("f16", "f32"), ("i8", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("binades", [100, 110, 118, -90, -100])
def test_keys_and_queries(cuda, binades, fmt, dtype, rows, chunk):
    s = Sequences([(rows, 333)], heads=8, kv_heads=1, hd=64, fmt=fmt, dtype=dtype)
    s.k, s.q = s.k * 2.0 ** binades, s.q * 2.0 ** -binades
    close(*run(s, chunk=chunk), s.dt)


@pytest.mark.parametrize("rows,chunk", [(1, 0), (1, 128), (3, 0), (8, 128), (70, 0), (70, 640)])
@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("f16", "f32"), ("i8", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("binades", [100, 110, 116, -80, -90])
def test_values(cuda, binades, fmt, dtype, rows, chunk):
    s = Sequences([(rows, 333)], heads=8, kv_heads=1, hd=64, fmt=fmt, dtype=dtype, spread=4.0)
    s.v = s.v * 2.0 ** binades
    got, want, most = run(s, chunk=chunk)
    close(got.cpu().double() * 2.0 ** -binades, want * 2.0 ** -binades, most * 2.0 ** -binades, s.dt)


@pytest.mark.parametrize("fmt", ["i8", "f16"])
@pytest.mark.parametrize("rows,chunk", [(1, 0), (8, 128), (70, 0)])
def test_many_small_weights_under_huge_values(cuda, fmt, rows, chunk):
    """One token 14 nats above thousands of others that together weigh as much as some thousandths of it."""
    s = Sequences([(rows, 5000)], heads=8, kv_heads=1, hd=64, fmt=fmt)
    u = torch.nn.functional.normalize(torch.ones(1, 64), dim=-1)
    s.q, s.k = s.q * 0.01 + 8 * u, s.k * 0.01
    s.k[0] = 14 * u
    s.v = s.v.abs() * 2.0 ** 117
    s.v[0] = s.v[0] * 2.0 ** -6
    got, want, most = run(s, chunk=chunk)
    off = (got.cpu().double() - want).abs() / most
    # (2^-17 of the row's values; without the small weights it would be 5000 e^-14 = 2^-7.9)
    assert off.max() <= 2.0 ** -17, float(off.max())
