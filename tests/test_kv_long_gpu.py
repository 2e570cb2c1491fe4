"""Long accumulations of the tensor-core attention kernel against what they
must give whatever is added: where all values of a head's element are equal,
the output is that value, however the scores lie.

Tolerances, relative to the value, for f32 rows.  Every instruction adds 16
tokens' products to the accumulator and cuts the sum off: at most a unit of the
last place, 2^-23, of the sum that stands there; a chunk of C tokens has C / 8
of them (two parts).  Weights keep 2^-22, and f32 operations outside the matrix
instructions (scales, the sum, the join, the division) add less than 2^-21.
 * First token far above the rest: the sum stands complete after its tile, whose
   8 instructions are the only ones that cut: 2^-20, with the rest 2^-19.
 * Equal scores: the sum grows evenly, so that half of C / 8 units are lost at
   most on the average, and all of them by no element.
"""
import math

import pytest
import torch

from test_kv_gpu import Sequences, held

pytestmark = pytest.mark.gpu


def off(s, **kw):
    """Relative error of outputs whose values are all equal."""
    s.v = s.v[:1].abs().clamp(min=0.5).expand_as(s.v).contiguous()
    s.cache.append(s.k.cuda(), s.v.cuda(), s.all)
    got = s.cache.attend(s.q.cuda(), s.batch(), **kw).cpu().double()
    want = held(s.v[:1], s.fmt)[0].repeat_interleave(s.heads // s.kv_heads, 0)
    s.cache.status()
    return (got - want) / want


@pytest.mark.parametrize("fmt", ["i8", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ctx,chunk", [(1536, 1536), (2560, 0), (9000, 0), (9000, 1 << 20)])
def test_a_first_token_that_outweighs_the_rest(cuda, fmt, hd, ctx, chunk):
    s = Sequences([(70, ctx - 70)], hd=hd, fmt=fmt)
    u = torch.nn.functional.normalize(torch.randn(2, hd, generator=torch.Generator().manual_seed(2)), dim=-1)
    s.q = s.q * 0.01 + 5 * math.sqrt(hd) * u.repeat_interleave(8, 0)
    s.k = s.k * 0.01
    s.k[0] = 5 * u  # 25 nats above the others
    e = off(s, chunk=chunk)
    assert e.abs().max() <= 2.0 ** -19, float(e.abs().max())


@pytest.mark.parametrize("fmt", ["i8", "f16"])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("ctx,chunk", [(1536, 1536), (2560, 640), (9000, 0), (9000, 1 << 20)])
def test_equal_scores(cuda, fmt, hd, ctx, chunk):
    s = Sequences([(70, ctx - 70)], hd=hd, fmt=fmt)
    s.q = s.q * 0.05
    e = off(s, chunk=chunk)
    units = 640 / 8 * 2.0 ** -23
    assert e.abs().max() <= units + 2.0 ** -20, float(e.abs().max())
    assert e.mean().abs() <= units / 2 + 2.0 ** -20, float(e.mean())
