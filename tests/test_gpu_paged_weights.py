"""Attention over a long cache in which one key has nearly all the weight: the
many weak ones, far below the smallest normal float16 each, still count.

One key has the score E ln 2, 2^13 others 0, so each of these has the weight
2^-E of the largest, and values of 0.5 to 1.5 against zeros of the one: out is
about 2^(13-E).  So many equal sequences share the cache that each is worked off in
one piece (in a piece without the strong key the weak ones are not weak).

The tolerance is that of test_gpu_paged with two terms of this case in place of
its estimates.  Float16 weights are rounded to multiples of 2^-24 at their
smallest, after a factor that keeps the largest within the type: 2^15 where a
sequence has at most 16 rows to a kv head, 2^7 (and a largest of up to 2^8) else,
so 2^-40 or 2^-32 of the largest each, and 2^13 of them times 1.5.  The f32 sums of
one piece have 2^13 / 16 products that may be cut off at 2^-23 each, and 2^13 / 32
additions rounded to 2^-24: 2^-14 + 2^-16 of out, 2^-16 in lse."""
import math

import pytest
from test_gpu_paged import UNIT, attend, clean, definition, make

pytestmark = pytest.mark.gpu
KEYS = 1 << 13


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("new,seqs", [(1, 1184), (20, 148)])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("power", [7.9, 8.1, 22.3, 24.6, 25.5, 26.7])
def test_many_weak_keys_beside_a_strong_one(power, place, new, seqs, kind):
    import torch
    s = make([new], [KEYS + new], 1, 1, 8, 1024, kind, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    s["k"].zero_()
    s["v"].copy_(torch.rand(s["v"].shape, device="cuda", generator=gen) + 0.5)
    s["q"].zero_()
    s["q"][:, :, 0] = 4.0
    at = {"first": 0, "middle": KEYS // 2 + 77, "last": KEYS}[place]  # (the last one that all rows see)
    page = int(s["table"][0, at // 1024])
    s["k"][page, at % 1024, 0, 0] = power * math.log(2.0) / 4.0
    s["v"][page, at % 1024] = 0.0
    ref, ref_lse, A, S = definition(s, scale=1.0)
    many = dict(s, q=s["q"].repeat(seqs, 1, 1), table=s["table"].expand(seqs, -1), ctx=s["ctx"].repeat(seqs),
                cu=torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device="cuda"))
    got, lse = attend(many, max_q=new, scale=1.0)
    clean()
    e = (8 / 8 + 8) * 2.0 ** -23 * (S + 1)
    floor = 0.0 if kind == "bfloat16" else 1.5 * KEYS * 2.0 ** (-40 if new == 1 else -32)
    tol = 1.05 * UNIT[kind] * (A + ref.abs()) + ((4 * e)[..., None] + 2.0 ** -14 + 2.0 ** -16) * A + floor + 2.0 ** -25
    off = (got.double().view(seqs, *ref.shape) - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert ((lse.double().view(seqs, *ref_lse.shape) - ref_lse).abs() <= 2 * e + 2.0 ** -16 + 2.0 ** -21 * (1 + ref_lse.abs())).all()
