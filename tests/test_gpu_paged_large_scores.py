"""Attention of scores so large that the rounding of an f32 score is worth more
than a factor of two in its weight."""
import pytest
from test_gpu_paged import attend, clean, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("new,ctx", [([1, 1], [3000, 500]), ([150, 40], [900, 40])])
@pytest.mark.parametrize("size", [1e6, 8.3e6, 1.7e7, 3.5e7, 1e9, 1e12])
def test_scores_so_large_that_their_rounding_is_whole_powers(size, new, ctx, kind):
    """Scores whose last bit is worth more than a factor of two: which key wins is open, but out is a mean of values."""
    import torch
    s = make(new, ctx, 4, 2, 64, 16, kind, seed=int(size) % 1000)
    got, lse = attend(s, max_q=max(new), scale=size / 100)
    clean()
    assert bool(got.isfinite().all()) and bool(lse.isfinite().all())
    held = torch.cat([s["table"][i, :-(-c // 16)] for i, c in enumerate(ctx)]).long()
    v = s["v"][held].float()
    assert float(got.float().abs().max()) <= 1.01 * float(v[v.isfinite()].abs().max())
