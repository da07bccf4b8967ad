"""The decoding operators at sizes that take their rarer ways: more lists than
the merge has threads, more sequences than a CTA has threads, many heads to a
kv head, large pages.  Definitions and tolerances are those of test_gpu_paged
and test_gpu_beam."""
import pytest
from test_gpu_beam import check_choice
from test_gpu_paged import attend, clean, definition, hold, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch,beams,keep,vocab", [
    (1, 16, 16, 50257), (2, 16, 64, 50257), (1, 8, 16, 120001), (1, 64, 64, 50257), (1, 64, 1, 131072), (1, 3, 64, 1 << 20)])
def test_choice_of_many_lists(batch, beams, keep, vocab, kind):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(beams + vocab)
    x = torch.randn((batch * beams, vocab), device="cuda", generator=gen) * 3
    scores = -2 * torch.rand(batch * beams, device="cuda", generator=gen)
    check_choice(x.to(getattr(torch, kind)), scores, beams, keep)
    # ties in all rows, a beam that has ended, one that does not take part
    x = ((x * 2).round() / 2).to(getattr(torch, kind))
    done = torch.zeros(batch * beams, dtype=torch.bool, device="cuda")
    done[1] = True
    scores[2] = -float("inf")
    check_choice(x, scores, beams, keep, done, vocab // 2)
    check_choice(torch.ones_like(x), scores, beams, keep)


@pytest.mark.parametrize("new,ctx", [
    ([1] * 700, [1 + i * 37 % 200 for i in range(700)]),                          # the rows kernel's scan: 320 at once
    ([i % 3 for i in range(650)], [i % 3 + i * 13 % 90 for i in range(650)]),     # some without rows
    ([i % 4 + 17 * (i % 5 == 0) for i in range(1300)], [40 + i * 7 % 100 for i in range(1300)])])  # the tile kernel's: 640
@pytest.mark.parametrize("window", [0, 30])
def test_attention_of_many_sequences(new, ctx, window):
    s = make(new, ctx, 2, 1, 64, 16, "float16", seed=len(new))
    hold(s, *attend(s, max_q=max(new), window=window), definition(s, window=window))
    clean()


@pytest.mark.parametrize("group", [17, 49, 64, 65, 100, 127, 128])
@pytest.mark.parametrize("new,ctx", [([1, 1], [700, 5]), ([3, 1, 30], [3, 900, 200])])
def test_attention_of_many_heads_to_a_kv_head(group, new, ctx):
    for dim, kind in ((64, "float16"), (128, "bfloat16")):
        s = make(new, ctx, 2 * group, 2, dim, 16, kind, seed=group)
        hold(s, *attend(s, max_q=max(new)), definition(s))
    clean()


@pytest.mark.parametrize("page", [512, 1024])
@pytest.mark.parametrize("dim", [24, 64, 72, 120, 128])
@pytest.mark.parametrize("new,ctx", [([1, 1, 2], [1, 3000, 1025]), ([130, 1, 40], [130, 2049, 1500])])
def test_attention_over_large_pages(new, ctx, dim, page):
    s = make(new, ctx, 4, 2, dim, page, "bfloat16", seed=dim, head_major=dim > 64)
    hold(s, *attend(s, max_q=max(new)), definition(s))
    hold(s, *attend(s, max_q=max(new), window=600), definition(s, window=600))
    clean()
