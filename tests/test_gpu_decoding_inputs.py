"""The decoding operators on the GPU: forms of input beside the plain ones
(expanded tensors, bounds that a call exceeds, empty and shared things)."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def i32(x):
    return _torch().tensor(x, dtype=_torch().int32, device="cuda")


# ---------------------------------------------------------------- expanded tensors
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [700, 50257])
def test_select_reads_expanded_logits_with_their_stride(vocab, kind):
    """One prompt's logits for all of its beams, as a search begins."""
    from test_gpu_beam import check_choice
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    # 15 rows lie behind the one that is expanded: what must not be read
    store = torch.randn((16, vocab), device="cuda", generator=gen).to(getattr(torch, kind))
    scores = -torch.rand(8, device="cuda", generator=gen)
    check_choice(store[:1].expand(8, vocab), scores, 4, 8)  # the definition, at its tolerance


def test_reorder_reads_an_expanded_table_with_its_stride():
    """The beams of one prompt start from its row of the table."""
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_reorder
    gen = torch.Generator(device="cuda").manual_seed(1)
    store = i32([[3, 0, -1, -1]] + [[5, 6, 7, 8]] * 3)  # three rows behind it
    row = store[:1].expand(4, 4)
    refs = i32([4, 0, 0, 4, 0, 0, 0, 0, 0])
    k = torch.randn((2, 9, 16, 2, 64), device="cuda", generator=gen).half()
    v = torch.randn_like(k)
    k2, v2 = k.clone(), v.clone()
    lens, parents = i32([21] * 4), i32([1, 0, 3, 2])
    got = beam_reorder(row, lens, parents, refs, k, v)
    want = beam_reorder(row.contiguous(), lens, parents, refs, k2, v2)
    assert got[0].tolist() == [[3, 0, -1, -1], [3, 1, -1, -1], [3, 2, -1, -1], [3, 4, -1, -1]]
    for a, b in zip(got + (k, v), want + (k2, v2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_and_append_read_an_expanded_table(new):
    """Sequences that share one row of the table."""
    torch = _torch()
    from tokenvector.inference_b200.generation import paged_append, paged_attention
    gen = torch.Generator(device="cuda").manual_seed(new)
    k = torch.randn((6, 32, 2, 64), device="cuda", generator=gen).half()
    v = torch.randn_like(k)
    q = torch.randn((3 * new, 4, 64), device="cuda", generator=gen).half()
    table = i32([[4, 1, 3], [9, 9, 9], [9, 9, 9]])[:1].expand(3, 3)
    ctx, cu = i32([96, 50, 70]), i32([0, new, 2 * new, 3 * new])
    kw = dict(max_q=new, return_lse=True)
    for a, b in zip(paged_attention(q, k, v, table, ctx, cu, **kw),
                    paged_attention(q, k, v, table.contiguous(), ctx, cu, **kw)):
        assert torch.equal(a, b)
    if new == 1:
        rows = torch.randn((3, 2, 64), device="cuda", generator=gen)
        k2, v2 = k.clone(), v.clone()
        paged_append(rows, rows, k, v, table, ctx)
        paged_append(rows, rows, k2, v2, table.contiguous(), ctx)
        assert torch.equal(k, k2) and torch.equal(v, v2)
