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


# ---------------------------------------------------------------- a bound on the new rows that a call exceeds
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("new,most,heads,kv_heads,dim", [
    ([1, 5, 1, 16, 2, 9], 1, 2, 2, 64), ([5, 1, 16, 3, 7, 1], 3, 4, 2, 128), ([16] * 6, 2, 8, 1, 64),
    ([90, 20, 300, 1, 65, 64], 64, 2, 2, 64), ([140, 3, 33, 500, 20, 1], 130, 4, 1, 128)])
def test_attention_takes_max_q_rows_of_a_sequence(new, most, heads, kv_heads, dim, window):
    """The first max_q rows of each sequence follow the definition; the others' outputs, and what lies behind the
    workspace, stay as they are."""
    import ctypes as C
    from test_gpu_paged import clean, definition, hold, make
    from tokenvector.inference_b200 import _native as N
    torch = _torch()
    ctx = [4000, 2500, 16, 900, 3100, 1700]
    s = make(new, ctx, heads, kv_heads, dim, 32, "float16", seed=most)
    rows, group = sum(new), heads // kv_heads
    i64 = lambda *v: (C.c_int64 * len(v))(*v)  # noqa: E731
    need = C.c_int64()
    N.call("tvq_paged_attention_workspace", heads, kv_heads, dim, len(new), rows, most, C.byref(need))
    ws = torch.full((need.value + 65536,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.full_like(s["q"], 77.0)
    lse = torch.full((rows, heads), 77.0, device="cuda")
    k, v, q, table = s["k"], s["v"], s["q"], s["table"]
    N.call("tvq_dev_paged_attention", N.TYPE_F16, q.data_ptr(), i64(*q.stride()[:2]), heads, k.data_ptr(), v.data_ptr(),
           i64(*k.shape), i64(*(k.stride()[:3] + v.stride()[:3])), table.data_ptr(), table.stride(0), table.shape[1],
           s["ctx"].data_ptr(), s["cu"].data_ptr(), len(new), rows, most, dim ** -0.5, window, out.data_ptr(),
           lse.data_ptr(), ws.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream)
    clean()
    assert group * most <= 16 or most > 16
    assert (ws[need.value:] == 0xA5).all()
    taken = torch.cat([torch.arange(n) < most for n in new]).cuda()
    assert (out[~taken] == 77.0).all() and (lse[~taken] == 77.0).all()
    want = definition(s, window=window)
    for t in want:  # a row that is not taken: nothing to compare
        t[~taken] = 0.0
    got, got_lse = out.clone(), lse.clone()
    got[~taken] = 0.0
    got_lse[~taken] = 0.0
    hold(s, got, got_lse, want)


# ---------------------------------------------------------------- several devices in a process
def test_operators_work_on_every_device():
    """Kernels with more than 48 KB of shared memory, on one GPU and then on another one of the process."""
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_select, paged_attention
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn((9, 16, 2, 64), generator=gen).half() for _ in range(2))
    q = torch.randn((40, 4, 64), generator=gen).half()
    x, scores = torch.randn((64, 9000), generator=gen), torch.zeros(64)
    table = torch.tensor([[3, 0, 8, 5]], dtype=torch.int32)
    results = []
    for dev in ("cuda:0", "cuda:1"):
        on = lambda t: t.to(dev)  # noqa: E731,B023
        ctx = torch.tensor([60], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, 40], dtype=torch.int32, device=dev)
        results.append([paged_attention(on(q[:1]), on(k), on(v), on(table), ctx),
                        paged_attention(on(q), on(k), on(v), on(table), ctx, cu),
                        *beam_select(on(x), on(scores), 64, 64)])
    for a, b in zip(*results):
        assert torch.equal(a.cpu(), b.cpu())


# ---------------------------------------------------------------- lengths out of range
@pytest.mark.parametrize("lens,same", [
    ([-3, 20, -16, -(1 << 31)], [0, 20, 0, 0]), ([(1 << 31) - 1, 37, (1 << 31) - 16, 1 << 30], [3 * 16 + 5, 37, 48, 48])])
def test_reorder_of_lengths_out_of_range(lens, same):
    """Below 0 is 0; behind the table's columns there is no room, whatever the length."""
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_reorder
    gen = torch.Generator(device="cuda").manual_seed(2)
    store = i32([[1 << 29] * 3] * 3 + [[0, 3, 6], [1, 4, 7], [2, 5, 8], [9, 10, 11]] + [[1 << 29] * 3] * 3)
    table = store[3:7]  # page numbers out of range in front and behind
    k = torch.randn((2, 16, 16, 2, 64), device="cuda", generator=gen).half()
    v, k2 = torch.randn_like(k), k.clone()
    v2 = v.clone()
    refs = [0] * 16
    for row, n in zip(table.tolist(), same):
        for p in row[:-(-n // 16)]:
            refs[p] += 1
    parents = i32([0, 1, 3, 2, 0])
    got = beam_reorder(table, i32(lens), parents, i32(refs), k, v)
    want = beam_reorder(table, i32(same), parents, i32(refs), k2, v2)
    assert got[1].tolist() == [max(0, lens[p]) for p in parents.tolist()]
    for a, b in zip((got[0], got[2], got[3], k, v), (want[0], want[2], want[3], k2, v2)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- a page that is one row's last and another's full one
def test_reorder_leaves_a_page_alone_that_another_row_holds_in_full():
    """Rows of different lengths over a shared prefix: the shorter one gets a copy, or its next token would overwrite
    the longer one's."""
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_reorder, paged_append
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn((1, 9, 16, 2, 64), device="cuda", generator=gen).half()
    v = torch.randn_like(k)
    #       ends in page 1    page 1 is full    the same tokens as row 0
    table = i32([[0, 1, -1, -1], [0, 1, 2, -1], [0, 1, -1, -1], [3, 4, -1, -1]])
    lens, refs = i32([20, 40, 21, 18]), i32([3, 3, 1, 1, 1, 0, 0, 0, 0])
    old = [k[0, p].clone() for p in range(9)]
    t, n, c, status = beam_reorder(table, lens, i32([0, 1, 2, 3, 3]), refs, k, v)
    assert t.tolist() == [[0, 5, -1, -1], [0, 1, 2, -1], [0, 6, -1, -1], [3, 4, -1, -1], [3, 7, -1, -1]]
    assert c.tolist() == [3, 1, 1, 2, 1, 1, 1, 1, 0] and status.tolist() == [3, 0]
    for dst, src, fill in ((5, 1, 4), (6, 1, 5), (7, 4, 2)):
        assert torch.equal(k[0, dst, :fill], old[src][:fill])
    # the rows' next tokens leave the other rows' as they are
    rows = torch.ones((5, 2, 64), device="cuda")
    paged_append(rows, rows, k[0], v[0], t, n + 1)
    assert torch.equal(k[0, 1], old[1]) and torch.equal(k[0, 0], old[0])
    assert torch.equal(k[0, 2, :8], old[2][:8]) and bool((k[0, 2, 8] == 1).all())


def test_reorder_keeps_a_last_page_of_rows_of_different_lengths():
    """A last page that only last pages share stays with the lowest row."""
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_reorder
    k = torch.zeros((1, 6, 16, 2, 64), device="cuda").half()
    t, n, c, status = beam_reorder(i32([[0, 1, -1], [0, 1, -1], [2, -1, -1]]), i32([20, 25, 0]), i32([1, 0, 2]),
                                   i32([2, 2, 0, 0, 0, 0]), k, k.clone())
    assert t.tolist() == [[0, 1, -1], [0, 2, -1], [3, -1, -1]] and c.tolist() == [2, 1, 1, 1, 0, 0]
    assert status.tolist() == [2, 0]


# ---------------------------------------------------------------- caches without pages, tables without columns
@pytest.mark.parametrize("cols", [0, 2])
@pytest.mark.parametrize("new,dim,page", [(1, 64, 16), (1, 128, 16), (1, 80, 8), (40, 64, 16), (40, 128, 128)])
def test_an_empty_cache_holds_empty_sequences(new, dim, page, cols):
    """Rows in front of the cache's first token: nothing to read or to write; a token that should be there is reported."""
    import math

    from test_gpu_paged import clean
    from tokenvector.inference_b200 import _native as N
    from tokenvector.inference_b200.generation import paged_append, paged_attention
    torch = _torch()
    k = torch.empty((0, page, 2, dim), dtype=torch.float16, device="cuda")
    table = torch.full((2, cols), 3, dtype=torch.int32, device="cuda")
    q = torch.ones((2 * new, 4, dim), dtype=torch.float16, device="cuda")
    cu, rows = i32([0, new, 2 * new]), q[:, :2].float()
    clean()
    for ctx in ([0, 0], [0, 5]):
        out, lse = paged_attention(q, k, k, table, i32(ctx), cu, max_q=new, return_lse=True)
        assert not out.any() and bool((lse[:new] == -math.inf).all())
        if ctx[1] == 0:
            assert bool((lse == -math.inf).all())
            paged_append(rows, rows, k, k.clone(), table, i32(ctx), cu)
            clean()
        else:
            assert N.lib().tvq_device_error(None) == N.TVQ_ERR_INVALID and "page" in N.last_error()
            assert abs(float(lse[-1, 0]) - math.log(5)) < 1e-5  # five keys of zeros
            paged_append(rows, rows, k, k.clone(), table, i32(ctx), cu)
            assert N.lib().tvq_device_error(None) == N.TVQ_ERR_INVALID and "page" in N.last_error()
    clean()


def test_reorder_without_pages():
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_reorder
    k = torch.empty((2, 0, 16, 2, 64), dtype=torch.float16, device="cuda")
    t, n, c, status = beam_reorder(i32([[-1, -1]] * 2), i32([0, 0]), i32([1, 0, -1]), i32([]), k, k.clone())
    assert t.tolist() == [[-1, -1]] * 3 and n.tolist() == [0, 0, 0] and c.numel() == 0 and status.tolist() == [0, 2]
