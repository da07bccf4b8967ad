"""The paged cache on the GPU: append against exact rounding, attention
against its definition in 64 bits.

Attention's tolerance, element by element.  w is the unit roundoff of the
cache's type (2^-11 for float16, 2^-8 for bfloat16), A = sum_j p_j |v_j| and
S = max_j |scale| sum_d |q_d k_jd| of the row in 64 bits.  The weights are
rounded to the type (w A; below float16's normal range 2^-25 absolute each,
against weights of at most 2^-8 of the row's largest), the result once more
(w |out|, 2^-25 absolute in float16), and the scores carry the f32 sums'
error e = (dim / 8 + 8) 2^-23 (S + 1), which moves each weight by a factor
e^(2 e).  lse: 2 e + 2^-21 (1 + |lse|)."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def make(new, ctx, heads, kv_heads, dim, page, kind, *, seed=0, head_major=False, spare=3, junk=True, wide_table=0):
    """Inputs of one call; every slot behind a sequence's end, and every spare page, holds NaN."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, kind)
    held = [-(-c // page) for c in ctx]
    pool = sum(held) + spare
    order = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)
    cols = max([1] + held)
    store = torch.full((len(ctx), cols + wide_table), -7, dtype=torch.int32, device="cuda")
    table = store[:, :cols]
    first = 0
    shape = (pool, kv_heads, page, dim) if head_major else (pool, page, kv_heads, dim)
    k = torch.randn(shape, device="cuda", generator=gen).to(dt)
    v = torch.randn(shape, device="cuda", generator=gen).to(dt)
    if head_major:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    if junk:
        for spare_page in order[sum(held):].tolist():
            k[spare_page] = float("nan")
            v[spare_page] = float("nan")
    for s, c in enumerate(ctx):
        pages = order[first:first + held[s]]
        table[s, :held[s]] = pages
        first += held[s]
        if junk and c % page:
            k[pages[-1], c % page:] = float("nan")
            v[pages[-1], c % page:] = float("inf")
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (torch.randn((cu[-1], heads, dim), device="cuda", generator=gen) * 1.5).to(dt)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(q=q, k=k, v=v, table=table, ctx=i32(ctx), cu=i32(cu), new=new, lens=ctx)


def definition(s, scale=None, window=0):
    """(out, lse, A, S) in 64 bits; rows without keys 0 and -inf."""
    torch = _torch()
    q, k, v = s["q"], s["k"], s["v"]
    heads, dim = q.shape[1:]
    page, kv_heads = k.shape[1:3]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    A = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    S = torch.zeros_like(lse)
    first = 0
    for i, (n, c) in enumerate(zip(s["new"], s["lens"])):
        rows = slice(first, first + n)
        first += n
        if n == 0 or c == 0:
            continue
        pages = s["table"][i, :-(-c // page)].long()
        pos = torch.arange(c - n, c, device="cuda")[:, None]
        j = torch.arange(c, device="cuda")[None]
        seen = (j <= pos) & ((j > pos - window) if window else (j >= 0))
        some = seen.any(1)
        for h in range(heads):
            kk = k[pages, :, h // group].reshape(-1, dim)[:c].double()
            vv = v[pages, :, h // group].reshape(-1, dim)[:c].double()
            a = (q[rows, h].double() @ kk.T) * scale
            a = a.masked_fill(~seen, -math.inf)
            p = torch.softmax(a, 1).masked_fill(~some[:, None], 0.0)
            out[rows, h] = p @ vv
            A[rows, h] = p @ vv.abs()
            lse[rows, h] = torch.logsumexp(a, 1)
            S[rows, h] = (q[rows, h].double().abs() @ kk.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(1)
    return out, lse, A, S


def hold(s, got, lse, want):
    torch = _torch()
    ref, ref_lse, A, S = want
    w = UNIT[str(s["q"].dtype).split(".")[1]]
    dim = s["q"].shape[2]
    e = (dim / 8 + 8) * 2.0 ** -23 * (S + 1)
    keys = max(s["lens"] + [1])
    flat = 2.0 ** -25 * (1 + keys * 2.0 ** -8 * 8) if w == 2.0 ** -11 else 0.0
    tol = 1.05 * w * (A + ref.abs()) + (4 * e)[..., None] * A + flat + 1e-30
    bad = (got.double() - ref).abs() > tol
    assert not bad.any() and not got.isnan().any(), (int(bad.sum()), float(((got.double() - ref).abs() / tol).max()))
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert not got[empty].any()
    off = (lse.double() - ref_lse)[~empty].abs()
    assert (off <= (2 * e + 2.0 ** -21 * (1 + ref_lse.abs()))[~empty]).all(), float(off.max())


def attend(s, **kw):
    from tokenvector.inference_b200.generation import paged_attention
    return paged_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["cu"], return_lse=True, **kw)


def clean():
    """No device error is left behind."""
    from tokenvector.inference_b200 import _native as N
    assert N.lib().tvq_device_error(None) == N.TVQ_OK, N.last_error()


# new rows, tokens in the cache, heads, kv heads, dim, page
SHAPES = [
    ([1], [1], 1, 1, 64, 16),
    ([1, 1, 1], [700, 1, 16], 12, 12, 64, 16),          # single tokens, an exact page end
    ([1] * 5, [0, 15, 17, 64, 129], 4, 4, 64, 16),      # an unused slot of a batch
    ([1, 1], [3000, 777], 8, 2, 128, 64),
    ([1, 1], [513, 40], 14, 2, 128, 32),                # seven heads to one
    ([1, 1, 1], [97, 300, 8], 5, 5, 80, 8),
    ([1], [20000], 1, 1, 32, 128),                      # one long row over the whole GPU
    ([1, 1], [1000, 333], 25, 1, 64, 16),               # all heads share one
    ([1, 1], [130, 260], 48, 1, 128, 16),
    ([4, 1, 6, 0], [40, 9, 1300, 12], 8, 2, 128, 32),
    ([7, 3], [5, 2], 4, 2, 64, 8),                      # more rows than tokens: some see nothing
    ([33, 2, 64], [33, 2, 700], 6, 2, 64, 16),
    ([100, 37, 64, 1], [100, 37, 64, 1], 2, 2, 64, 16),  # whole prompts
    ([300], [1100], 4, 1, 128, 128),
    ([257, 129], [257, 400], 3, 1, 128, 64),
    ([200], [333], 7, 1, 96, 16),
    ([130, 5, 1], [130, 900, 2000], 4, 4, 16, 256),     # prompts and single tokens in one call
    ([513], [513], 1, 1, 8, 8),
    ([140], [100], 2, 2, 128, 16),
    ([64], [4096], 16, 2, 128, 64),                     # few rows, many keys
    ([1] * 30, [2000 + 37 * i for i in range(30)], 8, 4, 128, 16),  # many tiles for every SM
    ([2] * 30, [4000 + 41 * i for i in range(30)], 4, 4, 64, 32),
    ([17 + i * 7 % 130 for i in range(200)], [17 + i * 7 % 130 for i in range(200)], 4, 4, 64, 16),  # many short prompts
    ([20 + i * 3 % 50 for i in range(150)], [20 + i * 3 % 50 + i * 11 % 300 for i in range(150)], 8, 4, 128, 32),
]


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c)[-40:])
def test_attention_follows_its_definition(case, kind):
    s = make(*case, kind, seed=len(case[0]) + case[4], head_major=case[5] % 32 == 0, wide_table=5)
    want = definition(s)
    for most in (max(case[0]), None):
        hold(s, *attend(s, max_q=most), want)
    clean()


@pytest.mark.parametrize("window", [1, 7, 64, 129, 5000])
@pytest.mark.parametrize("new,ctx", [([1, 1, 1], [5, 1000, 260]), ([9, 2], [700, 30]), ([300, 40], [300, 900])])
def test_attention_window(new, ctx, window):
    s = make(new, ctx, 4, 2, 64, 16, "float16", seed=window)
    hold(s, *attend(s, max_q=max(new), window=window), definition(s, window=window))
    clean()


@pytest.mark.parametrize("scale", [0.0, 0.01, 3.0, -0.5])
@pytest.mark.parametrize("new,ctx", [([1, 1], [500, 77]), ([150], [450])])
def test_attention_scale(new, ctx, scale):
    s = make(new, ctx, 4, 2, 128, 32, "bfloat16", seed=3)
    hold(s, *attend(s, max_q=max(new), scale=scale), definition(s, scale=scale))


@pytest.mark.parametrize("new,ctx", [([1, 1], [600, 77]), ([200], [600])])
def test_attention_of_large_scores(new, ctx):
    """Scores far apart: one key takes all the weight, the others underflow."""
    s = make(new, ctx, 2, 1, 64, 16, "float16", seed=4)
    s["q"] *= 30
    hold(s, *attend(s, max_q=max(new)), definition(s))


@pytest.mark.parametrize("new", [[1, 1], [180, 20]])
def test_attention_strided_rows_and_other_stream(new):
    """q as a slice of a projection's rows; the call on a stream of its own; the same bits again."""
    torch = _torch()
    from tokenvector.inference_b200.generation import paged_attention
    s = make(new, [400, 90], 6, 2, 64, 16, "bfloat16", seed=5)
    wide = torch.zeros((s["q"].shape[0], 10, 3 * 64), dtype=s["q"].dtype, device="cuda")
    wide[:, 2:8, 64:128] = s["q"]
    want, lse = attend(s, max_q=max(new))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got, lse2 = paged_attention(wide[:, 2:8, 64:128], s["k"], s["v"], s["table"], s["ctx"], s["cu"],
                                        max_q=max(new), return_lse=True)
            assert torch.equal(got, want) and torch.equal(lse, lse2)
    torch.cuda.current_stream().wait_stream(side)
    hold(s, got, lse2, definition(s))


@pytest.mark.parametrize("new", [1, 160])
def test_attention_offsets_past_32_bits(new):
    """Pages whose elements lie behind 2^31 of the cache's start."""
    torch = _torch()
    page, heads, dim = 64, 8, 128
    pages = (1 << 31) // (page * heads * dim) + 40
    k = torch.empty((pages, page, heads, dim), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[pages - 1, 3, pages - 5, pages - 17, 0]], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(9)
    for p in table[0].tolist():
        for t in (k, v):
            t[p] = torch.randn((page, heads, dim), device="cuda", generator=gen).half()
    q = torch.randn((new, heads, dim), device="cuda", generator=gen).half()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(q=q, k=k, v=v, table=table, ctx=i32([5 * page - 9]), cu=i32([0, new]), new=[new], lens=[5 * page - 9])
    hold(s, *attend(s, max_q=new), definition(s))


@pytest.mark.parametrize("new", [1, 150])
def test_attention_reads_no_page_outside_the_cache(new):
    """A page number out of range is reported and read as zeros; the context stays usable."""
    torch = _torch()
    from tokenvector.inference_b200 import _native as N
    clean()
    s = make([new], [300], 2, 2, 64, 16, "float16", seed=6)
    bad = dict(s, table=s["table"].clone())
    bad["table"][0, 3] = s["k"].shape[0] + 1000
    bad["table"][0, 5] = -1
    got, lse = attend(bad, max_q=new)
    assert N.lib().tvq_device_error(None) == N.TVQ_ERR_INVALID and "page" in N.last_error()
    clean()
    zero = dict(s, k=s["k"].clone(), v=s["v"].clone())
    for col in (3, 5):
        zero["k"][s["table"][0, col].long()] = 0
        zero["v"][s["table"][0, col].long()] = 0
    hold(zero, got, lse, definition(zero))


@pytest.mark.parametrize("page", [8, 64, 256])
@pytest.mark.parametrize("new,ctx", [([1, 1], [1000, 77]), ([9, 2], [700, 130]), ([300, 40], [1300, 900])])
def test_attention_reads_no_page_before_the_window(new, ctx, page):
    """Pages that lie before every window are free for others: any entry, any values."""
    torch = _torch()
    clean()
    window = 50
    s = make(new, ctx, 4, 2, 64, page, "float16", seed=page)
    want = definition(s, window=window)
    table = s["table"].clone()
    for i, (n, c) in enumerate(zip(new, ctx)):
        for col in range(max(0, c - n - window + 1) // page):
            old = table[i, col].long()
            s["k"][old] = float("nan")
            s["v"][old] = float("inf")
            if col % 2:
                table[i, col] = -1
    hold(s, *attend(dict(s, table=table), max_q=max(new), window=window), want)
    clean()


def test_attention_without_cu_and_without_rows():
    torch = _torch()
    from tokenvector.inference_b200.generation import paged_attention
    s = make([1, 1, 1], [30, 500, 64], 4, 4, 64, 16, "float16", seed=8)
    a, _ = attend(s, max_q=1)
    out = torch.empty_like(s["q"])
    b = paged_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], out=out)
    assert b is out and torch.equal(a, b)
    none = paged_attention(s["q"][:0], s["k"], s["v"], s["table"][:0], s["ctx"][:0])
    assert none.shape == (0, 4, 64)


def test_attention_in_a_captured_graph():
    torch = _torch()
    from tokenvector.inference_b200.generation import paged_attention
    s = make([1, 1], [900, 33], 8, 2, 128, 16, "bfloat16", seed=10)
    call = lambda: paged_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["cu"], max_q=1)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(got, want)
    assert torch.equal(call(), want)
    # a longer sequence in the same graph: the lengths are read on the device
    s["ctx"].copy_(torch.tensor([450, 20], dtype=torch.int32))
    s["lens"] = [450, 20]
    graph.replay()
    ref = definition(s)
    hold(s, got, ref[1].float(), ref)


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("source,kind", [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float16"),
                                         ("bfloat16", "bfloat16"), ("float16", "bfloat16"), ("bfloat16", "float16")])
@pytest.mark.parametrize("new,ctx,heads,kv_heads,dim,page", [
    ([1, 1, 1], [1, 16, 17], 4, 4, 64, 16), ([5, 0, 40, 1], [5, 9, 90, 300], 6, 2, 80, 8),
    ([300, 7], [300, 4], 8, 1, 128, 64), ([3], [3], 0, 25, 64, 16)])
def test_append_rounds_once_and_writes_only_its_slots(new, ctx, heads, kv_heads, dim, page, source, kind):
    torch = _torch()
    from tokenvector.inference_b200.generation import paged_append
    s = make(new, ctx, max(heads, kv_heads), kv_heads, dim, page, kind, seed=11, head_major=page == 64, junk=False)
    rows = sum(new)
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = (torch.randn((rows, (heads + 2 * kv_heads) * dim), device="cuda", generator=gen) * 3).to(getattr(torch, source))
    wide.view(-1)[::997] = 1e-7
    wide.view(-1)[5::1009] = 6.0e4
    q = wide[:, :heads * dim].unflatten(1, (heads, dim)) if heads else None
    k = wide[:, heads * dim:(heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    v = wide[:, (heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim))
    want_k, want_v = s["k"].clone(), s["v"].clone()
    r = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        for j in range(n):
            p = c - n + j
            if p >= 0:
                pg = int(s["table"][i, p // page])
                want_k[pg, p % page] = k[r].double().to(want_k.dtype)
                want_v[pg, p % page] = v[r].double().to(want_v.dtype)
            r += 1
    got = paged_append(k, v, s["k"], s["v"], s["table"], s["ctx"], s["cu"], q=q)
    assert torch.equal(s["k"], want_k) and torch.equal(s["v"], want_v)
    assert (got is None) if q is None else torch.equal(got, q.double().to(got.dtype))
    clean()


def test_append_drops_rows_without_a_page():
    torch = _torch()
    from tokenvector.inference_b200 import _native as N
    from tokenvector.inference_b200.generation import paged_append
    s = make([1, 1, 1], [17, 40, 90], 2, 2, 64, 16, "float16", seed=12, junk=False)
    table = s["table"].clone()
    table[0, 1] = -1
    table[1, 2] = s["k"].shape[0]
    before = s["k"].clone()
    x = torch.ones((3, 2, 64), device="cuda")
    paged_append(x, x, s["k"], s["v"], table[:, :5], s["ctx"])  # the third's page is behind the table's columns
    assert N.lib().tvq_device_error(None) == N.TVQ_ERR_INVALID and "page" in N.last_error()
    assert torch.equal(s["k"], before)
    clean()


def test_append_then_attend_is_one_decode_step():
    """A prompt in one call equals its tokens one at a time (each within the tolerance of the definition)."""
    torch = _torch()
    from tokenvector.inference_b200.generation import paged_append, paged_attention
    n, heads, dim = 41, 4, 64
    s = make([n], [n], heads, heads, dim, 16, "float16", seed=13, junk=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows = torch.randn((n, 3, heads, dim), device="cuda", generator=gen)
    q = paged_append(rows[:, 1], rows[:, 2], s["k"], s["v"], s["table"], s["ctx"], s["cu"], q=rows[:, 0])
    s["q"] = q
    want = definition(s)
    hold(s, *attend(s), want)
    step = torch.empty_like(q)
    lse = torch.empty((n, heads), device="cuda")
    s["k"].fill_(float("nan"))
    s["v"].fill_(float("nan"))
    for t in range(n):
        ctx = torch.tensor([t + 1], dtype=torch.int32, device="cuda")
        one = paged_append(rows[t:t + 1, 1], rows[t:t + 1, 2], s["k"], s["v"], s["table"], ctx, q=rows[t:t + 1, 0])
        step[t:t + 1], lse[t:t + 1] = paged_attention(one, s["k"], s["v"], s["table"], ctx, return_lse=True)
    hold(s, step, lse, want)
    clean()
