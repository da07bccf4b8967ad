"""Beam search on the GPU: the choice against its definition in 64 bits, the
reordering of the caches against a step-by-step model of it.

The choice's tolerance: a total is score + ((x - max) - z) in f32, three
roundings of 2^-24 relative to terms of at most T = |score| + |x - max| + |z|,
z = ln of an f32 sum (2^-21 relative, so 2^-21 absolute): 2^-22 T + 2^-20.
Logits are given on a coarse grid (2^-5) with scores apart, or checked to be
apart by more than that, so the chosen tokens have to be equal."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


# ---------------------------------------------------------------- selection
def choose(logits, scores, beams, keep, finished=None, eos=None):
    """The definition: lists of each beam, then the best of a request's lists."""
    torch = _torch()
    x = logits.double().cpu()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    rows, vocab = x.shape
    if finished is not None:
        for r in range(rows):
            if finished[r]:
                x[r] = -math.inf
                x[r, eos] = 0.0
    out = []
    for b in range(rows // beams):
        cands = []
        for w in range(beams):
            r = b * beams + w
            order = torch.sort(x[r], descending=True, stable=True)
            top = float(order.values[0])
            z = float((x[r] - top).exp().sum().log())
            for i in range(keep):
                t = float(scores[r]) + ((float(order.values[i]) - top) - z)
                t = -math.inf if math.isnan(t) else t
                terms = abs(float(scores[r])) + abs(float(order.values[i]) - top) + abs(z)
                cands.append((t, w, i, int(order.indices[i]), terms))
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        out.append(cands)
    return out


def check_choice(logits, scores, beams, keep, finished=None, eos=None):
    from tokenvector.inference_b200.generation import beam_select
    got, tokens, parents = beam_select(logits, scores, beams, keep, finished=finished, eos=eos)
    lists = choose(logits, scores.cpu(), beams, keep, None if finished is None else finished.cpu(), eos)
    assert got.shape == tokens.shape == parents.shape == (len(lists), keep)
    got, tokens, parents = got.cpu(), tokens.cpu(), parents.cpu()
    for b, cands in enumerate(lists):
        for i in range(keep):
            t, w, _, token, terms = cands[i]
            tol = 2.0 ** -22 * terms + 2.0 ** -20
            assert (t == -math.inf and got[b, i] == -math.inf) or abs(float(got[b, i]) - t) <= tol, (b, i, t, got[b, i])
            near = [c for c in cands if c[0] == t or abs(c[0] - t) <= 2 * tol]
            if len(near) == 1 or t == -math.inf or all(c[0] == t and c[1] == w for c in near):
                assert (int(parents[b, i]), int(tokens[b, i])) == (w, token), (b, i)
            else:  # totals that f32 cannot tell apart: one of them
                assert (int(parents[b, i]), int(tokens[b, i])) in [(c[1], c[3]) for c in near], (b, i)
        chosen = list(zip(parents[b].tolist(), tokens[b].tolist()))
        assert len(set(chosen)) == keep
    return got, tokens, parents


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("batch,beams,keep,vocab", [
    (1, 1, 1, 1), (1, 1, 1, 50257), (1, 4, 8, 50257), (3, 5, 7, 1001), (2, 8, 16, 50257), (2, 3, 64, 64),
    (1, 64, 64, 4099), (5, 2, 4, 31), (1, 2, 33, 200003), (9, 4, 8, 8192), (2, 16, 32, 12289)])
def test_select_follows_its_definition(batch, beams, keep, vocab, kind):
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(batch + vocab)
    x = torch.randn((batch * beams, vocab), device="cuda", generator=gen) * 3
    scores = -8 * torch.rand(batch * beams, device="cuda", generator=gen)
    check_choice(x.to(getattr(torch, kind)), scores, beams, keep)
    # a coarse grid: ties inside every row
    check_choice(((x * 2).round() / 2).to(getattr(torch, kind)), scores, beams, keep)


@pytest.mark.parametrize("vocab", [1000, 50257])
def test_select_ties_masks_and_extremes(vocab):
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(3)
    beams, keep = 4, 8
    x = (torch.randn((6 * beams, vocab), device="cuda", generator=gen) * 64).round() / 32
    scores = -torch.rand(6 * beams, device="cuda", generator=gen) * 4
    x[0:4] = 1.25                           # all logits equal: the lowest tokens, the best beam
    x[4] = -math.inf                        # a beam without tokens
    x[5, 3:] = -math.inf                    # a beam with three
    x[8:12] = -math.inf                     # a request without any: the lowest places of beam 0
    x[12, ::2] = math.nan                   # masked by NaN
    x[13] = torch.finfo(torch.float32).min  # masked by the lowest value, all of it
    x[14, 7] = 1e30                         # one token takes all
    x[16, 5] = math.inf                     # no distribution
    x[17] = -0.0
    x[17, 9] = 0.0                          # zeros of both signs tie
    scores[20] = -math.inf                  # beams that do not take part
    scores[21] = -math.inf
    got, tokens, parents = check_choice(x, scores, beams, keep)
    assert (got[2] == -math.inf).all() and tokens[2].tolist() == list(range(keep)) and not parents[2].any()
    assert 0 not in parents[4].tolist() or (got[4] == -math.inf).any()


def test_select_sorted_rows_and_one_region():
    """The largest logits side by side, where a part of the row holds all of the list."""
    torch = _torch()
    vocab, beams, keep = 50257, 2, 64
    up = torch.arange(vocab, device="cuda", dtype=torch.float32) / 512
    x = torch.stack([up, up.flip(0), up.roll(25000), (up % 64)])
    check_choice(x, torch.zeros(4, device="cuda"), beams, keep)


def test_select_finished_beams():
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(5)
    beams, keep, vocab = 4, 8, 5003
    x = (torch.randn((3 * beams, vocab), device="cuda", generator=gen) * 64).round() / 32
    x[1] = math.nan  # what a finished beam's logits hold has no influence
    scores = -torch.rand(3 * beams, device="cuda", generator=gen) * 3
    done = torch.zeros(3 * beams, dtype=torch.bool, device="cuda")
    done[[1, 4, 5, 6, 7]] = True
    got, tokens, parents = check_choice(x, scores, beams, keep, done, 7)
    assert tokens[1][:4].tolist() == [7] * 4 and torch.equal(got[1][:4], scores[4:8].cpu().sort(descending=True).values)


def test_select_strided_rows_unaligned_and_other_stream():
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_select
    gen = torch.Generator(device="cuda").manual_seed(6)
    for kind in ("float32", "float16"):
        wide = torch.randn((8, 5021), device="cuda", generator=gen).to(getattr(torch, kind))
        x, scores = wide[:, 3:5004], torch.zeros(8, device="cuda")
        want = check_choice(x, scores, 4, 8)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                got = beam_select(x, scores, 4, 8)
                assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
        torch.cuda.current_stream().wait_stream(side)


# ---------------------------------------------------------------- reordering
def model(table, lens, parents, refs, page):
    """The definition, one row after another: (table, lens, refs, status, copies)."""
    rows, cols = len(table), len(table[0])
    counts = list(refs)
    used = lambda n: min(cols, -(-n // page))  # noqa: E731
    held = [0] * len(refs)
    for r in range(rows):
        for c in range(used(lens[r])):
            if 0 <= table[r][c] < len(refs):
                held[table[r][c]] += 1
                counts[table[r][c]] -= 1
    free = [p for p, n in enumerate(refs) if n == 0]
    out, out_lens, copies, taken, without, tails = [], [], [], 0, 0, set()
    for q in parents:
        if q < 0:
            out.append([-1] * cols)
            out_lens.append(0)
            continue
        n = lens[q]
        row = [table[q][c] if c < used(n) else -1 for c in range(cols)]
        at, fill = n // page, n % page
        tail = row[at] if fill and at < cols else None
        if tail is not None and tail not in tails and refs[tail] == held[tail]:
            tails.add(tail)
        else:
            if tail is not None:
                tails.add(tail)
            if at < cols:
                row[at] = -1
            if at < cols and free:
                row[at] = free.pop(0)
                taken += 1
                if tail is not None:
                    copies.append((tail, row[at], fill))
            else:
                without += 1
        for p in row:
            if p >= 0:
                counts[p] += 1
        out.append(row)
        out_lens.append(n)
    return out, out_lens, counts, [taken, without], copies


def reorder_case(batch, beams, page, prompt, made, layers, heads, dim, seed, *, spare=None, outside=False, major=False):
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    import random
    rng = random.Random(seed)
    shared, total = prompt // page, prompt + made
    mine = -(-total // page) - shared
    rows, cols = batch * beams, -(-(total + 1) // page) + 1
    pool = batch * shared + rows * mine + (2 * rows if spare is None else spare)
    order = list(range(pool))
    rng.shuffle(order)
    table, refs = [], [0] * pool
    for b in range(batch):
        base = order[b * shared:(b + 1) * shared]
        for w in range(beams):
            i = batch * shared + (b * beams + w) * mine
            row = base + order[i:i + mine]
            for p in row:
                refs[p] += 1
            table.append(row + [-1] * (cols - len(row)))
    if outside:  # someone else keeps the first request's pages too
        for p in table[0]:
            if p >= 0:
                refs[p] += 1
    parents = [b * beams + rng.randrange(beams) for b in range(batch) for _ in range(beams)]
    shape = (layers, pool, heads, page, dim) if major else (layers, pool, page, heads, dim)
    k = torch.randn(shape, device="cuda", generator=gen).half()
    v = torch.randn(shape, device="cuda", generator=gen).half()
    if major:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    return table, [total] * rows, parents, refs, k, v, page


def check_reorder(table, lens, parents, refs, k, v, page):
    torch = _torch()
    from tokenvector.inference_b200.generation import beam_reorder
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    want = model(table, lens, parents, refs, page)
    want_k, want_v = k.clone(), v.clone()
    for src, dst, fill in want[4]:
        want_k[:, dst, :fill] = want_k[:, src, :fill]
        want_v[:, dst, :fill] = want_v[:, src, :fill]
    for _ in range(2):  # the inputs stay as they are: again gives the same
        t, n, c, status = beam_reorder(i32(table), i32(lens), i32(parents), i32(refs), k, v)
        assert t.tolist() == want[0]
        assert n.tolist() == want[1]
        assert c.tolist() == want[2]
        assert status.tolist() == want[3]
        assert torch.equal(k, want_k) and torch.equal(v, want_v)
    return want


@pytest.mark.parametrize("batch,beams,page,prompt,made,layers,heads,dim", [
    (1, 1, 16, 5, 1, 1, 1, 64), (1, 4, 16, 40, 9, 3, 2, 64), (3, 5, 8, 23, 1, 2, 3, 80), (2, 8, 32, 64, 32, 2, 4, 128),
    (4, 3, 16, 0, 1, 1, 2, 64), (32, 8, 16, 100, 43, 2, 2, 64), (150, 9, 8, 17, 3, 1, 1, 8), (1, 2, 128, 1000, 77, 2, 2, 128)])
def test_reorder_follows_its_definition(batch, beams, page, prompt, made, layers, heads, dim):
    check_reorder(*reorder_case(batch, beams, page, prompt, made, layers, heads, dim, batch + page, major=beams == 5))


def test_reorder_fans_one_prompt_out_to_its_beams():
    """A prompt's row becomes four beams; the prefix stays shared, the last page is copied for three of them."""
    table, lens, _, refs, k, v, page = reorder_case(2, 1, 16, 37, 3, 2, 2, 64, 1, spare=9)
    want = check_reorder(table, lens, [0] * 4 + [1] * 4, refs, k, v, page)
    assert want[3] == [6, 0] and want[2][table[0][0]] == 4
    # beams that shared their last page already, and rows that end
    check_reorder(want[0], want[1], [0, 0, 3, -1, 4, 5, -1, 5], want[2], k, v, page)


def test_reorder_with_pages_kept_outside_and_mixed_lengths():
    case = list(reorder_case(3, 4, 16, 20, 6, 2, 2, 64, 2, outside=True))
    case[1] = [26, 17, 16, 1, 0, 31, 32, 26, 5, 16, 20, 30]
    held = [0] * len(case[3])
    for r in range(12):
        for c in range(-(-case[1][r] // 16)):
            held[case[0][r][c]] += 1
    case[3] = [h + (1 if p in case[0][0][:2] else 0) for p, h in enumerate(held)]
    check_reorder(*case)


def test_reorder_without_free_pages_or_columns():
    table, lens, parents, refs, k, v, page = reorder_case(2, 4, 16, 32, 7, 1, 2, 64, 3, spare=2)
    want = check_reorder(table, lens, [0] * 4 + [5] * 4, refs, k, v, page)
    assert want[3] == [2, 4]
    full = [[p for p in row if p >= 0] for row in table]
    want = check_reorder(full, [3 * 16] * 8, list(range(8)), refs, k, v, page)
    assert want[3] == [0, 8]


def test_reorder_reports_bad_parents_and_pages():
    torch = _torch()
    from tokenvector.inference_b200 import _native as N
    from tokenvector.inference_b200.generation import beam_reorder
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lens, _, refs, k, v, page = reorder_case(1, 3, 16, 32, 7, 1, 2, 64, 4)
    assert N.lib().tvq_device_error(None) == N.TVQ_OK
    t, n, _, _ = beam_reorder(i32(table), i32(lens), i32([0, 3, 1]), i32(refs), k, v)
    assert N.lib().tvq_device_error(None) == N.TVQ_ERR_INVALID
    assert t[1].tolist() == [-1] * len(table[0]) and int(n[1]) == 0
    table[1][2] = len(refs) + 5
    before = k.clone()
    beam_reorder(i32(table), i32(lens), i32([0, 1, 1]), i32(refs), k, v)
    assert N.lib().tvq_device_error(None) == N.TVQ_ERR_INVALID and "page" in N.last_error()
    assert torch.equal(k, before)
    assert N.lib().tvq_device_error(None) == N.TVQ_OK
