"""What the decoding operators refuse, before any device work (no GPU needed:
the pointers are never dereferenced)."""
import ctypes as C

import pytest

from tokenvector.inference_b200 import _native as N

FAKE = C.c_void_p(4096)
ODD = C.c_void_p(4098)


def i64(*v):
    return (C.c_int64 * len(v))(*v)


def append(**kw):
    a = dict(type=N.TYPE_F16, src=N.TYPE_F32, k=FAKE, v=FAKE, q=None, ss=i64(128, 64, 128, 64, 0, 0), qh=0, qo=None,
             kp=FAKE, vp=FAKE, shape=i64(10, 16, 2, 64), st=i64(2048, 128, 64, 2048, 128, 64), table=FAKE, ts=4,
             cols=4, ctx=FAKE, cu=None, n_seq=3, n_rows=3)
    a.update(kw)
    return N.lib().tvq_dev_paged_append(*a.values(), None)


def attend(**kw):
    a = dict(type=N.TYPE_F16, q=FAKE, qs=i64(128, 64), qh=2, kp=FAKE, vp=FAKE, shape=i64(10, 16, 2, 64),
             st=i64(2048, 128, 64, 2048, 128, 64), table=FAKE, ts=4, cols=4, ctx=FAKE, cu=None, n_seq=3, n_rows=3,
             max_q=1, scale=0.125, window=0, out=FAKE, lse=None, ws=None, wb=0)
    a.update(kw)
    return N.lib().tvq_dev_paged_attention(*a.values(), None)


def select(**kw):
    a = dict(type=N.TYPE_F32, x=FAKE, stride=100, scores=FAKE, fin=None, batch=2, beams=4, keep=8, vocab=100, eos=-1,
             s=FAKE, t=FAKE, p=FAKE, ws=None, wb=0)
    a.update(kw)
    return N.lib().tvq_dev_beam_select(*a.values(), None)


def reorder(**kw):
    a = dict(table=FAKE, ts=4, lens=FAKE, rows=3, cols=4, parents=FAKE, new=3, refs=FAKE, k=FAKE, v=FAKE,
             shape=i64(10, 16, 2, 64, 1), st=i64(0, 2048, 128, 64, 0, 2048, 128, 64), nt=C.c_void_p(8192),
             nl=C.c_void_p(8192), nr=C.c_void_p(8192), status=FAKE, ws=None, wb=0)
    a.update(kw)
    return N.lib().tvq_dev_beam_reorder(*a.values(), None)


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("change,code", [
    (dict(type=N.TYPE_F32), N.TVQ_ERR_INVALID), (dict(type=9), N.TVQ_ERR_INVALID),
    (dict(shape=None), N.TVQ_ERR_INVALID), (dict(st=None), N.TVQ_ERR_INVALID),
    (dict(shape=i64(10, 12, 2, 64)), N.TVQ_ERR_UNSUPPORTED), (dict(shape=i64(10, 4, 2, 64)), N.TVQ_ERR_UNSUPPORTED),
    (dict(shape=i64(10, 2048, 2, 64)), N.TVQ_ERR_UNSUPPORTED), (dict(shape=i64(10, 16, 0, 64)), N.TVQ_ERR_INVALID),
    (dict(shape=i64(10, 16, 2, 60)), N.TVQ_ERR_UNSUPPORTED), (dict(shape=i64(10, 16, 2, 136)), N.TVQ_ERR_UNSUPPORTED),
    (dict(shape=i64(10, 16, 2, 0)), N.TVQ_ERR_UNSUPPORTED), (dict(shape=i64(-1, 16, 2, 64)), N.TVQ_ERR_INVALID),
    (dict(shape=i64(1 << 31, 16, 2, 64)), N.TVQ_ERR_UNSUPPORTED),
    (dict(n_rows=-1), N.TVQ_ERR_INVALID), (dict(n_seq=-1, n_rows=-1), N.TVQ_ERR_INVALID),
    (dict(n_rows=4), N.TVQ_ERR_SIZE), (dict(ts=3), N.TVQ_ERR_SIZE), (dict(table=None), N.TVQ_ERR_INVALID),
    (dict(ctx=None), N.TVQ_ERR_INVALID), (dict(kp=None), N.TVQ_ERR_INVALID), (dict(vp=ODD), N.TVQ_ERR_UNSUPPORTED),
    (dict(st=i64(2048, 124, 64, 2048, 128, 64)), N.TVQ_ERR_UNSUPPORTED),
    (dict(st=i64(2048, -128, 64, 2048, 128, 64)), N.TVQ_ERR_UNSUPPORTED),
    (dict(cols=1 << 31, ts=1 << 31), N.TVQ_ERR_UNSUPPORTED)])
def test_cache_refusals(call, change, code):
    assert call(**change) == code, N.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(src=7), N.TVQ_ERR_INVALID), (dict(k=None), N.TVQ_ERR_INVALID), (dict(v=ODD), N.TVQ_ERR_UNSUPPORTED),
    (dict(ss=i64(126, 64, 128, 64, 0, 0)), N.TVQ_ERR_UNSUPPORTED), (dict(ss=None), N.TVQ_ERR_INVALID),
    (dict(src=N.TYPE_F16, ss=i64(132, 64, 128, 64, 0, 0)), N.TVQ_ERR_UNSUPPORTED),
    (dict(q=FAKE, qh=2), N.TVQ_ERR_INVALID), (dict(q=FAKE, qh=2, qo=ODD), N.TVQ_ERR_UNSUPPORTED),
    (dict(qh=-1), N.TVQ_ERR_INVALID)])
def test_append_refusals(change, code):
    assert append(**change) == code, N.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(qh=3), N.TVQ_ERR_INVALID), (dict(qh=0), N.TVQ_ERR_INVALID), (dict(q=None), N.TVQ_ERR_INVALID),
    (dict(out=None), N.TVQ_ERR_INVALID), (dict(out=ODD), N.TVQ_ERR_UNSUPPORTED), (dict(qs=None), N.TVQ_ERR_INVALID),
    (dict(qs=i64(127, 64)), N.TVQ_ERR_UNSUPPORTED), (dict(max_q=-1), N.TVQ_ERR_INVALID),
    (dict(window=-1), N.TVQ_ERR_INVALID)])
def test_attention_refusals(change, code):
    assert attend(**change) == code, N.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(type=5), N.TVQ_ERR_INVALID), (dict(beams=0), N.TVQ_ERR_UNSUPPORTED), (dict(beams=65), N.TVQ_ERR_UNSUPPORTED),
    (dict(keep=0), N.TVQ_ERR_UNSUPPORTED), (dict(keep=65), N.TVQ_ERR_UNSUPPORTED),
    (dict(keep=9, vocab=8), N.TVQ_ERR_SIZE), (dict(stride=99), N.TVQ_ERR_SIZE), (dict(batch=-1), N.TVQ_ERR_INVALID),
    (dict(fin=FAKE), N.TVQ_ERR_INVALID), (dict(fin=FAKE, eos=100), N.TVQ_ERR_INVALID), (dict(x=None), N.TVQ_ERR_INVALID),
    (dict(x=ODD), N.TVQ_ERR_UNSUPPORTED), (dict(t=None), N.TVQ_ERR_INVALID), (dict(), N.TVQ_ERR_SIZE),
    (dict(ws=ODD, wb=1 << 30), N.TVQ_ERR_INVALID)])
def test_select_refusals(change, code):
    assert select(**change) == code, N.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(shape=i64(10, 24, 2, 64, 1)), N.TVQ_ERR_UNSUPPORTED), (dict(shape=i64(10, 16, 2, 65, 1)), N.TVQ_ERR_UNSUPPORTED),
    (dict(rows=70000), N.TVQ_ERR_UNSUPPORTED), (dict(new=-1), N.TVQ_ERR_INVALID), (dict(ts=2), N.TVQ_ERR_SIZE),
    (dict(nt=FAKE), N.TVQ_ERR_INVALID), (dict(nr=FAKE), N.TVQ_ERR_INVALID), (dict(nl=FAKE), N.TVQ_ERR_INVALID),
    (dict(status=None), N.TVQ_ERR_INVALID), (dict(parents=None), N.TVQ_ERR_INVALID), (dict(k=None), N.TVQ_ERR_INVALID),
    (dict(st=i64(4, 2048, 128, 64, 0, 2048, 128, 64)), N.TVQ_ERR_UNSUPPORTED), (dict(), N.TVQ_ERR_SIZE)])
def test_reorder_refusals(change, code):
    assert reorder(**change) == code, N.last_error()


def test_nothing_to_do_is_no_error():
    assert append(n_seq=0, n_rows=0, k=None, kp=None, table=None) == N.TVQ_OK
    assert attend(n_seq=0, n_rows=0, q=None, kp=None, table=None) == N.TVQ_OK
    assert select(batch=0, x=None) == N.TVQ_OK


def test_python_refusals():
    torch = pytest.importorskip("torch")
    from tokenvector.inference_b200 import generation as G
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    t = torch.zeros((1, 2), dtype=torch.int32)
    n = torch.ones(1, dtype=torch.int32)
    row = torch.zeros((1, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        G.paged_attention(row, k, k, t, n)
    with pytest.raises(ValueError, match="CUDA"):
        G.paged_append(row, row, k, k, t, n)
    with pytest.raises(ValueError, match="CUDA"):
        G.beam_select(torch.zeros((4, 9)), torch.zeros(4), 4, 4)
    with pytest.raises(ValueError, match="CUDA"):
        G.beam_reorder(t, n, n, n, k[None], k[None])
    with pytest.raises(ValueError, match="int32"):
        G.beam_reorder(t.long(), n, n, n, k[None], k[None])
