"""Forms of input that the decoding operators and the generator take or refuse
before any device work (no GPU needed: no pointer is dereferenced)."""
import ctypes as C

import pytest

from tokenvector.inference_b200 import _native as N

FAKE = C.c_void_p(4096)


def i64(*v):
    return (C.c_int64 * len(v))(*v)


def test_rows_may_coincide_but_not_overlap():
    """A stride of 0 gets as far as the check of the workspace, a stride below the row does not."""
    for stride, why in ((0, "workspace"), (100, "workspace"), (1, "overlap"), (99, "overlap"), (-1, "overlap")):
        assert N.lib().tvq_dev_beam_select(N.TYPE_F32, FAKE, stride, FAKE, None, 2, 4, 8, 100, -1, FAKE, FAKE, FAKE, None, 0,
                                           None) == N.TVQ_ERR_SIZE
        assert why in N.last_error()
    apart = C.c_void_p(8192)
    for stride, why in ((0, "workspace"), (4, "workspace"), (1, "table_stride"), (-4, "table_stride")):
        assert N.lib().tvq_dev_beam_reorder(FAKE, stride, FAKE, 3, 4, FAKE, 3, FAKE, FAKE, FAKE, i64(10, 16, 2, 64, 1),
                                            i64(0, 2048, 128, 64, 0, 2048, 128, 64), apart, apart, apart, FAKE, None, 0,
                                            None) == N.TVQ_ERR_SIZE
        assert why in N.last_error()


# ---------------------------------------------------------------- the generator
@pytest.fixture
def generator():
    """A generator without a session: what is refused is refused before the device is touched."""
    torch = pytest.importorskip("torch")
    from tokenvector.inference_b200.generation import GPT2Generator
    from tokenvector.inference_b200.gpt2 import GPT2Config
    g = GPT2Generator.__new__(GPT2Generator)
    g.cfg = GPT2Config(vocab=320, d_model=128, n_heads=2, n_layers=2, d_ffn=512, max_pos=64)
    g.page, g.dtype, g.dev = 16, torch.float16, torch.device("cuda", 0)
    return g


@pytest.mark.parametrize("ids", [[320], [3, -1], [2 ** 40], [1, 2, 2 ** 70], [1.5, 2.0], [True, False], [], [[1, 2]], "12"])
def test_generator_refuses_ids_outside_the_vocabulary(generator, ids):
    with pytest.raises(ValueError):
        generator.log_probs(ids)
    with pytest.raises(ValueError):
        generator.generate([[1, 2, 3], ids], 2, 4)


def test_generator_refuses_sequences_longer_than_its_positions(generator):
    with pytest.raises(ValueError, match="positions"):
        generator.log_probs([1] * 65)
    with pytest.raises(ValueError, match="positions"):
        generator.generate([[1], [2] * 62], 2, 3)


@pytest.mark.parametrize("max_new", [0, -1])
def test_generator_refuses_to_make_no_token(generator, max_new):
    with pytest.raises(ValueError, match="max_new"):
        generator.generate([[1, 2]], 2, max_new)


# ---------------------------------------------------------------- several devices
def test_kernel_limits_are_set_on_every_device(tmp_path):
    """The flag that the launchers keep for a kernel's attribute (the two-GPU test of it is in test_gpu_decoding_inputs)."""
    import os
    import shutil
    import subprocess
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "once")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-o", exe, os.path.join(here, "native", "once_per_device.cpp")])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
    csrc = os.path.join(here, "..", "tokenvector", "inference_b200", "csrc")
    for name in ("tvq_paged_attn.cu", "tvq_beam.cu"):  # no flag of the process beside it
        with open(os.path.join(csrc, name)) as f:
            text = f.read()
        assert "cudaFuncSetAttribute" not in text and "allow_smem<" in text


@pytest.mark.parametrize("change", [dict(vocab=319), dict(vocab=321), dict(d_model=64), dict(max_pos=63), dict(n_layers=1),
                                    dict(n_layers=3)])
def test_generator_refuses_weights_of_another_shape(change):
    """Before the session is asked for anything: it is a stand-in."""
    pytest.importorskip("torch")
    from types import SimpleNamespace

    from tokenvector.inference_b200.generation import GPT2Generator
    from tokenvector.inference_b200.gpt2 import GPT2Config, GPT2Weights
    cfg = dict(vocab=320, d_model=128, n_heads=2, n_layers=2, d_ffn=256, max_pos=64)
    session = SimpleNamespace(cfg=GPT2Config(**cfg), device=0)
    with pytest.raises(ValueError, match="shape"):
        GPT2Generator(session, GPT2Weights.random(GPT2Config(**{**cfg, **change})))


# ---------------------------------------------------------------- caches that are written
@pytest.mark.parametrize("place", range(6))
def test_append_refuses_a_cache_whose_entries_coincide(place):
    def append(shape, strides):
        return N.lib().tvq_dev_paged_append(N.TYPE_F16, N.TYPE_F32, FAKE, FAKE, None, i64(128, 64, 128, 64, 0, 0), 0, None,
                                            FAKE, FAKE, i64(*shape), i64(*strides), FAKE, 4, 4, FAKE, None, 3, 3, None)
    strides = [2048, 128, 64, 2048, 128, 64]
    strides[place] = 0
    assert append((10, 16, 2, 64), strides) == N.TVQ_ERR_INVALID and "strides of 0" in N.last_error()


@pytest.mark.parametrize("place", range(8))
def test_reorder_refuses_a_cache_whose_entries_coincide(place):
    strides = [20480, 2048, 128, 64] * 2
    strides[place] = 0
    apart = C.c_void_p(8192)

    def reorder(layers):
        return N.lib().tvq_dev_beam_reorder(FAKE, 4, FAKE, 3, 4, FAKE, 3, FAKE, FAKE, FAKE, i64(10, 16, 2, 64, layers),
                                            i64(*strides), apart, apart, apart, FAKE, None, 0, None)
    assert reorder(3) == N.TVQ_ERR_INVALID and "strides of 0" in N.last_error()
    if place % 4 == 0:  # of a single layer any stride will do
        assert reorder(1) == N.TVQ_ERR_SIZE and "workspace" in N.last_error()


# ---------------------------------------------------------------- gradients
def test_operators_without_a_backward_pass_say_so():
    torch = pytest.importorskip("torch")
    from tokenvector.inference_b200 import generation as G
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    t, n = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    row, x, scores = torch.zeros((1, 2, 64), dtype=torch.float16), torch.zeros((4, 9)), torch.zeros(4)
    grad = lambda a: a.clone().requires_grad_()  # noqa: E731
    calls = [lambda: G.paged_attention(grad(row), k, k, t, n), lambda: G.paged_attention(row, grad(k), k, t, n),
             lambda: G.paged_attention(row, k, grad(k), t, n), lambda: G.paged_append(grad(row), row, k, k, t, n),
             lambda: G.paged_append(row, grad(row), k, k, t, n), lambda: G.paged_append(row, row, k, grad(k), t, n),
             lambda: G.paged_append(row, row, k, k, t, n, q=grad(row)), lambda: G.beam_select(grad(x), scores, 4, 4),
             lambda: G.beam_select(x, grad(scores), 4, 4), lambda: G.beam_reorder(t, n, n, n, grad(k[None]), k[None])]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # (as far as the next check)
            call()
