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
