"""CPU checks of what the paged cache operators refuse at the ends of their
arguments' ranges."""
import ctypes as C

import numpy as np
import pytest

from test_paged_ops import plan, refused


def test_scales_whose_base_2_form_overflows_are_refused():
    """Scores are taken in units of log2: scale * log2(e) has to be a float."""
    from llm_inference_edu_b200 import _lib
    L = _lib.lib()
    _, p = plan(np.arange(8).reshape(2, 4), [0, 3], [2, 1])
    cache = _lib.PagedCacheC(1 << 20, 2 << 20, None, None, 64, 2, 64, 1)
    for scale in (3e38, 2.3587e38, 3.4028235e38):
        assert L.qb_paged_attention(C.c_void_p(3 << 20), 3 * 896, 896, C.byref(cache), C.byref(p), C.c_void_p(1 << 20),
                                    C.c_void_p(9 << 20), 3 * 896, scale, None, p.workspace_bytes, None) == 27


def test_counts_past_the_table_are_refused_before_anything_is_sized_by_them():
    many = 64
    e = refused("Full", np.zeros((many, 4), np.int32), [0] * many, [2**32 - 1] * many)
    assert (e.index, e.expected, e.actual) == (0, 64, 2**32 - 1)
    e = refused("Full", np.zeros((many, 4), np.int32), [0] * many, [1] * (many - 1) + [2**32 - 1])
    assert e.index == many - 1
