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


def test_positions_stay_below_a_tile_of_two_to_the_31():
    """The kernels count a tile past a sequence's end in 32 bits."""
    from llm_inference_edu_b200 import _lib
    tables = np.zeros((1, 4), np.int32)      # only the first entry is looked at
    start, one = np.array([0], np.uint32), np.array([1], np.uint32)
    out, words = _lib.PagedPlanC(), np.zeros(4, np.int32)

    def build(width):
        step = _lib.PagedStepC(tables.ctypes.data, start.ctypes.data, one.ctypes.data, 1, width, 64, 2, 64, 14, 0, 0, 0, 1)
        return _lib.lib().qb_paged_plan_build(C.byref(step), words.ctypes.data, 4, C.byref(out))

    assert build(0x07fffff0) == 3            # InvalidLength: four words do not hold it
    assert build(0x07fffff1) == build(0x07ffffff) == build(2**40) == refused_kind("DimensionOverflow")


def refused_kind(kind):
    """The status of an error kind, from a call that is refused with it."""
    from llm_inference_edu_b200 import _lib
    refused(kind, np.zeros((1, 4), np.int32), [0], [1], pages=2**40)
    step = _lib.PagedStepC(None, None, None, 1, 4, 2**40, 2, 64, 14, 0, 0, 0, 1)
    return _lib.lib().qb_paged_plan_build(C.byref(step), None, 0, C.byref(_lib.PagedPlanC()))
