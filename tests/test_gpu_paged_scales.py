"""Attention over INT8 pages whose V rows have scales far apart, rows of
zeros among them, or scales that are not finite.  The bounds are
paged_helpers.attention's: a row's largest weight times V scale keeps its
place whatever rows the token does not see, or sees with next to no weight,
or sees without a nonzero byte."""
import numpy as np
import pytest

import paged_helpers as ph
from test_gpu_paged import Step

pytestmark = pytest.mark.gpu

SIZES = [("f32", 64), ("bf16", 64), ("f32", 128), ("bf16", 128)]


def place(s, i, p):
    """(page, row) of position p of sequence i."""
    return int(s.tables[i][p // 16]), p % 16


def scale_values(s, i, p, octaves):
    page, row = place(s, i, p)
    s.cache.v_scales[page, :, row] *= 2.0**octaves


def shift_scores(s, where, octaves):
    """Moves the scores of the keys at `where` by about `octaves` factors of
    two, in every head: the queries get a large first element, and those keys
    the first element that goes with it."""
    import torch
    s.q[:, :, 0] = 20.0
    s.rows[:, :s.heads, 0] = 20.0
    k = s.host[0].copy()
    for i, p in where:
        page, row = place(s, i, p)
        k[page, :, row, 0] = octaves * s.hd**0.5 / (20.0 * 1.4427)
    q, sc = ph.quantize(k)
    s.cache.k.copy_(torch.from_numpy(q))
    s.cache.k_scales.copy_(torch.from_numpy(sc))


# Chunks for the tile kernel (more than 16 packed rows) beside rows for the
# step kernel (one token, two).
STARTS, COUNTS = [40, 0, 300, 129, 90], [60, 30, 1, 2, 150]


@pytest.mark.parametrize("values,hd", SIZES)
@pytest.mark.parametrize("octaves", [20, 40, 100])
def test_value_scales_of_later_tokens(values, hd, octaves):
    """The last token of each chunk has V rows that are much larger: earlier
    tokens do not see them."""
    s = Step(STARTS, COUNTS, 14, 2, hd, values, "int8", seed=octaves)
    for i, (a, c) in enumerate(zip(STARTS, COUNTS)):
        scale_values(s, i, a + c - 1, octaves)
    s.refresh()
    s.check()


@pytest.mark.parametrize("values,hd", SIZES)
@pytest.mark.parametrize("octaves", [20, 40, 100])
def test_value_scales_that_left_the_window(values, hd, octaves):
    """The chunk's first token alone sees the large V row."""
    starts, counts, window = [200, 333], [80, 2], 50
    s = Step(starts, counts, 14, 2, hd, values, "int8", window, 3, seed=octaves)
    for i, a in enumerate(starts):
        scale_values(s, i, a + 1 - window, octaves)
    s.refresh()
    s.check()


@pytest.mark.parametrize("values,hd", SIZES)
@pytest.mark.parametrize("octaves,down", [(40, 20), (40, 60), (60, 60), (30, 50)])
def test_value_scales_of_keys_with_little_weight(values, hd, octaves, down):
    s = Step(STARTS, COUNTS, 14, 2, hd, values, "int8", seed=down)
    where = [(i, p) for i, a in enumerate(STARTS) if a for p in (3, a // 2)]
    shift_scores(s, where, -down)
    for i, p in where:
        scale_values(s, i, p, octaves)
    s.refresh()
    s.check()
