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


def written(starts, counts, heads, hd, values, size, zeros, seed):
    """A step whose whole sequences went through kv_write: V about `size`,
    its rows zero at the positions `zeros` (a function of a sequence)."""
    import torch
    import llm_inference_edu_b200 as qb
    s = Step(starts, counts, heads, 2, hd, values, "int8", seed=seed)
    ends = [a + c for a, c in zip(starts, counts)]
    rng = np.random.default_rng(seed + 1)
    x = rng.standard_normal((2, sum(ends), 2, hd)).astype(np.float32)
    x[1] *= size
    for i, e in enumerate(ends):
        rows = x[1, sum(ends[:i]):sum(ends[:i]) + e]
        rows[[p for p in zeros(i) if p < e]] = 0
    k, v = (torch.from_numpy(t).to(s.q.dtype).cuda() for t in x)
    qb.kv_write(k, v, s.cache, qb.PagedPlan(s.cache, s.tables, [0] * len(ends), ends, heads, dtype=values))
    s.refresh()
    return s


@pytest.mark.parametrize("values,hd", SIZES)
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-5, 1e-7, 1e-9, 1e-18])
def test_value_rows_of_zeros(values, hd, size):
    """A stored row of zeros has scale 1 whatever the others' scales are."""
    starts, counts = [40, 0, 300, 129, 90, 2500], [60, 30, 1, 2, 150, 1]
    few = lambda i: [5, 17, 33, 34, 100, 131] if i != 4 else range(32, 200)  # noqa: E731 (whole pages and tiles of zeros)
    written(starts, counts, 14, hd, values, size, few, seed=3).check()


@pytest.mark.parametrize("values,hd", SIZES)
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-9])
@pytest.mark.parametrize("up", [25, 45])
def test_value_row_of_zeros_with_most_of_the_weight(values, hd, size, up):
    """A first token that takes the attention and has no value: what is left
    of the others is small, and exact."""
    s = written(STARTS, COUNTS, 14, hd, values, size, lambda i: [0], seed=up)
    shift_scores(s, [(i, 0) for i in range(len(STARTS))], up)
    s.refresh()
    s.check()


@pytest.mark.parametrize("values,hd", SIZES)
def test_values_that_are_all_zero(values, hd):
    s = written(STARTS, COUNTS, 14, hd, values, 1.0, lambda i: range(300), seed=1)
    got = s.attend()
    seen = np.repeat(STARTS, COUNTS) < 300
    assert seen.sum() == sum(COUNTS) - 1 and (got[seen] == 0).all()


@pytest.mark.parametrize("values,hd", SIZES)
@pytest.mark.parametrize("order", ["small first", "large first", "mixed", "zeros first"])
def test_value_scales_further_apart_than_a_float(values, hd, order):
    """Equal weights of values that differ by 2^150: the small ones count in
    the denominator.  (Zeros first: rows of zeros, then scales of 2^60.)"""
    import torch
    starts, counts = [40, 0, 300, 129, 90, 6000], [60, 30, 1, 2, 150, 1]
    s = Step(starts, counts, 14, 2, hd, values, "int8", seed=7)
    rng = np.random.default_rng(5)
    c = s.cache
    for i, (a, n) in enumerate(zip(starts, counts)):
        for j, page in enumerate(s.tables[i][:-(-(a + n) // 16)]):
            late = j * 32 >= a + n
            if order == "zeros first":
                if late:
                    c.v_scales[page] *= 2.0**60
                else:
                    c.v[page] = 0
                    c.v_scales[page] = 1.0
                continue
            up = torch.from_numpy(rng.choice([-75.0, 75.0], (2, 16))).float().cuda()
            if order != "mixed":
                up[:] = 75.0 if late == (order == "small first") else -75.0
            c.v_scales[page] *= torch.exp2(up)
    s.refresh()
    s.check()


@pytest.mark.parametrize("values,hd", SIZES)
@pytest.mark.parametrize("how", ["far below", "-inf"])
def test_nan_scale_of_a_key_without_weight(values, hd, how):
    """0 * NaN is NaN for every row that sees the key, wherever its page and
    its tile end, and no other row notices."""
    starts, counts = [40, 0, 300, 129, 90, 3], [60, 30, 1, 2, 150, 1]
    where = [(0, 70), (0, 42), (1, 29), (2, 300), (3, 130), (4, 160), (5, 2)]
    s = Step(starts, counts, 14, 2, hd, values, "int8", seed=12)
    if how == "far below":
        shift_scores(s, where, -300)
    s.refresh()
    want, bound = s.want()
    spoiled = np.zeros(sum(counts), bool)
    for i, p in where:
        page, row = place(s, i, p)
        s.cache.v_scales[page, :, row] = float("nan")
        if how == "-inf":
            # Scores of -inf, or of +inf, which make the row NaN by themselves.
            s.cache.k_scales[page, :, row] = float("inf")
        t0 = sum(counts[:i])
        spoiled[t0 + max(p - starts[i], 0):t0 + counts[i]] = True
    got = s.attend()
    assert np.isnan(got[spoiled]).all()
    assert (np.abs(got - want) <= bound)[~spoiled].all()


@pytest.mark.parametrize("values,hd", SIZES)
def test_scores_that_are_large_before_their_factor(values, hd):
    """Tiny queries, huge keys: scaled Q times bytes times the key's scale
    passes a float's range, the score itself does not.  A token that sees
    only such scores, all negative, still has its result."""
    starts, counts = [0, 0, 40, 0, 129], [1, 40, 60, 2, 1]
    s = Step(starts, counts, 14, 2, hd, values, "int8", seed=21)
    s.q.mul_(2.0**-100)
    s.rows[:, :14] = s.q.float().cpu().numpy()
    s.cache.k_scales.mul_(2.0**115)
    s.refresh()
    s.check()
