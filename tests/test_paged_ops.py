"""CPU checks of the paged cache operators: the plan's admission and layout,
and the refusals that need no device."""
import ctypes as C

import numpy as np
import pytest


def plan(tables, starts, counts, pages=64, kv=2, hd=64, heads=14, window=0, sinks=0, values="f32", cache="bf16"):
    from llm_inference_edu_b200.api import _paged_plan_words
    return _paged_plan_words(tables, starts, counts, pages, kv, hd, heads, window, sinks, values, cache)


def refused(kind, *a, **k):
    from llm_inference_edu_b200 import CacheError
    with pytest.raises(CacheError) as e:
        plan(*a, **k)
    assert e.value.kind == kind
    return e.value


def items(words, p):
    """(small, tile, merges) records of a plan."""
    s = words[p.off_small:p.off_small + 12 * p.small_items].reshape(-1, 12)
    t = words[p.off_tile:p.off_tile + 12 * p.tile_items].reshape(-1, 12)
    m = words[p.off_merges:p.off_merges + 8 * p.merges].reshape(-1, 8)
    return s, t, m


def test_plan_refusals():
    t = np.arange(8).reshape(2, 4)
    refused("ZeroDimension", np.zeros((0, 4), np.int32), [], [])
    refused("ZeroDimension", t, [0, 3], [0, 0])
    refused("ZeroDimension", t, [0, 0], [1, 1], heads=0)
    refused("ZeroDimension", t, [0, 0], [1, 1], pages=0)
    refused("InvalidShape", t, [0, 0], [1, 1], heads=13)
    refused("InvalidShape", t, [0, 0], [1, 1], hd=257)
    refused("DimensionOverflow", t, [0, 0], [1, 1], pages=2**40)
    e = refused("Full", t, [0, 60], [1, 5])
    assert (e.index, e.expected, e.actual) == (1, 64, 65)
    refused("Full", t, [2**32 - 1, 0], [2, 1])
    with pytest.raises(ValueError):
        plan(t, [0, -1], [1, 1])
    with pytest.raises(ValueError):
        plan(t, [0, 0], [1, 1], window=-1)
    with pytest.raises(ValueError):
        plan(t, [0, 0], [1, 1], window=4, sinks=2**64)
    with pytest.raises(ValueError):
        plan(t * 1.0, [0, 0], [1, 1])
    with pytest.raises(ValueError):
        plan(t, [0], [1, 1])


def test_plan_page_ids():
    t = np.arange(8).reshape(2, 4)
    for bad in (64, -1, 2**31, 2**32 + 1):
        x = t.astype(np.int64)
        x[1, 2] = bad
        e = refused("InvalidParameters", x, [0, 40], [1, 1])
        assert (e.index, e.expected) == (6, 64)
        # Nobody looks at the page: past the end, or before the window.
        plan(x, [0, 30], [1, 1])
        # Position 60 sees 60 - window + 1 and later; the bad page ends at 47.
        plan(x, [0, 60], [1, 4], window=13)
        refused("InvalidParameters", x, [0, 60], [1, 4], window=14)
        refused("InvalidParameters", x, [0, 60], [1, 4], window=12, sinks=33)
        plan(x, [0, 60], [1, 4], window=12, sinks=32)
    # A sequence without new tokens is not followed.
    x[1, :] = -1
    plan(x, [0, 2**32 - 1], [1, 0])


def test_plan_marks_rows_that_two_tokens_share():
    t = np.array([[0, 1], [2, 1]])
    assert not plan(t, [3, 0], [1, 1])[1].shared_rows
    assert plan(t, [16, 16], [1, 1])[1].shared_rows      # both write page 1
    assert not plan(t, [16, 16], [1, 0])[1].shared_rows
    assert plan(np.array([[5, 5]]), [15], [2])[1].shared_rows
    assert not plan(np.array([[5, 5]]), [16], [2])[1].shared_rows


def test_plan_words_too_short():
    from llm_inference_edu_b200 import _lib
    t = np.arange(4, dtype=np.int32).reshape(1, 4)
    one = np.array([1], np.uint32)
    step = _lib.PagedStepC(t.ctypes.data, one.ctypes.data, one.ctypes.data, 1, 4, 64, 2, 64, 14, 0, 0, 0, 1)
    words, p = np.full(4096, 7, np.int32), _lib.PagedPlanC()
    L = _lib.lib()
    assert L.qb_paged_plan_build(C.byref(step), words.ctypes.data, 3, C.byref(p)) == 3
    d = _lib.Detail()
    L.qb_last_detail(C.byref(d))
    assert d.buffer == 2 and d.expected > 3 and d.actual == 3 and (words == 7).all()
    assert L.qb_paged_plan_build(C.byref(step), words.ctypes.data, d.expected, C.byref(p)) == 0
    assert p.words == d.expected and (words[p.words:] == 7).all()
    assert L.qb_paged_plan_build(None, words.ctypes.data, 4096, C.byref(p)) == 27
    step.cache_dtype = 3
    assert L.qb_paged_plan_build(C.byref(step), words.ctypes.data, 4096, C.byref(p)) == 39
    step.cache_dtype, step.value_dtype = 1, 2
    assert L.qb_paged_plan_build(C.byref(step), words.ctypes.data, 4096, C.byref(p)) == 39


def test_plan_slots():
    t = np.array([[9, 4, 7], [3, 8, 1]])
    words, p = plan(t, [14, 5], [5, 2])
    slots = words[p.off_slots:p.off_slots + 7]
    assert list(slots) == [9 * 16 + 14, 9 * 16 + 15, 4 * 16, 4 * 16 + 1, 4 * 16 + 2, 3 * 16 + 5, 3 * 16 + 6]


SHAPES = [dict(), dict(window=50, sinks=3), dict(window=17), dict(window=1000, sinks=100), dict(window=1),
          dict(window=40, sinks=33)]


@pytest.mark.parametrize("kw", SHAPES)
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (28, 4, 128), (3, 3, 16), (8, 1, 64)])
@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "int8"), ("f32", "f32")])
def test_plan_items_cover_what_is_seen_once(kw, heads, kv, hd, values, cache):
    """Every (row, KV head) is in one block; a block's items cover its list of
    units without a gap or overlap; every position that a row sees is in one
    unit of its block's list; merges name the items that leave parts."""
    from paged_helpers import sees
    rng = np.random.default_rng(heads * 7 + hd)
    starts = [0, 0, 5, 63, 200, 1200, 4000, 511]
    counts = [1, 70, 1, 2, 33, 1, 300, 0]
    width = 300
    tables = rng.permutation(8 * width).reshape(8, width)
    words, p = plan(tables, starts, counts, pages=8 * width, kv=kv, hd=hd, heads=heads, values=values, cache=cache, **kw)
    G, window, sinks = heads // kv, kw.get("window", 0), kw.get("sinks", 0)
    small, tile, merges = items(words, p)
    assert len(small) + len(tile)
    rows = {}
    parts = {}
    for part, unit in ((small, p.small_unit), (tile, p.tile_unit)):
        cost = part[:, 11]
        assert (np.diff(cost) <= 0).all()
        for seq, g, r0, n, i0, i1, ns, u0, w0, hi, slot, _ in part.tolist():
            assert n > 0 and i0 < i1
            parts.setdefault((seq, g, r0, n, ns, u0, unit), []).append((i0, i1, slot))
    for (seq, g, r0, n, ns, u0, unit), cuts in parts.items():
        for r in range(r0, r0 + n):
            assert (seq, g, r) not in rows
            rows[seq, g, r] = 1
        cuts.sort()
        assert cuts[0][0] == 0 and all(a[1] == b[0] for a, b in zip(cuts, cuts[1:]))
        units = [i if i < ns else u0 + i - ns for i in range(cuts[-1][1])]
        assert len(set(units)) == len(units)
        keys = np.concatenate([np.arange(u * unit, (u + 1) * unit) for u in units])
        for r in {r0, r0 + n // 2, r0 + n - 1}:
            pos = starts[seq] + r // G
            want = np.nonzero(sees(pos, np.arange(pos + 1), window, sinks))[0]
            assert np.isin(want, keys).all()
        mine = [m for m in merges.tolist() if m[:3] == [seq, g, r0]]
        if len(cuts) == 1:
            assert cuts[0][2] == -1 and not mine
        else:
            assert len(mine) == 1 and mine[0][3] == n and mine[0][5] == len(cuts)
            assert [c[2] for c in cuts] == [mine[0][4] + z * mine[0][6] for z in range(len(cuts))]
            assert mine[0][6] >= n * (hd + 2)
            assert (mine[0][4] + len(cuts) * mine[0][6]) * 4 <= p.workspace_bytes
    assert set(rows) == {(s, g, r) for s, c in enumerate(counts) for g in range(kv) for r in range(c * G)}


def test_call_refusals_need_no_device():
    from llm_inference_edu_b200 import _lib
    L = _lib.lib()
    words, p = plan(np.arange(8).reshape(2, 4), [0, 3], [2, 1])
    w = C.c_void_p(1 << 20)
    cache = _lib.PagedCacheC(1 << 20, 2 << 20, None, None, 64, 2, 64, 1)
    x, n = C.c_void_p(3 << 20), 2 * 128 + 128
    q, nq = C.c_void_p(3 << 20), 2 * 896 + 896

    def write(c=cache, pl=p, kn=n, ks=128, vn=n, vs=128, kp=x, wp=w):
        return L.qb_kv_write(kp, kn, ks, x, vn, vs, C.byref(c), C.byref(pl), wp, None)

    def attend(c=cache, pl=p, qn=nq, qs=896, yn=nq, scale=0.125, ws=None, wn=None, yp=C.c_void_p(9 << 20)):
        return L.qb_paged_attention(q, qn, qs, C.byref(c), C.byref(pl), w, yp, yn, scale, ws,
                                    pl.workspace_bytes if wn is None else wn, None)

    assert L.qb_kv_write(x, n, 128, x, n, 128, None, C.byref(p), w, None) == 27
    assert L.qb_kv_read(C.byref(cache), None, w, x, n, 128, x, n, 128, None) == 27
    assert write(kn=n - 1) == 3 and write(vn=n + 1) == 3 and write(ks=127) == 5
    d = _lib.Detail()
    assert write(vn=5) == 3
    L.qb_last_detail(C.byref(d))
    assert (d.buffer, d.expected, d.actual) == (1, n, 5)
    assert write(kp=None) == 27 and write(wp=None) == 27 and write(wp=C.c_void_p((1 << 20) + 4)) == 27
    for field, value in (("pages", 65), ("kv_heads", 1), ("head_dim", 32), ("dtype", 0)):
        other = _lib.PagedCacheC(1 << 20, 2 << 20, None, None, 64, 2, 64, 1)
        setattr(other, field, value)
        assert write(c=other) == 5 and attend(c=other) == 5
    odd = _lib.PagedCacheC((1 << 20) + 8, 2 << 20, None, None, 64, 2, 64, 1)
    assert write(c=odd) == 27 and attend(c=odd) == 27
    _, pq = plan(np.arange(8).reshape(2, 4), [0, 3], [2, 1], cache="int8")
    noscale = _lib.PagedCacheC(1 << 20, 2 << 20, None, None, 64, 2, 64, 2)
    assert write(c=noscale, pl=pq) == 27
    _, twice = plan(np.array([[0, 1], [0, 2]]), [0, 0], [2, 1])
    assert write(pl=twice) == 24
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(scale=bad) == 27
    assert attend(qn=1) == 3 and attend(yn=1) == 3 and attend(yp=None) == 27
    # Y and Q share memory; rows of one buffer side by side do not.
    assert attend(yp=C.c_void_p((3 << 20) + 4)) == 27
    read = lambda kp, ks, vp, vs: L.qb_kv_read(C.byref(cache), C.byref(p), w, kp, 2 * ks + 128, ks, vp,  # noqa: E731
                                               2 * vs + 128, vs, None)
    base = 3 << 20
    assert read(base, 128, base, 128) == 27
    assert read(base, 256, base + 4 * 127, 256) == 27
    assert read(base, 256, base + 4 * 129, 256) == 27
    assert read(base, 256, base + 4 * 200, 300) == 27
    _, long = plan(np.arange(64).reshape(1, 64), [1000], [1])
    if long.workspace_bytes:
        a = 896
        assert attend(pl=long, qn=a, yn=a, wn=long.workspace_bytes - 1, ws=C.c_void_p(1 << 20)) == 3
        assert attend(pl=long, qn=a, yn=a, ws=None) == 27
        assert attend(pl=long, qn=a, yn=a, ws=C.c_void_p((1 << 20) + 4)) == 27


def test_rows_in_the_cache_are_refused():
    # Outputs over the pools or scales that other rows are read from, inputs
    # over those that are written, K's rows stored over V's.
    from llm_inference_edu_b200 import _lib
    L = _lib.lib()
    tables, starts, counts = np.arange(8).reshape(2, 4), [0, 3], [2, 1]
    w, mb = C.c_void_p(1 << 30), 1 << 20
    pool, scales, n = 64 * 2 * 16 * 64, 64 * 2 * 16 * 4, 3 * 128
    for kind, dt, size in (("f32", 0, 4), ("bf16", 1, 2), ("int8", 2, 1)):
        _, p = plan(tables, starts, counts, cache=kind)
        at = [mb, 2 * mb] + ([3 * mb, 4 * mb] if dt == 2 else [None, None])
        cache = _lib.PagedCacheC(*at, 64, 2, 64, dt)

        def write(kp, vp, c=cache):
            return L.qb_kv_write(kp, n, 128, vp, n, 128, C.byref(c), C.byref(p), w, None)

        def read(kp, vp):
            return L.qb_kv_read(C.byref(cache), C.byref(p), w, kp, n, 128, vp, n, 128, None)

        def attend(yp):
            return L.qb_paged_attention(20 * mb, 3 * 896, 896, C.byref(cache), C.byref(p), w, yp, 3 * 896, 0.125, None,
                                        p.workspace_bytes, None)

        inside = [at[0], at[0] + pool * size - 4, at[1], at[1] + 1024, at[1] - n * 4 + 4]
        inside += [at[2], at[2] + scales - 4, at[3] - n * 4 + 4] if dt == 2 else []
        for x in inside:
            for call in (write, read):
                assert call(x, 10 * mb) == 27 and call(10 * mb, x) == 27, (kind, x)
            assert attend(x) == 27, (kind, x)
        for other in ((at[0], at[0] + pool * size - 16, at[2], at[3]), (at[0], at[0], at[2], at[3])):
            assert write(10 * mb, 11 * mb, _lib.PagedCacheC(*other, 64, 2, 64, dt)) == 27
        if dt == 2:
            assert write(10 * mb, 11 * mb, _lib.PagedCacheC(at[0], at[1], at[2], at[2], 64, 2, 64, dt)) == 27


def test_python_wrappers_refuse_host_tensors():
    import torch
    import llm_inference_edu_b200 as qb
    k = torch.zeros(4, 2, 16, 64)
    with pytest.raises(ValueError):
        qb.PagedCache.from_tensors(k, k)
    with pytest.raises(ValueError):
        qb.PagedCache.from_tensors(k.half(), k.half())
    with pytest.raises(ValueError):
        qb.PagedCache.from_tensors(k.to(torch.int8), k.to(torch.int8))
    with pytest.raises(ValueError):
        qb.PagedCache.from_tensors(k[:, :, :8], k[:, :, :8])
