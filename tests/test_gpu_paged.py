"""The paged cache operators on the device against plain 64-bit forms."""
import numpy as np
import pytest

import paged_helpers as ph

pytestmark = pytest.mark.gpu

VALUES = {"f32": 2.0**-24, "bf16": 2.0**-8}


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8}[name]


class Step:
    """Pools full of data, a step over them and its packed rows, all from one
    seed; `k`/`v`/`q` are slices of one fused row when `fused`."""

    def __init__(self, starts, counts, heads=14, kv=2, hd=64, values="f32", cache="bf16", window=0, sinks=0, seed=0,
                 fused=True, shift=0, spare=3):
        import torch
        import llm_inference_edu_b200 as qb
        rng = np.random.default_rng(seed)
        self.starts, self.counts, self.heads, self.kv, self.hd = starts, counts, heads, kv, hd
        self.values, self.cache_dtype, self.window, self.sinks = values, cache, window, sinks
        ends = [a + c for a, c in zip(starts, counts)]
        width = max(1, -(-max(ends) // 16)) + 1
        pages = sum(-(-e // 16) for e in ends) + spare
        order = rng.permutation(pages)
        self.tables = np.full((len(starts), width), -1, np.int64)
        at = 0
        for s, e in enumerate(ends):
            n = -(-e // 16)
            self.tables[s, :n] = order[at:at + n]
            at += n
        T = sum(counts)
        row = rng.standard_normal((T, heads + 2 * kv, hd)).astype(np.float32)
        row[:, :heads] *= 1.5
        if values == "bf16":
            row = ph.bf16(row)
        self.rows = row
        t = torch.from_numpy(row.reshape(T, -1)).to(torch_dtype(values))
        if fused:
            # `shift` elements off the allocation's alignment.
            buf = torch.zeros(T * t.shape[1] + shift, dtype=t.dtype, device="cuda")
            buf[shift:] = t.cuda().reshape(-1)
            t = buf[shift:].view(T, heads + 2 * kv, hd)
            self.q, self.k, self.v = t[:, :heads], t[:, heads:heads + kv], t[:, heads + kv:]
        else:
            t = t.cuda().view(T, heads + 2 * kv, hd)
            self.q, self.k, self.v = (x.contiguous() for x in (t[:, :heads], t[:, heads:heads + kv], t[:, heads + kv:]))
        pools = []
        self.host = []
        for _ in range(2):
            x = rng.standard_normal((pages, kv, 16, hd)).astype(np.float32)
            if cache == "int8":
                q, s = ph.quantize(x)
                pools += [torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()]
                self.host.append(q.astype(np.float64) * s.astype(np.float64)[..., None])
            else:
                x = ph.bf16(x) if cache == "bf16" else x
                pools += [torch.from_numpy(x).to(torch_dtype(cache)).cuda(), None]
                self.host.append(x.astype(np.float64))
        self.cache = qb.PagedCache.from_tensors(pools[0], pools[2], pools[1], pools[3])
        self.plan = qb.PagedPlan(self.cache, self.tables, starts, counts, heads, window=window, sinks=sinks,
                                 dtype=values)
        self.y = torch.full((T, heads, hd), 7.0, dtype=torch_dtype(values), device="cuda")

    def refresh(self):
        """The host pools from what the device holds."""
        c = self.cache
        for i, (p, s) in enumerate(((c.k, c.k_scales), (c.v, c.v_scales))):
            x = p.double()
            if s is not None:
                x = x * s.double()[..., None]
            self.host[i] = x.cpu().numpy()

    def attend(self, **kw):
        import llm_inference_edu_b200 as qb
        qb.paged_attention(self.q, self.cache, self.plan, self.y, **kw)
        return self.y.double().cpu().numpy()

    def want(self, scale=None):
        return ph.attention(self.rows[:, :self.heads].astype(np.float64), *self.host, self.tables, self.starts,
                            self.counts, self.window, self.sinks, scale, bf16_weights=self.values == "bf16",
                            half_step=VALUES[self.values], f16_weights=self.cache_dtype == "int8")

    def check(self, **kw):
        got = self.attend(**kw)
        y, bound = self.want(kw.get("scale"))
        err = np.abs(got - y)
        assert np.isfinite(got).all()
        worst = np.unravel_index(np.argmax(err / bound), err.shape)
        assert (err <= bound).all(), (worst, got[worst], y[worst], bound[worst], float((err > bound).mean()))


SHAPES = [(14, 2, 64), (28, 4, 128), (4, 2, 16), (3, 1, 80), (8, 8, 64), (16, 1, 128), (2, 2, 1), (5, 5, 256), (12, 4, 8)]


# ------------------------------------------------------------ rows -------

@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("values", ["f32", "bf16"])
@pytest.mark.parametrize("cache", ["f32", "bf16", "int8"])
def test_write_and_read_back(heads, kv, hd, values, cache):
    """Stored exactly as the definition says; every other row, scales too,
    keeps its bits."""
    import torch
    import llm_inference_edu_b200 as qb
    s = Step([0, 30, 15, 5, 47], [1, 3, 18, 0, 33], heads, kv, hd, values, cache, seed=hd)
    c = s.cache
    s.rows[3, heads:] = 0.0   # a zero row
    s.k[3], s.v[3] = 0, 0
    before = [None if t is None else t.cpu().clone() for t in (c.k, c.v, c.k_scales, c.v_scales)]
    qb.kv_write(s.k, s.v, c, s.plan)
    ok, ov = (torch.full((sum(s.counts), kv, hd), 3.0, dtype=torch_dtype(values), device="cuda") for _ in range(2))
    qb.kv_read(c, s.plan, ok, ov)
    tok = [(s.tables[i][p // 16], p % 16) for i in range(5) for p in range(s.starts[i], s.starts[i] + s.counts[i])]
    for z, (pool, scales, out) in enumerate(((c.k, c.k_scales, ok), (c.v, c.v_scales, ov))):
        x = s.rows[:, heads + z * kv:heads + (z + 1) * kv]
        want, wscale = before[z], before[2 + z]
        if cache == "int8":
            q, sc = ph.quantize(x)
            back = (q.astype(np.float32) * sc[..., None]).astype(np.float32)
        else:
            back = ph.bf16(x) if cache == "bf16" else x
            q = back
        for i, (page, row) in enumerate(tok):
            want[page, :, row] = torch.from_numpy(q[i]).to(want.dtype)
            if cache == "int8":
                wscale[page, :, row] = torch.from_numpy(sc[i])
        assert torch.equal(pool.cpu(), want)
        if cache == "int8":
            assert torch.equal(scales.cpu(), wscale)
        assert torch.equal(out.cpu(), torch.from_numpy(back).to(out.dtype))


@pytest.mark.parametrize("hd", [64, 128, 80])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_rows_of_any_alignment(hd, shift):
    import torch
    import llm_inference_edu_b200 as qb
    for values in ("f32", "bf16"):
        s = Step([3, 0], [20, 5], 6, 2, hd, values, "int8", shift=shift, seed=shift)
        qb.kv_write(s.k, s.v, s.cache, s.plan)
        n = sum(s.counts) * 2 * hd
        bufs = [torch.full((n + shift,), 3.0, dtype=torch_dtype(values), device="cuda") for _ in range(2)]
        ok, ov = (b[shift:].view(-1, 2, hd) for b in bufs)
        qb.kv_read(s.cache, s.plan, ok, ov)
        for z, out in enumerate((ok, ov)):
            q, sc = ph.quantize(s.rows[:, 6 + 2 * z:8 + 2 * z])
            back = torch.from_numpy((q.astype(np.float32) * sc[..., None]).astype(np.float32))
            assert torch.equal(out.cpu(), back.to(out.dtype))
        assert all((b[:shift] == 3.0).all() for b in bufs)


@pytest.mark.parametrize("hd", [16, 64, 128])
def test_write_edges_of_the_encode(hd):
    """Halves round away from zero; zero, subnormal, huge and non-finite rows."""
    import torch
    import llm_inference_edu_b200 as qb
    s = Step([0], [12], 2, 2, hd, "f32", "int8", fused=False)
    x = np.zeros((12, 2, hd), np.float32)
    x[0, 0, :6] = [127, 0.5, -0.5, 1.5, -2.5, 126.5]
    x[1, 0, 3] = 1e-45
    x[1, 1, :2] = [1e-38, -3e-39]
    x[2, 0, :3] = [3.4e38, -3.4e38, 1.7e38]
    x[2, 1, 5] = np.nan
    x[3, 0, 1] = np.inf
    x[3, 1, hd - 1] = -np.inf
    x[4:] = np.random.default_rng(1).standard_normal((8, 2, hd)) * 10.0 ** np.arange(-20, 20, 5)[:, None, None]
    t = torch.from_numpy(x).cuda()
    qb.kv_write(t, t, s.cache, s.plan)
    q, sc = ph.quantize(x)
    pages = s.tables[0]
    for i in range(12):
        for pool, scales in ((s.cache.k, s.cache.k_scales), (s.cache.v, s.cache.v_scales)):
            assert np.array_equal(pool[pages[0], :, i].cpu().numpy(), q[i]), i
            assert np.array_equal(scales[pages[0], :, i].cpu().numpy(), sc[i], equal_nan=True), i
    ok, ov = torch.empty_like(t), torch.empty_like(t)
    qb.kv_read(s.cache, s.plan, ok, ov)
    with np.errstate(over="ignore"):
        back = q.astype(np.float32) * sc[..., None]
    assert np.array_equal(ok.cpu().numpy(), back, equal_nan=True)


def test_read_whole_sequences_that_share_pages():
    import torch
    import llm_inference_edu_b200 as qb
    s = Step([40], [1], 2, 2, 64, "bf16", "int8")
    t = np.array([s.tables[0][:3], s.tables[0][:3]])
    plan = qb.PagedPlan(s.cache, t, [0, 0], [41, 17], 2, dtype="bf16")
    k, v = (torch.zeros(58, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    qb.kv_read(s.cache, plan, k, v)
    flat = torch.from_numpy(s.host[0][t[0]]).permute(0, 2, 1, 3).reshape(48, 2, 64).float().to(torch.bfloat16)
    assert torch.equal(k.cpu(), torch.cat([flat[:41], flat[:17]]))
    with pytest.raises(qb.CacheError) as e:
        qb.kv_write(k, v, s.cache, plan)
    assert e.value.kind == "InvalidState"


# ------------------------------------------------------- attention -------

@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("values", ["f32", "bf16"])
@pytest.mark.parametrize("cache", ["f32", "bf16", "int8"])
def test_single_tokens(heads, kv, hd, values, cache):
    Step([0, 1, 15, 16, 31, 100, 257], [1] * 7, heads, kv, hd, values, cache, seed=hd + heads).check()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "int8"), ("bf16", "int8"), ("f32", "f32")])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("start", [1023, 4095, 20000])
def test_one_long_sequence(values, cache, heads, kv, hd, start):
    Step([start], [1], heads, kv, hd, values, cache, seed=start).check()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "int8"), ("bf16", "int8")])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (28, 4, 128), (4, 4, 128), (16, 2, 64), (9, 1, 64), (6, 2, 24)])
def test_chunks(values, cache, heads, kv, hd):
    """From two tokens to several hundred, from position 0 and behind odd
    lengths, with single tokens and an idle sequence among them."""
    Step([0, 7, 300, 64, 0, 129, 33], [2, 3, 5, 1, 37, 128, 0], heads, kv, hd, values, cache, seed=hd).check()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "int8"), ("bf16", "int8")])
@pytest.mark.parametrize("heads,kv,hd,start,count", [(14, 2, 64, 0, 512), (7, 1, 128, 0, 301), (7, 1, 128, 1500, 260),
                                                     (2, 2, 64, 1000, 515), (2, 1, 128, 3000, 65), (1, 1, 64, 0, 1)])
def test_long_chunks(values, cache, heads, kv, hd, start, count):
    Step([start], [count], heads, kv, hd, values, cache, seed=count).check()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "int8"), ("f32", "int8"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 0), (100, 20), (128, 130), (1000, 4), (64, 64)])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (7, 1, 128)])
def test_windows(values, cache, window, sinks, heads, kv, hd):
    Step([0, 5, 63, 700, 1200, 90], [1, 40, 1, 3, 70, 200], heads, kv, hd, values, cache, window, sinks,
         seed=window + sinks).check()


@pytest.mark.parametrize("window", [271, 288, 2**31 - 1])
@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "int8"), ("f32", "f32")])
def test_windows_about_as_long_as_the_sequence(window, values, cache):
    Step([0, 71], [1, 200], 14, 2, 64, values, cache, window, 3, seed=2).check()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "int8")])
@pytest.mark.parametrize("scale", [1.0, 0.01, 3.5])
def test_scales(values, cache, scale):
    Step([100, 0, 40], [1, 3, 50], 14, 2, 64, values, cache, seed=5).check(scale=scale)


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("values", ["f32", "bf16"])
def test_queries_of_any_alignment(shift, values):
    Step([100, 0, 40], [1, 3, 50], 14, 2, 64, values, "bf16", shift=shift).check()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "int8"), ("bf16", "int8")])
@pytest.mark.parametrize("hd", [64, 128, 32])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5)])
def test_hidden_values_have_no_influence(values, cache, hd, window, sinks):
    """NaN and infinity wherever a row may not look: behind the sequence's
    end, in pages out of the window, in free pages, and in later tokens of
    the same chunk (those rows themselves see them and turn NaN)."""
    import torch
    starts, counts = [100, 10, 0, 333, 70], [1, 2, 70, 40, 150]
    s = Step(starts, counts, 14, 2, hd, values, cache, window, sinks, seed=hd)
    want, bound = s.want()
    c = s.cache
    hidden = np.ones((c.pages, 16), bool)
    for i, (a, n) in enumerate(zip(starts, counts)):
        for p in range(a + n):
            if any(ph.sees(t, p, window, sinks) for t in range(a, a + n)):
                hidden[s.tables[i][p // 16], p % 16] = False
    page, row = (torch.from_numpy(x).cuda() for x in np.nonzero(hidden))
    # The last two tokens of the chunks of 2, 70, 40 and 150 spoil the rows that see them.
    spoiled = np.zeros(sum(counts), bool)
    where = [(1, 11), (2, 68), (2, 69), (3, 371), (4, 219), (4, 150)]
    for i, p in where:
        t0 = sum(counts[:i])
        for t in range(counts[i]):
            spoiled[t0 + t] |= bool(ph.sees(starts[i] + t, p, window, sinks))
    for bad in (float("nan"), float("inf"), -float("inf")):
        if cache == "int8":
            for t in (c.k_scales, c.v_scales):
                t[page, :, row] = bad
        else:
            for t in (c.k, c.v):
                t[page, :, row] = bad
        for i, p in where:
            g, r = int(s.tables[i][p // 16]), p % 16
            for t in ((c.k_scales, c.v_scales) if cache == "int8" else (c.k, c.v)):
                t[g, :, r] = float("nan")
        got = s.attend()
        assert np.isnan(got[spoiled]).all(), bad
        assert (np.abs(got - want) <= bound)[~spoiled].all(), bad


def test_infinite_values_among_visible_ones():
    """What the formula gives: an infinite V element reaches the rows that
    see it, in its dimension only."""
    for hd, cache in ((64, "bf16"), (128, "bf16"), (32, "f32")):
        s = Step([40, 0], [30, 60], 7, 1, hd, "f32", cache, seed=3)
        g, r = int(s.tables[0][3]), 2     # position 50 of sequence 0
        s.cache.v[g, 0, r, 5] = float("inf")
        want, bound = s.want()            # without it
        got = s.attend()
        after = np.zeros(got.shape, bool)
        after[10:30, :, 5] = True         # tokens at positions 50 .. 69
        assert (got[after] == np.inf).all()
        assert (np.abs(got - want) <= bound)[~after].all()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "int8"), ("f32", "int8"), ("bf16", "bf16")])
@pytest.mark.parametrize("hd", [64, 128])
def test_large_scores(values, cache, hd):
    """Scores far apart and far from zero: the softmax of one dominant key,
    of a maximum that comes late, and of equal scores of large size."""
    s = Step([600, 300, 0], [1, 90, 40], 14, 2, hd, values, cache, seed=9)
    import torch
    s.q[:, ::2] *= 30
    s.rows[:, 0:14:2] *= 30
    if values == "bf16":
        s.rows[:, :14] = s.q.float().cpu().numpy()
    s.q[:, 1] = 0
    s.rows[:, 1] = 0
    s.check()


@pytest.mark.parametrize("values,cache", [("f32", "bf16"), ("bf16", "int8"), ("f32", "int8"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("hd", [64, 128])
def test_queries_that_are_not_finite(values, cache, hd):
    """A NaN or infinity in a query makes that head's row NaN and no other."""
    s = Step([100, 5, 40], [1, 3, 60], 14, 2, hd, values, cache, seed=6)
    want, bound = s.want()
    spoiled = np.zeros(want.shape[:2], bool)
    for t, h, d, x in ((0, 3, 0, np.nan), (2, 0, 5, np.inf), (30, 13, hd - 1, -np.inf), (63, 7, 1, np.nan)):
        s.q[t, h, d] = x
        spoiled[t, h] = True
    got = s.attend()
    assert np.isnan(got[spoiled]).all()
    assert (np.abs(got - want) <= bound)[~spoiled].all()


@pytest.mark.parametrize("values", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("up", [1e-30, 1e-12, 1e12, 1e25])
def test_sizes_of_quantised_rows(values, hd, up):
    """Queries against keys, and values, of sizes far from 1: the powers of
    two that the f16 operands are taken at."""
    import torch
    s = Step([300, 5, 40], [1, 3, 60], 14, 2, hd, values, "int8", seed=8)
    s.cache.v_scales.mul_(up if up < 1e20 else 1e20)
    s.cache.k_scales.mul_(1.0 / up)
    s.q.mul_(up)
    s.rows[:, :14] = s.q.float().cpu().numpy()
    s.refresh()
    s.check()


def test_value_rows_of_very_different_sizes():
    """V scales that vary by 2^20 within a page, and zero scales."""
    import torch
    for values in ("f32", "bf16"):
        s = Step([300, 5, 40], [1, 3, 60], 14, 2, 64, values, "int8", seed=11)
        e = torch.randint(-10, 11, s.cache.v_scales.shape, device="cuda").float()
        s.cache.v_scales.mul_(torch.exp2(e))
        s.cache.v_scales[::3] = 0
        s.refresh()
        s.check()
    s.cache.v_scales.zero_()
    assert (s.attend() == 0).all()


def test_order_of_items_does_not_change_results():
    """The same call twice, and each sequence alone, bit for bit where the
    plan cuts them alike; a repeated call always."""
    s = Step([900, 20, 0, 511], [1, 60, 200, 4], 14, 2, 64, "f32", "int8", seed=4)
    a = s.attend()
    s.y.fill_(5)
    assert np.array_equal(a, s.attend())


# ------------------------------------------------------------ calls ------

def test_a_step_through_the_operators():
    """Prompt chunk, then single tokens, through rope, write and attention as
    a layer makes them, against 64-bit attention over what was stored."""
    import torch
    import llm_inference_edu_b200 as qb
    H, KV, hd = 14, 2, 64
    cache = qb.PagedCache(40, KV, hd, "int8")
    rng = np.random.default_rng(0)
    tables = rng.permutation(40).reshape(2, 20)
    lens = [0, 0]
    for counts in ([70, 33], [1, 1], [1, 1], [0, 5], [3, 1]):
        T = sum(counts)
        rows = torch.from_numpy(rng.standard_normal((T, (H + 2 * KV) * hd)).astype(np.float32)).cuda()
        at = 0
        for s in range(2):
            for lo, heads in ((0, H), (H * hd, KV)):
                if not counts[s]:
                    continue
                x = rows[at:at + counts[s], lo:lo + heads * hd].contiguous()
                y = torch.empty_like(x)
                qb.rope(x, y, counts[s], heads, hd, lens[s], 1e6)
                rows[at:at + counts[s], lo:lo + heads * hd] = y
            at += counts[s]
        q = rows[:, :H * hd].view(T, H, hd)
        k = rows[:, H * hd:(H + KV) * hd].view(T, KV, hd)
        v = rows[:, (H + KV) * hd:].view(T, KV, hd)
        plan = qb.PagedPlan(cache, tables, lens, counts, H, window=60, sinks=4)
        y = torch.empty(T, H, hd, device="cuda")
        qb.kv_write(k, v, cache, plan)
        qb.paged_attention(q, cache, plan, y)
        host = [(p.double() * s.double()[..., None]).cpu().numpy()
                for p, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales))]
        want, bound = ph.attention(q.double().cpu().numpy(), *host, tables, lens, counts, 60, 4)
        assert (np.abs(y.double().cpu().numpy() - want) <= bound).all()
        lens = [a + c for a, c in zip(lens, counts)]


def test_captured_and_replayed():
    """Write and attention in a CUDA graph, replayed over other values and
    beside eager calls on another stream that use the same plan."""
    import torch
    import llm_inference_edu_b200 as qb
    s = Step([2000, 100, 0], [1, 20, 3], 14, 2, 64, "f32", "int8", seed=1)
    qb.kv_write(s.k, s.v, s.cache, s.plan)
    qb.paged_attention(s.q, s.cache, s.plan, s.y)
    torch.cuda.synchronize()
    graphs = []
    outs = [torch.zeros_like(s.y) for _ in range(2)]
    for y in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qb.kv_write(s.k, s.v, s.cache, s.plan)
            qb.paged_attention(s.q, s.cache, s.plan, y)
        graphs.append(g)
    s.q.mul_(0.5)
    s.k.mul_(2.0)
    torch.cuda.synchronize()
    qb.kv_write(s.k, s.v, s.cache, s.plan)
    qb.paged_attention(s.q, s.cache, s.plan, s.y)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(3)]
    third = torch.zeros_like(s.y)
    for _ in range(3):
        for g, st in zip(graphs, side):
            with torch.cuda.stream(st):
                g.replay()
        qb.paged_attention(s.q, s.cache, s.plan, third, stream=side[2].cuda_stream)
    torch.cuda.synchronize()
    for y in outs + [third]:
        assert torch.equal(y, s.y)


def test_other_streams():
    import torch
    import llm_inference_edu_b200 as qb
    s = Step([3000, 100], [1, 40], 14, 2, 64, "f32", "bf16", seed=2)
    first = s.attend()
    st = torch.cuda.Stream()
    y = torch.zeros_like(s.y)
    with torch.cuda.stream(st):
        qb.paged_attention(s.q, s.cache, s.plan, y)
    st.synchronize()
    assert np.array_equal(first, y.double().cpu().numpy())
    y.zero_()
    torch.cuda.synchronize()
    qb.paged_attention(s.q, s.cache, s.plan, y, stream=0)
    torch.cuda.synchronize()
    assert np.array_equal(first, y.double().cpu().numpy())


def test_refusals_leave_outputs_alone():
    import torch
    import llm_inference_edu_b200 as qb
    s = Step([100, 3], [1, 2], 14, 2, 64, "f32", "bf16")
    before = s.cache.k.clone()
    with pytest.raises(qb.CacheError):
        qb.paged_attention(s.q[:2], s.cache, s.plan, s.y)
    with pytest.raises(qb.CacheError):
        qb.paged_attention(s.q, s.cache, s.plan, s.y, scale=float("nan"))
    with pytest.raises(qb.CacheError):
        qb.kv_write(s.k[:1], s.v, s.cache, s.plan)
    with pytest.raises(qb.CacheError):
        qb.kv_write(s.k[:1].expand(3, -1, -1), s.v, s.cache, s.plan)
    for bad in (s.k.to(torch.bfloat16), s.k[..., :32], s.k.transpose(0, 1), s.k.cpu()):
        with pytest.raises(ValueError):
            qb.kv_write(bad, s.v, s.cache, s.plan)
    with pytest.raises(ValueError):
        qb.paged_attention(s.q, s.cache, s.plan, torch.empty(6, 14, 64, device="cuda")[::2])
    with pytest.raises(qb.CacheError):
        qb.paged_attention(s.y, s.cache, s.plan, s.y)
    with pytest.raises(qb.CacheError):
        qb.kv_read(s.cache, s.plan, s.k, s.k)
    other = qb.PagedCache(4, 2, 64, "bf16")
    with pytest.raises(qb.CacheError):
        qb.paged_attention(s.q, other, s.plan, s.y)
    torch.cuda.synchronize()
    assert (s.y == 7.0).all() and torch.equal(s.cache.k, before)


def test_offsets_past_32_bits():
    """Pages in the last gigabytes of pools whose byte and element offsets
    pass 2^31 and 2^32."""
    import torch
    import llm_inference_edu_b200 as qb
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 24 GB")
    KV, hd, H = 4, 128, 8
    pages = (4_300_000_000 // (KV * 16 * hd)) + 50        # 4.3e9 elements a pool
    for cache in ("int8", "bf16"):
        dt = torch_dtype(cache)
        k, v = (torch.empty((pages, KV, 16, hd), dtype=dt, device="cuda") for _ in range(2))
        ks, vs = ((torch.empty((pages, KV, 16), device="cuda") for _ in range(2)) if cache == "int8" else (None, None))
        c = qb.PagedCache.from_tensors(k, v, ks, vs)
        tables = pages - 1 - np.arange(20).reshape(2, 10)
        starts, counts = [0, 0], [150, 2]
        plan = qb.PagedPlan(c, tables, starts, counts, H, dtype="f32")
        x = torch.randn(152, H + 2 * KV, hd, device="cuda")
        y = torch.empty(152, H, hd, device="cuda")
        qb.kv_write(x[:, H:H + KV], x[:, H + KV:], c, plan)
        qb.paged_attention(x[:, :H], c, plan, y)
        lo = pages - 20
        host = []
        for p, s in ((k, ks), (v, vs)):
            t = p[lo:].double()
            host.append((t * s[lo:].double()[..., None] if s is not None else t).cpu().numpy())
        want, bound = ph.attention(x[:, :H].double().cpu().numpy(), *host, tables - lo, starts, counts)
        assert (np.abs(y.double().cpu().numpy() - want) <= bound).all()
        del k, v, ks, vs, c
        torch.cuda.empty_cache()
