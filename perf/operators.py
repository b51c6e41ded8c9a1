"""The paged cache operators as they are measured: storing K/V rows (quantised) and reading them back, and attention of
new tokens over the pages, full or with a sliding window and sinks.

A cache is two page pools [pages][kv_heads][16][head_dim] (bf16, or int8 with one f32 scale a row); a sequence's table
maps its positions 16 j .. 16 j + 15 to one page.  Sequence i of a case has `first` new tokens (i = 0) or `rest` (i > 0)
behind `lo` .. `hi` cached positions (spread evenly over the logarithm), so a case's shapes follow from its numbers.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16


def listed():
    return [
        # One decode step's K/V of a 64-sequence batch at the 0.5B shape: the write that every layer of every step makes.
        dict(name="store_step", kind="store", heads=14, kv=2, hd=64, sequences=64, first=1, rest=1, lo=0, hi=1000,
             window=0, sinks=0, values="f32", cache="int8"),
        # A whole prompt of the 7B shape, stored and read back (prefix reuse).
        dict(name="store_prompt", kind="store", heads=28, kv=4, hd=128, sequences=1, first=8192, rest=0, lo=0, hi=0,
             window=0, sinks=0, values="f32", cache="int8"),
        # Several odd chunks behind odd lengths, bf16 activations.
        dict(name="store_ragged", kind="store", heads=28, kv=4, hd=128, sequences=9, first=1531, rest=333, lo=5, hi=4001,
             window=0, sinks=0, values="bf16", cache="int8"),
        # The batch-1 step of the decode benchmark (a context of some hundred positions): latency.
        dict(name="step_one", kind="attend", heads=14, kv=2, hd=64, sequences=1, first=1, rest=0, lo=199, hi=199,
             window=0, sinks=0, values="f32", cache="bf16"),
        # One token behind the longest context that the 0.5B configuration allows.
        dict(name="step_long", kind="attend", heads=14, kv=2, hd=64, sequences=1, first=1, rest=0, lo=32767, hi=32767,
             window=0, sinks=0, values="f32", cache="bf16"),
        # A serving step: 64 sequences of very different lengths over a quantised cache, 7B shape.
        dict(name="step_batch", kind="attend", heads=28, kv=4, hd=128, sequences=64, first=1, rest=1, lo=100, hi=8191,
             window=0, sinks=0, values="bf16", cache="int8"),
        # Five drafted tokens a sequence, checked in one pass.
        dict(name="draft_check", kind="attend", heads=28, kv=4, hd=128, sequences=16, first=5, rest=5, lo=77, hi=4091,
             window=0, sinks=0, values="bf16", cache="bf16"),
        # The 512-token prompt of the benchmark, from position 0.
        dict(name="chunk_512", kind="attend", heads=14, kv=2, hd=64, sequences=1, first=512, rest=0, lo=0, hi=0,
             window=0, sinks=0, values="f32", cache="bf16"),
        # The second half of a long prompt, 7B shape: the largest.
        dict(name="chunk_long", kind="attend", heads=28, kv=4, hd=128, sequences=1, first=4096, rest=0, lo=4096, hi=4096,
             window=0, sinks=0, values="bf16", cache="bf16"),
        # A step that carries one prompt chunk among single tokens, f32 activations over a quantised cache.
        dict(name="mixed", kind="attend", heads=28, kv=4, hd=128, sequences=24, first=509, rest=1, lo=2999, hi=131,
             window=0, sinks=0, values="f32", cache="int8"),
        # Steps that see their last 1024 positions and the first 4, far into their sequences.
        dict(name="window_step", kind="attend", heads=14, kv=2, hd=64, sequences=32, first=1, rest=1, lo=500, hi=32767,
             window=1024, sinks=4, values="f32", cache="int8"),
        # A chunk deep in a long document under an odd window.
        dict(name="window_chunk", kind="attend", heads=28, kv=4, hd=128, sequences=1, first=2001, rest=0, lo=10007, hi=10007,
             window=1001, sinks=4, values="bf16", cache="bf16"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    # The 0.5B and 7B shapes, and what a rank of two holds of them.
    heads, kv, hd = rng.choice([(14, 2, 64), (28, 4, 128), (7, 1, 64), (14, 2, 128)])
    c = dict(heads=heads, kv=kv, hd=hd, window=0, sinks=0, values=rng.choice(["f32", "bf16"]),
             cache=rng.choice(["bf16", "int8"]))
    form = rng.choice(["store", "step", "draft", "chunk", "mixed", "window_step", "window_chunk"])
    if form == "store":
        n = spread(1, 64)
        c.update(kind="store", sequences=n, first=spread(1, 8192 // n + 1), rest=spread(1, 4096 // n + 1), lo=rng.randrange(500),
                 hi=spread(1, 4000))
    elif form in ("step", "window_step"):
        n = spread(1, 64)
        c.update(kind="attend", sequences=n, first=1, rest=1, lo=spread(1, 1000), hi=spread(100, 32000 if n < 16 else 8000))
    elif form == "draft":
        t = rng.randrange(2, 17)
        c.update(kind="attend", sequences=spread(1, 32), first=t, rest=t, lo=spread(1, 1000), hi=spread(100, 4000))
    elif form in ("chunk", "window_chunk"):
        lo = rng.choice([0, spread(1, 4000)])
        c.update(kind="attend", sequences=1, first=spread(17, 4000), rest=0, lo=lo, hi=lo)
    else:
        c.update(kind="attend", sequences=rng.randrange(2, 33), first=spread(17, 512), rest=1, lo=spread(1, 4000),
                 hi=spread(1, 4000))
    if form.startswith("window"):
        c.update(window=spread(16, 4000), sinks=rng.choice([0, 1, 4, 17, 64]))
    return c


def _shapes(case):
    """Cached positions and new tokens of every sequence."""
    n = case["sequences"]
    lo, hi = max(case["lo"], 1), max(case["hi"], 1)
    starts = [int(round(lo * (hi / lo) ** (i / max(n - 1, 1)))) for i in range(n)] if max(case["lo"], case["hi"]) else [0] * n
    if case["lo"] == 0:
        starts[0] = 0
    counts = [case["first"]] + [case["rest"]] * (n - 1)
    return starts, counts


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.default_rng(seed)
    starts, counts = _shapes(case)
    n, H, KV, hd = case["sequences"], case["heads"], case["kv"], case["hd"]
    ends = [a + b for a, b in zip(starts, counts)]
    width = -(-max(ends) // PAGE)
    # Every sequence has its own pages, handed out in no order, and some of the pool is free.
    pages = sum(-(-e // PAGE) for e in ends) + 7
    order = host.permutation(pages)
    tables, at = np.zeros((n, width), np.int32), 0
    for s, e in enumerate(ends):
        k = -(-e // PAGE)
        tables[s, :k] = order[at:at + k]
        at += k
    tokens = sum(counts)
    dt = torch.float32 if case["values"] == "f32" else torch.bfloat16
    # The rows of a fused Q, K, V product: the operators take their slices.
    qkv = torch.randn(tokens, (H + 2 * KV) * hd, device="cuda", generator=g)
    qkv[:, :H * hd] *= 1.5
    # A few channels are much larger than the others, as in trained keys.
    loud = torch.from_numpy(host.choice(hd, max(1, hd // 32), replace=False)).cuda()
    qkv.view(tokens, H + 2 * KV, hd)[:, H:H + KV, loud] *= 4.0
    qkv = qkv.to(dt)
    st = dict(case=case, tables=tables, starts=np.array(starts, np.int32), counts=np.array(counts, np.int32), qkv=qkv,
              q=qkv[:, :H * hd].view(tokens, H, hd), k=qkv[:, H * hd:(H + KV) * hd].view(tokens, KV, hd),
              v=qkv[:, (H + KV) * hd:].view(tokens, KV, hd))
    for name in ("k", "v"):
        pool = torch.randn(pages, KV, PAGE, hd, device="cuda", generator=g)
        if name == "k":
            pool[..., loud] *= 4.0
        if case["cache"] == "int8":
            scales = pool.abs().amax(-1) / 127.0
            st[name + "_scales"] = scales
            st[name + "_pool"] = torch.round(pool / scales[..., None]).clamp_(-127, 127).to(torch.int8)
        else:
            st[name + "_scales"] = None
            st[name + "_pool"] = pool.to(torch.bfloat16)
        del pool
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    starts, counts = st["starts"], st["counts"]
    # Where the packed tokens are: their sequence, index in it and position.
    seq = np.repeat(np.arange(len(counts)), counts)
    idx = np.arange(int(counts.sum())) - np.repeat(np.cumsum(counts) - counts, counts)
    st["seq"], st["idx"] = torch.from_numpy(seq).cuda(), torch.from_numpy(idx).cuda()
    st["pos"] = torch.from_numpy(starts[seq] + idx).cuda()
    st["starts_dev"], st["ends_dev"] = torch.from_numpy(starts).cuda().long(), torch.from_numpy(starts + counts).cuda().long()
    st["most"] = int(counts.max())
    st["tables_dev"] = torch.from_numpy(st["tables"]).cuda().long()
    if case["kind"] == "store":
        st["out_k"], st["out_v"] = (torch.empty(st["k"].shape, dtype=st["k"].dtype, device="cuda") for _ in range(2))
    else:
        st["y"] = torch.empty(st["q"].shape, dtype=st["q"].dtype, device="cuda")
    if own:
        import llm_inference_edu_b200 as qb
        st["cache"] = qb.PagedCache.from_tensors(st["k_pool"], st["v_pool"], st["k_scales"], st["v_scales"])
        # One plan a step: every layer's calls of the step go by it.
        st["plan"] = qb.PagedPlan(st["cache"], st["tables"], starts, counts, case["heads"], window=case["window"],
                                  sinks=case["sinks"], dtype=case["values"])
        st["qb"] = qb
    return st


def _store(x, pool, scales, page, row):
    """The rows' stored form, written into the pool and read back as f32."""
    x = x.float()
    if scales is None:
        pool[page, :, row] = x.to(torch.bfloat16)
        return pool[page, :, row].float()
    scale = x.abs().amax(-1) / 127.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    r = x / scale[..., None]
    r = torch.where(r < 0, -torch.floor(-r + 0.5), torch.floor(r + 0.5)).clamp(-127, 127)
    pool[page, :, row] = r.to(torch.int8)
    scales[page, :, row] = scale
    return pool[page, :, row].float() * scales[page, :, row][..., None]


def _gathered(pool, scales, tables):
    """[sequences][kv_heads][positions][head_dim] in f32."""
    x = pool[tables].float()
    if scales is not None:
        x = x * scales[tables][..., None]
    n, width, kv, page, hd = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, kv, width * page, hd)


def _attend(st):
    case = st["case"]
    n, H, KV, hd, G = case["sequences"], case["heads"], case["kv"], case["hd"], case["heads"] // case["kv"]
    k = _gathered(st["k_pool"], st["k_scales"], st["tables_dev"])
    v = _gathered(st["v_pool"], st["v_scales"], st["tables_dev"])
    most, length = st["most"], k.shape[2]
    q = torch.zeros(n, most, H, hd, device="cuda")
    q[st["seq"], st["idx"]] = st["q"].float()
    q = q.view(n, most, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(n, KV, G * most, hd)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    p = st["starts_dev"][:, None, None] + torch.arange(most, device="cuda")[None, :, None]
    j = torch.arange(length, device="cuda")[None, None, :]
    seen = (j <= p) & (j < st["ends_dev"][:, None, None])
    if case["window"]:
        seen &= (j > p - case["window"]) | (j < case["sinks"])
    seen = seen[:, None, None]
    s = s.view(n, KV, G, most, length).masked_fill_(~seen, -math.inf)
    s = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    total = s.sum(-1, keepdim=True)
    y = torch.matmul(s.view(n, KV, G * most, length), v).view(n, KV, G, most, hd) / total
    y = y.permute(0, 3, 1, 2, 4).reshape(n, most, H, hd)
    return y[st["seq"], st["idx"]].to(st["q"].dtype)


def run(st):
    if own:
        qb = st["qb"]
        if st["case"]["kind"] == "store":
            qb.kv_write(st["k"], st["v"], st["cache"], st["plan"])
            qb.kv_read(st["cache"], st["plan"], st["out_k"], st["out_v"])
            return st["out_k"], st["out_v"]
        qb.paged_attention(st["q"], st["cache"], st["plan"], st["y"])
        return st["y"]
    if st["case"]["kind"] == "store":
        page, row = st["tables_dev"][st["seq"], st["pos"] // PAGE], st["pos"] % PAGE
        return (_store(st["k"], st["k_pool"], st["k_scales"], page, row).to(st["k"].dtype),
                _store(st["v"], st["v_pool"], st["v_scales"], page, row).to(st["v"].dtype))
    return _attend(st)


def _visible(case):
    """Visible (query, key) pairs a head, and the keys of each sequence that any of its queries sees."""
    pairs = keys = 0
    w, sinks = case["window"], case["sinks"]
    for a, c in zip(*_shapes(case)):
        p = np.arange(a, a + c, dtype=np.int64)
        if not w:
            pairs += int((p + 1).sum())
            keys += (a + c) if c else 0
            continue
        first = np.maximum(p - w + 1, 0)
        pairs += int((p + 1 - first + np.minimum(first, sinks)).sum())
        keys += (a + c - int(first[0]) + min(int(first[0]), sinks)) if c else 0
    return pairs, keys


def work(case):
    H, KV, hd = case["heads"], case["kv"], case["hd"]
    tokens = sum(_shapes(case)[1])
    vb = 4 if case["values"] == "f32" else 2
    row = 2 * KV * (hd + 4 if case["cache"] == "int8" else 2 * hd)  # a position's K and V in the cache
    if case["kind"] == "store":
        # Values in, rows stored, rows read back, values out.
        return {"bytes": tokens * (2 * 2 * KV * hd * vb + 2 * row), "flops": tokens * 2 * KV * hd * 4}
    pairs, keys = _visible(case)
    return {"bytes": 2 * tokens * H * hd * vb + keys * row, "flops": 4 * hd * H * pairs}


def exact(case, seed):
    st = _inputs(case, seed)
    KV, hd, G = case["kv"], case["hd"], case["heads"] // case["kv"]
    if case["kind"] == "store":
        found = []
        for name in ("k", "v"):
            x = st[name].double()
            if case["cache"] == "int8":
                # The scale and the quotient are f32 numbers by definition; a 64-bit quotient of two f32 numbers, rounded
                # to f32, is the f32 quotient.
                scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()
                scale[scale == 0] = 1.0
                r = (x / scale).float().double()
                x = (torch.sign(r) * torch.floor(r.abs() + 0.5)).clamp(-127, 127) * scale
            else:
                x = x.to(torch.bfloat16).double()
            found.append(x)
        return tuple(found)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (a, c) in enumerate(zip(st["starts"].tolist(), st["counts"].tolist())):
        table = torch.from_numpy(st["tables"][s, :-(-(a + c) // PAGE)]).cuda().long()
        for h in range(KV):
            kv = []
            for name in ("k", "v"):
                x = st[name + "_pool"][table, h].double()
                if st[name + "_scales"] is not None:
                    x = x * st[name + "_scales"][table, h].double()[..., None]
                kv.append(x.reshape(-1, hd)[:a + c])
            # A thousand queries at a time, for memory.
            for b in range(0, c, 1024):
                m = min(1024, c - b)
                p = torch.arange(a + b, a + b + m, device="cuda")[:, None]
                j = torch.arange(a + c, device="cuda")[None]
                hidden = j > p
                if case["window"]:
                    hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
                q = st["q"][at + b:at + b + m, h * G:(h + 1) * G].double().transpose(0, 1)
                e = (q @ kv[0].T / math.sqrt(hd)).masked_fill(hidden, -math.inf).softmax(-1)
                out[at + b:at + b + m, h * G:(h + 1) * G] = (e @ kv[1]).transpose(0, 1)
        at += c
    return out
