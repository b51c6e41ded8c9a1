"""Plain 64-bit forms of the paged cache operators and the error bounds that
the tests hold the kernels to."""
import numpy as np

PAGE = 16


def quantize(x):
    """qb_kv_write's INT8 encode of float32 rows [..., hd], step by step in
    float32: (values, scales)."""
    x = np.asarray(x, np.float32)
    m = np.max(np.abs(x), -1)
    with np.errstate(invalid="ignore"):
        scale = (m * (np.float32(1) / np.float32(127))).astype(np.float32)
    scale = np.where(scale == 0, np.float32(1), scale)
    bad = ~np.isfinite(x).all(-1)
    with np.errstate(invalid="ignore"):
        r = (x / scale[..., None]).astype(np.float32)
        q = np.clip(np.sign(r) * np.floor(np.abs(r.astype(np.float64)) + 0.5), -127, 127)
    q = np.where(bad[..., None], 0, q).astype(np.int8)
    return q, np.where(bad, np.float32(np.nan), scale)


def bf16(x):
    """float32 rounded to bfloat16 (nearest even), as float32."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & np.uint32(0xFFFF0000)).astype(np.uint32)
    return np.where(np.isnan(x), np.float32(np.nan), r.view(np.float32))


def sees(p, j, window, sinks):
    return (j <= p) & ((window == 0) | (j > p - window) | (j < sinks))


def attention(q, k, v, tables, starts, counts, window=0, sinks=0, scale=None, bf16_weights=False, half_step=2.0**-24,
              f16_weights=False):
    """(y, bound): attention over dequantised float64 pools [pages][kv][16][hd]
    for packed float64 queries, and how far a kernel may be from it.

    With u = 2^-24: a product summed in FP32 over n terms, each term exact
    or split into three bf16 planes (a remainder under 2^-24 of it), is off by
    at most (n + 4) u sum|terms|.  So a score is off by
    d = (hd + 8) u scale sum|q||k| (four more for the scales of quantised rows and the
    product with `scale`), and t = score log2(e) - max by another 2 u |t|;
    2^t then carries 2^-21 (the hardware's 2 ulp, its flush of values under
    2^-126 being nothing next to the largest, which is 1).  Numerator and
    denominator each carry that: w = 2 (max d + 4 u max|s - m| + 2^-21), to
    first order.  Weights kept as one bf16 number add 2^-8.  The sum over n
    keys, its rescaling (once a unit of keys) and the join of the parts add
    (2 n + 16) u.  The result's own rounding is half_step |y|.
    Over INT8 rows (`f16_weights`) a weight with its row's scale may be one
    or two f16 numbers, taken so that the largest is at least 2^7: below
    f16's normal numbers the spacing is 2^-24, so each is off by up to 2^-25,
    which is 2^-32 of the largest, times up to 127 of its row.  V scales below
    2^-90 are not made up for: the largest is then smaller by their ratio to
    2^-90, and the same 2^-25 is that much more of it."""
    T, H, hd = q.shape
    KV = k.shape[1]
    G = H // KV
    scale = hd ** -0.5 if scale is None else scale
    y, bound = np.zeros((T, H, hd)), np.zeros((T, H, hd))
    u, at = 2.0**-24, 0
    for s, (a, c) in enumerate(zip(starts, counts)):
        n = a + c
        for i in range(c):
            p = a + i
            j = np.arange(n)
            seen = np.nonzero(sees(p, j, window, sinks))[0]
            pages, rows = np.asarray(tables[s])[seen // PAGE], seen % PAGE
            for h in range(H):
                kk, vv = k[pages, h // G, rows], v[pages, h // G, rows]
                qq = q[at + i, h]
                t = scale * (kk @ qq)
                d = (hd + 8) * u * scale * np.max(np.abs(kk) @ np.abs(qq))
                m = t.max()
                e = np.exp(t - m)
                w = e / e.sum()
                y[at + i, h] = w @ vv
                rel = 2 * (d + 4 * u * np.max(m - t) + 2.0**-21) + (2 * len(seen) + 16) * u
                rel += 2.0**-8 if bf16_weights else 0.0
                if f16_weights:
                    small = max(1.0, 2.0**-90 / max(np.abs(vv).max() / 127, 1e-300))
                    bound[at + i, h] += 2.0**-32 * small * len(seen) * np.max(w * np.abs(vv).max(-1))
                bound[at + i, h] += 1.01 * rel * (w @ np.abs(vv)) + half_step * np.abs(y[at + i, h]) * 1.01 + 1e-37
        at += c
    return y, bound
