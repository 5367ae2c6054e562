"""The 8-bit paged cache in 64 bits, row by row, as the header states it: quantiser, append, attention, and how far a kernel's
result may be from it.  numpy only."""
import numpy as np

DIM, GROUP = 128, 16


def bf16(x):
    """Nearest bf16 value (ties to even) of finite float64 numbers, through float32."""
    b = np.asarray(x, dtype=np.float32).view(np.uint32)
    r = (b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000
    return r.astype(np.uint32).view(np.float32).astype(np.float64)


def e4m3_values():
    c = np.arange(256)
    e, m, s = (c >> 3) & 15, c & 7, np.where(c & 128, -1.0, 1.0)
    v = s * np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    v[(c & 127) == 127] = np.nan
    return v


VALUE = e4m3_values()


def e4m3(x):
    """Codes of the nearest e4m3 values, ties to even, saturating; -0.0 keeps its sign."""
    a = np.abs(x)
    _, ex = np.frexp(a)
    step = 2.0 ** (np.maximum(ex - 1, -6) - 3)
    q = np.minimum(np.round(a / step) * step, 448.0)
    mags = VALUE[:127]
    return (np.searchsorted(mags, q) | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_of(amax):
    if not np.isfinite(amax) or amax > 448.0 * 2.0 ** 60:
        return np.nan
    if amax == 0:
        return 2.0 ** -126
    m, ex = np.frexp(amax)
    return 2.0 ** max(ex - 9 if m <= 0.875 else ex - 8, -126)


def rotate(x, pos, theta):
    if theta == 0:
        return x
    ang = pos * theta ** (-np.arange(0, DIM, 2) / DIM)
    c, s = np.cos(ang), np.sin(ang)
    lo, hi = x[..., :DIM // 2], x[..., DIM // 2:]
    return np.concatenate([lo * c - hi * s, lo * s + hi * c], axis=-1)


def page_of(table, pos, page, num_blocks):
    i = pos // page
    if pos < 0 or i >= len(table) or not 0 <= table[i] < num_blocks:
        return -1
    return int(table[i])


def append(codes, scales, x, table, first, theta, page):
    """x [n, kv_heads, 128] (float64) behind position `first` into codes [blocks, kv_heads, page, 128] (uint8) and scales, in place."""
    n = x.shape[0]
    for g in range(first // GROUP, (first + n - 1) // GROUP + 1):
        a, b = max(first, g * GROUP), min(first + n, (g + 1) * GROUP)
        if b <= max(a, 0) or g < 0:
            continue
        blk = page_of(table, a, page, codes.shape[0])
        if blk < 0:
            continue
        sub, r0 = a % page // GROUP, a % GROUP
        for h in range(x.shape[1]):
            y = np.stack([rotate(x[p - first, h], p, theta) if theta is not None else x[p - first, h] for p in range(a, b)])
            bad = not np.all(np.isfinite(y))
            s = np.nan if bad else scale_of(np.abs(y).max())
            rows = codes[blk, h, sub * GROUP:(sub + 1) * GROUP]
            if r0:
                old = float(scales[blk, h, sub])
                s = np.nan if np.isnan(old) or np.isnan(s) else max(s, old)
                rows[:r0] = 0 if np.isnan(s) else e4m3(VALUE[rows[:r0]] * (old / s))
            rows[r0:r0 + b - a] = 0 if np.isnan(s) else e4m3(y / s)
            scales[blk, h, sub] = s


def attend(q, k_codes, k_scales, v_codes, v_scales, table, length, window=0, sinks=0, scale=DIM ** -0.5):
    """q [n, heads, 128] -> (result, how far a kernel's bf16 result may be from it), both [n, heads, 128].

    The bound: the bf16 result is off by half a step, 2^-9 |o| for a number in the lower half of its binade and no more than 2^-8 |o|.
    A weight is off by 2^-8 of itself: two e4m3 numbers, half a step 2^-4 of the residual of half a step 2^-4; f16 and bf16 less.  It
    also has an absolute error: weights times V scales are brought to a largest of at least 2^6, and the second number counts in
    steps of 2^-9 with a factor 2^-4, so half a step is 2^-14, 2^-20 of the largest.  That meets the token's CODE, up to 448 where the
    largest one's may be small: 2^-20 (largest weight times scale) (sum of code magnitudes).  Where weights are f16 they are not
    taken times the scales, and what is below 2^-14 of the largest is off by 2^-25 of it: 2^-25 (largest weight) (largest scale) (sum
    of code magnitudes).  A score is off by d: the query's split
    leaves 2^-17 of the row's largest element per dim, fp32 sums 2^-18 of the sum of magnitudes, exponents 2^-20.  A weight's relative
    error counts twice, above and below the line."""
    n, heads, _ = q.shape
    blocks, kv_heads, page, _ = k_codes.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        p = length - n + i
        seen = [j for j in range(max(p + 1, 0)) if (window == 0 or p - j < window or j < sinks) and page_of(table, j, page, blocks) >= 0]
        if not seen:
            continue
        blk = np.array([page_of(table, j, page, blocks) for j in seen])
        at = np.array(seen) % page
        for h in range(heads):
            kh = h // (heads // kv_heads)
            k = VALUE[k_codes[blk, kh, at]] * k_scales[blk, kh, at // GROUP].astype(np.float64)[:, None]
            v = VALUE[v_codes[blk, kh, at]] * v_scales[blk, kh, at // GROUP].astype(np.float64)[:, None]
            x = k @ q[i, h] * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            out[i, h] = w @ v
            d = scale * (2.0 ** -17 * np.abs(q[i, h]).max() * np.abs(k).sum(1).max() + 2.0 ** -18 * (np.abs(k) @ np.abs(q[i, h])).max()) + 2.0 ** -20
            vs = v_scales[blk, kh, at // GROUP].astype(np.float64)
            top = (w * vs).max() + 2.0 ** -5 * w.max() * vs.max()
            tol[i, h] = 2.0 ** -8 * np.abs(out[i, h]) + (2.0 ** -8 + 2 * d) * 2 * (w @ np.abs(v)) + 2.0 ** -20 * top * np.abs(VALUE[v_codes[blk, kh, at]]).sum(0) + 1e-37
    return out, tol
