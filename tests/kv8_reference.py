"""The 8-bit cache's operators in 64 bits on the CPU, for the tests."""
import numpy as np

E4M3, INT8 = 0, 1
TOP = {E4M3: 448.0, INT8: 127.0}


def code_values(code):
    """The value of each of the 256 codes."""
    c = np.arange(256)
    if code == INT8:
        return np.where(c > 127, c - 256, c).astype(np.float64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8.0 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c > 127, -v, v)


def encode(x, code):
    """Codes of values within the format's range, to nearest, ties to even."""
    x = np.asarray(x, np.float64)
    if code == INT8:
        return np.rint(x).astype(np.int64).astype(np.uint8)
    mag = np.abs(x)
    e = np.floor(np.log2(np.maximum(mag, 2.0 ** -6)))
    r = np.rint(mag / 2.0 ** (e - 3)) * 2.0 ** (e - 3)
    e = np.floor(np.log2(np.maximum(r, 2.0 ** -6)))
    bits = np.where(r < 2.0 ** -6, r * 2.0 ** 9, (e + 7) * 8 + r / 2.0 ** (e - 3) - 8).astype(np.uint8)
    return np.where(np.signbit(x), bits | 128, bits).astype(np.uint8)


def scale_of(amax, code):
    """The smallest power of two, 2^-126 at least, by which amax fits."""
    s = 2.0 ** -126
    while amax / s > TOP[code]:
        s *= 2.0
    return s


def write(codes, scales, slots, x, code):
    """kv8_write of one of K and V, in place: codes [blocks][H][bt][D], scales [blocks][H]."""
    bt = codes.shape[2]
    x = np.asarray(x, np.float64)
    values = code_values(code)
    r = 0
    while r < len(slots):
        if slots[r] < 0 or slots[r] >= codes.shape[0] * bt:
            r += 1
            continue
        n = 1
        while r + n < len(slots) and slots[r + n] == slots[r] + n and slots[r + n] % bt:
            n += 1
        b, place = divmod(int(slots[r]), bt)
        for h in range(codes.shape[1]):
            rows = x[r:r + n, h]
            fine = rows[np.isfinite(rows)]
            s = scale_of(np.abs(fine).max() if fine.size else 0.0, code)
            if place:
                before = max(float(scales[b, h]), 0.0)
                if s > before:
                    codes[b, h, :place] = encode(values[codes[b, h, :place]] * (before / s), code)
                s = max(s, before)
            scales[b, h] = s
            y = np.where(np.isnan(rows), 0.0, np.clip(rows / s, -TOP[code], TOP[code]))
            codes[b, h, place:place + n] = encode(y, code)
        r += n


def batch_map(cached, new, free, tables, bt, num_blocks, n_rows):
    """(ctx_lens, row_starts, slots, positions, counts); tables [B][pages] in place."""
    slots, positions = np.full(n_rows, -1, np.int64), np.full(n_rows, -1, np.int32)
    starts, ctx, taken = [0], [], 0
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        for page in range(-(-c // bt), min(-(-(c + n) // bt), tables.shape[1])):
            tables[b, page] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(n):
            r, pos = starts[-1] + i, c + i
            if r < n_rows:
                positions[r] = pos
                block = tables[b, pos // bt] if pos // bt < tables.shape[1] else -1
                if 0 <= block < num_blocks:
                    slots[r] = int(block) * bt + pos % bt
        starts.append(starts[-1] + n)
        ctx.append(c + n)
    return (np.array(ctx, np.int32), np.array(starts, np.int32), slots, positions,
            np.array([taken, starts[-1]], np.int32))


def attention(q, k, v, positions, scale=0.0, softcap=0.0, window=0, slopes=None, prefix=0,
              present=None, steps=1.0, unit=0.0):
    """Rows q [R][H][D] at `positions` over k, v [N][Hkv][D] (values): the result, and how far a
    kernel may be from it through its scores and f32 sums.

    The bound.  A score's parts reach it with a few roundings of 2^-24 each relative to
    A = sum |q_d k_d| scale (+ the cap and the bias): two-term q 2^-22, at most 2 D / 32 + 4 steps of
    f32 sums, the scale's and the cap's own; together below 2^-20 A (`steps` times that where q
    has one term).  d(out) = sum p_j (v_j - out) d(s_j) carries it to the output.  The weights' own
    roundings (exp2 2^-22, two binary16 terms 2^-22, the f32 sums of N terms in chains of N / 16 and
    less) are relative to sum p |v|.
    Two-term values end at binary16's smallest step, 2^-24: with the largest weight times the largest
    V scale at 2^14 a term is off by up to 2^-25, that is 2^-39 of it, whatever the weight, so N
    terms by N 2^-39 `unit` (the largest scale times the largest code); with the largest q at 2^13
    or more, an element of q by 2^-38 of that."""
    R, H, D = q.shape
    N, Hkv = k.shape[0], k.shape[1]
    scale = scale if scale > 0 else D ** -0.5
    out, bound = np.zeros((R, H, D)), np.zeros((R, H, D))
    key = np.arange(N)
    pos = np.asarray(positions)[:, None]
    seen = (key <= pos) | (key < prefix)
    if window > 0:
        seen &= pos - key < window
    if present is not None:
        seen &= present[None, :]
    seen &= (pos >= 0)
    for h in range(H):
        kk, vv = k[:, h * Hkv // H].copy(), v[:, h * Hkv // H].copy()
        hidden = ~seen.any(0)
        kk[hidden], vv[hidden] = 0.0, 0.0
        s = q[:, h] @ kk.T * scale
        a = (np.abs(q[:, h]) + np.abs(q[:, h]).max(1, keepdims=True) * 2.0 ** -18) @ np.abs(kk).T * scale
        if softcap > 0:
            s, a = softcap * np.tanh(s / softcap), a + 0.25 * softcap
        if slopes is not None:
            bias = slopes[h] * np.abs(pos - key)
            s, a = s - bias, a + bias
        s = np.where(seen, s, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
        total = p.sum(1, keepdims=True)
        p = p / np.where(total > 0, total, 1.0)
        o = p @ vv
        pa = p * (a * 1.5 * 2.0 ** -20 * steps)  # 1.5 > log2(e): s in log2 units
        out[:, h] = o
        bound[:, h] = (pa @ np.abs(vv) + pa.sum(1, keepdims=True) * np.abs(o)
                       + (p @ np.abs(vv) + np.abs(o)) * (2.0 ** -20 + (N / 16 + 40) * 2.0 ** -24)
                       + N * 2.0 ** -39 * unit)
    return out, bound
