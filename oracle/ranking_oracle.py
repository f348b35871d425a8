"""Plain numpy forms, in 64 bits, of the ranking operators (4-bit microscaled tables and their score
product, score adjustments, the k best of a row).  The reference has none of them (it ends at
predict_all, src/als.py:347-364): parity unpinned, these are the definitions themselves."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx4_quantize(x):
    """(codes [n, 16 b] uint8, scales [n, b] uint8) of the rows of x (any float type)."""
    x = np.asarray(x, dtype=np.float64)
    n, width = x.shape
    b = (width + 31) // 32
    blocks = np.zeros((n, b * 32))
    blocks[:, :width] = x
    blocks = blocks.reshape(n, b, 32)
    top = np.abs(blocks).max(axis=-1)
    bad = ~np.isfinite(blocks).all(axis=-1)
    _, e = np.frexp(np.where(bad, 1.0, top))
    e = np.where(top == 0, -127, np.clip(e - 3, -127, 127))
    size = np.ldexp(np.where(bad[..., None], 0.0, np.abs(blocks)), -e[..., None])
    code = np.zeros(size.shape, dtype=np.uint8)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        # a tie goes to the even code: up from an odd one, down from an even one
        code += (size >= mid) if i % 2 else (size > mid)
    code += 8 * np.signbit(blocks).astype(np.uint8)
    code[bad] = 0
    code = code.reshape(n, b * 32)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def mx4_values(codes, scales, width):
    """float64 values; NaN under scale byte 255."""
    n = codes.shape[0]
    both = np.stack((codes & 15, codes >> 4), axis=-1).reshape(n, -1)
    v = GRID[both & 7] * np.where(both & 8, -1.0, 1.0)
    unit = np.ldexp(1.0, scales.astype(np.int64) - 127)
    unit = np.where(scales == 255, np.nan, unit)
    return (v.reshape(n, -1, 32) * unit[..., None]).reshape(n, -1)[:, :width]


def adjust_scores(scores, history=None, history_rows=None, repetition=1.0, frequency=0.0,
                  presence=0.0, exclude=False, item_bias=None, row_bias=None, mask=None,
                  mask_rows=None):
    """(values in float64, the largest magnitude met on the way to each of them)."""
    x = np.array(scores, dtype=np.float64)
    n, m = x.shape
    mag = np.where(np.isfinite(x), np.abs(x), 0.0)
    per_row = lambda v: np.broadcast_to(np.asarray(v, dtype=np.float64), (n,))
    rep, freq, pres = per_row(repetition), per_row(frequency), per_row(presence)
    for r in range(n):
        if history is not None:
            l = r if history_rows is None else int(history_rows[r])
            seen = np.zeros(0, dtype=np.int64)
            if 0 <= l < len(history[0]) - 1:
                seen = np.asarray(history[1][history[0][l]:history[0][l + 1]], dtype=np.int64)
            seen = seen[(seen >= 0) & (seen < m)]
            ids, count = np.unique(seen, return_counts=True)
            if exclude:
                x[r, ids] = -np.inf
            else:
                s = x[r, ids]
                with np.errstate(invalid='ignore'):
                    s = np.where(s > 0, s / rep[r], s * rep[r])
                mag[r, ids] = np.maximum(mag[r, ids], np.where(np.isfinite(s), np.abs(s), 0))
                mag[r, ids] += np.abs(freq[r]) * count + np.abs(pres[r])
                x[r, ids] = s - (freq[r] * count + pres[r])
        if item_bias is not None:
            x[r] += np.asarray(item_bias, dtype=np.float64)
            mag[r] += np.abs(item_bias)
        if row_bias is not None:
            for e in range(int(row_bias[0][r + 1]) - 1, int(row_bias[0][r]) - 1, -1):
                i = int(row_bias[1][e])
                if 0 <= i < m and i not in row_bias[1][e + 1:int(row_bias[0][r + 1])]:
                    x[r, i] += float(row_bias[2][e])
                    mag[r, i] += abs(float(row_bias[2][e]))
        if mask is not None:
            g = (0 if len(mask) == 1 else r) if mask_rows is None else int(mask_rows[r])
            if g >= len(mask):
                x[r] = -np.inf
            elif g >= 0:
                bits = np.unpackbits(np.ascontiguousarray(mask[g]).view(np.uint8),
                                     bitorder='little')[:m]
                x[r, bits == 0] = -np.inf
    return x, mag


def order_image(scores):
    """Integers that order like the scores' bits: -0.0 below +0.0, NaN by its sign above or
    below everything."""
    s = np.asarray(scores)
    u = {4: np.uint32, 8: np.uint64, 2: np.uint16}[s.dtype.itemsize]
    bits = s.view(u)
    top = u(1) << u(8 * s.dtype.itemsize - 1)
    return np.where(bits & top, ~bits, bits | top)


def topk_rows(scores, k):
    """Indices of the k best of every row, equal scores by the smaller index."""
    key = order_image(scores)
    flipped = np.iinfo(key.dtype).max - key
    return np.argsort(flipped, axis=1, kind='stable')[:, :k].astype(np.int32)
