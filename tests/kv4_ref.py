"""The 4-bit cache in numpy: the format, the layout as include/madi_q8.h states
it, and attention over it in float64."""
import numpy as np


def quantise(x):
    """Codes (int, -7..7) and scales (f16) of rows [..., d], from the definition.
    |x| / s + 1/2 is compared with whole numbers exactly: 2|x| >= (2c + 1) s in
    float64 holds or not without rounding (24 bits against 11 + 4)."""
    x = np.where(np.isnan(x), 0, x).astype(np.float64)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(b).max(-1)
    with np.errstate(over="ignore"):
        s = (np.minimum(top, 3e38).astype(np.float32) / np.float32(7)).astype(np.float16)
    s = np.where(s <= np.float16(9352), s, np.float16(9352)).astype(np.float16)
    s64 = s.astype(np.float64)[..., None]
    q = sum((2 * np.abs(b) >= (2 * c + 1) * s64).astype(int) for c in range(7)) * (s64 > 0)
    return (np.sign(b) * q).astype(int).reshape(x.shape), s


def value(q, s):
    return (q.reshape(*s.shape, 32) * s.astype(np.float64)[..., None]).reshape(q.shape)


def block_bytes(page, d):
    return page * d * 9 // 8


def put(data, page, d, p, h, t, kq, ks, vq, vs):
    """Token t of page p, head h: the layout comment, literally.  data is u8
    [n_pages][heads][block_bytes]; returns nothing."""
    nb, blk, u = d // 32, data[p, h], t // 4
    for b in range(nb):
        for g in range(4):
            word = 0
            for j in range(4):
                word |= int(kq[32 * b + 8 * g + 2 * j] + 8) << (4 * j)
                word |= int(kq[32 * b + 8 * g + 2 * j + 1] + 8) << (4 * (4 + j))
            at = t * d // 2 + (g * nb + b) * 4
            blk[at:at + 4] = np.frombuffer(np.uint32(word).tobytes(), np.uint8)
        for c in range(16):
            byte = {0: 0, 2: 1, 1: 2, 3: 3}[t % 4]
            at = page * d // 2 + u * 2 * d + (c * nb + b) * 4 + byte
            blk[at] = int(vq[32 * b + c] + 8) | int(vq[32 * b + 16 + c] + 8) << 4
        for x, s in ((0, ks), (1, vs)):
            at = page * d + u * d // 2 + ((x * nb + b) * 4 + t % 4) * 2
            blk[at:at + 2] = np.frombuffer(np.float16(s[b]).tobytes(), np.uint8)


def rows_of(n, rows):
    """Positions of a sequence's rows (negative: none)."""
    return range(n - rows, n)


def attention(q, keys, values, there, pos, causal, window, scale):
    """q [rows][G][d], keys and values [n][d] float64, there [n]; returns out
    [rows][G][d], the mean |v| with the same weights, and the sum of |v| over
    the visible keys."""
    n = keys.shape[0]
    j = np.arange(n)[None]
    p = np.asarray(pos)[:, None]
    seen = np.broadcast_to(there[None], (len(pos), n)).copy()
    if causal:
        seen &= j <= p
        if window:
            seen &= j > p - window
    x = np.einsum("rgd,nd->rgn", q.astype(np.float64), keys) * scale
    x = np.where(seen[:, None], x, -np.inf)
    top = x.max(-1, keepdims=True, initial=-1e300)
    e = np.where(seen[:, None], np.exp(x - np.where(top < -1e299, 0, top)), 0)
    den = e.sum(-1, keepdims=True)
    w = e / np.where(den == 0, 1, den)
    return np.einsum("rgn,nd->rgd", w, values), np.einsum("rgn,nd->rgd", w, np.abs(values)), \
        (seen.astype(np.float64) @ np.abs(values))[:, None]


def score_error(q, ks, scale):
    """Bound on a score's error, per (row, head): products of f16 and 4-bit
    numbers are exact; a block's 32 (64 with low parts) add up in f32 in some
    order, no partial sum above 7 sum|q|, then the blocks: fewer than 80 roundings of
    2^-24 on 7 sum_b s_b sum|q|_b in all."""
    qb = np.abs(q.astype(np.float64)).reshape(*q.shape[:-1], q.shape[-1] // 32, 32).sum(-1)  # [rows][G][b]
    top = (qb[:, :, None] * ks.astype(np.float64)[None, None]).sum(-1).max(-1, initial=0)
    return 80 * 2.0 ** -24 * 7 * abs(scale) * top
