"""A numpy restatement of the 4-bit key/value cache (include/dscq.h, dscq_kv_*).

The row rule runs in fp32 with one rounding an operation, as the kernels', so stored bytes
are compared bit for bit; attention runs in 64 bits on the numbers the bytes stand for.
Bytes are placed one nibble at a time from the layout's definition.
"""
import numpy as np

NAN_WORD = 0x7FC00000
KEY_NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]


def hadamard(x):
    """H_D x over the last axis in fp32, index bits in ascending order."""
    x = np.array(x, np.float32)
    D = x.shape[-1]
    h = 1
    while h < D:
        y = x.reshape(*x.shape[:-1], D // (2 * h), 2, h)
        x = np.stack((y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]), -2).reshape(x.shape)
        h *= 2
    return x


def turn(x, cos, sin, interleaved):
    """[T, H, D] with the first 2 cos.shape[1] elements of each head turned; cos, sin [T, R/2]."""
    x = np.array(x, np.float32)
    half = cos.shape[1]
    a = np.arange(half) * (2 if interleaved else 1)
    b = a + (1 if interleaved else half)
    c, s = cos[:, None].astype(np.float32), sin[:, None].astype(np.float32)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def quantize(x):
    """(codes uint8 [..., D], words uint32 [...]) of fp32 rows."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], np.float32(0), x)
    lo = np.minimum(x.min(-1), np.float32(0))
    hi = np.maximum(x.max(-1), np.float32(0))
    base = np.maximum((hi - lo) / np.float32(15), np.float32(1e-8))
    bits = (base.view(np.uint32) + np.uint32(15)) & ~np.uint32(15)
    zero = np.clip(np.rint(-lo / bits.view(np.float32)), 0, 15).astype(np.float32)
    words = bits | zero.astype(np.uint32)
    t = x / words.view(np.float32)[..., None] + zero[..., None]
    codes = np.clip(np.rint(t), 0, 15).astype(np.uint8)
    return codes, np.where(bad, np.uint32(NAN_WORD), words)


def places(P, D):
    """(byte, shift) [2, P, D] of every nibble of a block: keys, values."""
    t, d = np.arange(P)[:, None], np.arange(D)[None, :]
    word = ((t // 16 * 4 + d // (D // 4)) * 16 + t % 16) * (D // 32) + d % (D // 4) // 8
    n = np.array(KEY_NIBBLE)[d % 8]
    k = (word * 4 + n // 2, 4 * (n % 2) + 0 * word)
    c, m, j = d // (D // 16), d % (D // 16) // 4, d % 4
    word = ((t // 4 * 16 + c) * 2 + t % 4 // 2) * (D // 64) + m
    n = t % 2 * 4 + j
    v = (P * D // 2 + word * 4 + n // 2, 4 * (n % 2) + 0 * word)
    return k, v


def put(cache, slots, k, v):
    """The fp32 rows k, v [T, H, D] (keys already turned and rotated) into cache, in place."""
    pages, H, P, E = cache.shape
    D = E - 8
    flat = cache.reshape(pages, H, P * E)
    where = places(P, D)
    for which, x in enumerate((k, v)):
        codes, words = quantize(x)
        byte, shift = where[which]
        for i, slot in enumerate(slots):
            if not 0 <= slot < pages * P:
                continue
            page, t = divmod(int(slot), P)
            for h in range(H):
                for d in range(D):
                    at, s = byte[t, d], shift[t, d]
                    flat[page, h, at] = (flat[page, h, at] & ~(15 << s) & 255) | codes[i, h, d] << s
                at = P * D + (which * P + t) * 4
                flat[page, h, at:at + 4] = np.array([words[i, h]], "<u4").view(np.uint8)


def values(cache):
    """(keys, values) [pages, P, H, D] that the cache holds, in fp32 (exactly rounded once)."""
    pages, H, P, E = cache.shape
    D = E - 8
    flat = cache.reshape(pages, H, P * E)
    got = []
    for which, (byte, shift) in enumerate(places(P, D)):
        codes = (flat[:, :, byte] >> shift.astype(np.uint8)) & 15
        at = P * D + which * P * 4
        words = np.ascontiguousarray(flat[:, :, at:at + 4 * P]).view("<u4")
        zero = (words & 15).astype(np.float32)
        x = (codes.astype(np.float32) - zero[..., None]) * words.view(np.float32)[..., None]
        got.append(x.transpose(0, 2, 1, 3))
    return got


def attention(q, k, v, place, scale, window=0, hidden=None):
    """One sequence in 64 bits: q [n, Hq, D], k, v [L, H, D]; query i is at place[i].

    Returns (out [n, Hq, D], lse [n, Hq], spread [n, Hq, D]) with spread = sum p |v|, the size
    that a relative error of the weights shows at."""
    n, Hq, D = q.shape
    L, H, _ = k.shape
    out = np.zeros((n, Hq, D))
    lse = np.full((n, Hq), -np.inf)
    spread = np.zeros((n, Hq, D))
    if L == 0:
        return out, lse, spread
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    j = np.arange(L)
    for i in range(n):
        seen = j <= place[i]
        if window:
            seen &= j > place[i] - window
        if hidden is not None:
            seen &= ~hidden
        if not seen.any():
            continue
        for h in range(Hq):
            g = h // (Hq // H)
            s = scale * (k[seen, g] @ q[i, h])
            m = s.max()
            p = np.exp(s - m)
            lse[i, h] = m + np.log(p.sum())
            p = p / p.sum()
            out[i, h] = p @ v[seen, g]
            spread[i, h] = p @ np.abs(v[seen, g])
    return out, lse, spread
