"""MX4 values and the 8-bit paged cache, restated on the CPU in 64 bits.

mx4_quantize / mx4_decode: the 4-bit microscaling format (E2M1 codes, E8M0 scales, blocks of 32).
append / attention: the paged cache's writes, exactly, and softmax attention over it.
"""
import math

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _nearest_even(u, grid):
    """Index of the grid value nearest u >= 0 (saturating); of two equally near, the even index."""
    hi = np.searchsorted(grid, u).clip(0, len(grid) - 1)
    lo = (hi - 1).clip(0)
    dl, dh = u - grid[lo], grid[hi] - u
    return np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)) | (u >= grid[-1]), hi, lo)


def mx4_quantize(x):
    """x [rows, K] -> codes uint8 [rows, kb, 16], scales uint8 [rows, kb]."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    kb = -(-K // 32)
    z = np.zeros((rows, kb * 32))
    z[:, :K] = x
    z = z.reshape(rows, kb, 32)
    bad = ~np.isfinite(z).all(-1)
    z = np.where(bad[..., None], 0.0, z)
    top = np.abs(z).max(-1)
    byte = np.where(top > 0, np.frexp(top)[1] - 1 + 125, 0).clip(0)
    u = np.abs(z) / np.ldexp(1.0, byte - 127)[..., None]
    code = _nearest_even(u, E2M1) + 8 * np.signbit(z)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), np.where(bad, 255, byte).astype(np.uint8)


def mx4_decode(codes, scales):
    """-> float64 [rows, kb * 32]."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(*scales.shape, 32)
    v = E2M1[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return (v * s[..., None]).reshape(scales.shape[0], scales.shape[1] * 32)


def e4m3_table():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * np.ldexp(1.0, e - 7))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


E4M3 = e4m3_table()


def decode8(codes, kind):
    """uint8 storage -> float64 values."""
    return codes.view(np.int8).astype(np.float64) if kind == "int8" else E4M3[codes]


def encode8(x, kind):
    """Nearest code, ties to even; |x| at most the largest code."""
    if kind == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    return (_nearest_even(np.abs(x), E4M3[:127]) | (np.signbit(x).astype(int) << 7)).astype(np.uint8)


QMAX = {"int8": 127.0, "e4m3": 448.0}


def exponent(r, kind):
    e = max(-126, math.frexp(r)[1] - 12)
    while r > QMAX[kind] * 2.0 ** e:
        e += 1
    return e


def append(x, codes, scales, table, lengths, counts, kind):
    """x [T, H, D] into codes uint8 [P, H, page, D], scales float32 [P, H], in place. Returns whether a row was left out."""
    page, P = codes.shape[2], codes.shape[0]
    first, bad = 0, False
    for b, n in enumerate(counts):
        at = int(lengths[b]) - n
        while at < lengths[b]:
            stop = min(int(lengths[b]), (at // page + 1) * page)
            pi = at // page
            p = int(table[b, pi]) if 0 <= pi < table.shape[1] else -1
            if not 0 <= p < P:
                bad = True
            else:
                lo = first + at - (int(lengths[b]) - n)
                s = at - pi * page
                for h in range(codes.shape[1]):
                    new = np.asarray(x[lo:lo + stop - at, h], np.float64)
                    old = np.float32(0) if s == 0 else scales[p, h]
                    top = np.abs(new).max()
                    if not np.isfinite(new).all():
                        now = np.float32(np.nan)
                    elif not old != 0:
                        now = np.float32(2.0 ** exponent(float(top), kind)) if top else np.float32(0)
                    elif not old > 0 or np.isinf(old):
                        now = old
                    else:
                        (mt, et), (mo, eo) = math.frexp(top), math.frexp(old)  # a float32 quotient of any exponent
                        g = max(0, exponent(float(np.float32(mt) / np.float32(mo)), kind) + et - eo) if top else 0
                        now = np.float32(float(old) * 2.0 ** g)
                        if g:
                            codes[p, h, :s] = encode8(decode8(codes[p, h, :s], kind) / 2.0 ** g, kind)
                    scales[p, h] = now
                    if now > 0 and np.isfinite(now):
                        with np.errstate(over="ignore", under="ignore"):
                            y = (new.astype(np.float32) / now).astype(np.float64)
                        codes[p, h, s:s + stop - at] = encode8(y.clip(-QMAX[kind], QMAX[kind]), kind)
                    else:
                        codes[p, h, s:s + stop - at] = 0
            at = stop
        first += n
    return bad


def attention(q, k_codes, v_codes, k_scales, v_scales, table, lengths, counts, kind, *, scale, causal=True, window=0):
    """-> (o float64 [T, Hq, D], sum of p |v| alike, largest sum of |q k| scale of each row [T, Hq])."""
    q = np.asarray(q, np.float64)
    T, Hq, D = q.shape
    P, H, page, _ = k_codes.shape
    o, av, aqk = np.zeros((T, Hq, D)), np.zeros((T, Hq, D)), np.zeros((T, Hq))
    first = 0
    for b, n in enumerate(counts):
        L = int(lengths[b])
        if L > 0 and n:
            t = np.arange(L)
            idx = t // page
            pages = np.where(idx < table.shape[1], table[b, np.minimum(idx, table.shape[1] - 1)], -1)
            have = (pages >= 0) & (pages < P)
            pages = np.where(have, pages, 0)
            K = decode8(k_codes[pages, :, t % page], kind) * k_scales[pages].astype(np.float64)[..., None]
            V = decode8(v_codes[pages, :, t % page], kind) * v_scales[pages].astype(np.float64)[..., None]
            for i in range(n):
                p = L - n + i
                see = have.copy()
                if causal:
                    see &= t <= p
                if window:
                    see &= t > p - window
                if not see.any():
                    continue
                for h in range(Hq):
                    kk, vv = K[see, h // (Hq // H)], V[see, h // (Hq // H)]
                    s = kk @ q[first + i, h] * scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    o[first + i, h], av[first + i, h] = w @ vv, w @ np.abs(vv)
                    aqk[first + i, h] = (np.abs(kk) @ np.abs(q[first + i, h])).max() * abs(scale)
        first += n
    return o, av, aqk


def attention_of_all(q, k_codes, v_codes, k_scales, v_scales, table, lengths, counts, kind, *, scale, causal=True, window=0):
    """What attention gives, with all rows of a key head at once, for caches whose values are finite."""
    q = np.asarray(q, np.float64)
    T, Hq, D = q.shape
    P, H, page, _ = k_codes.shape
    G = Hq // H
    o, av, aqk = np.zeros((T, Hq, D)), np.zeros((T, Hq, D)), np.zeros((T, Hq))
    first = 0
    for b, n in enumerate(counts):
        L = int(lengths[b])
        if L > 0 and n:
            t, p = np.arange(L), np.arange(L - n, L)[:, None]
            pages = np.where(t // page < table.shape[1], table[b, np.minimum(t // page, table.shape[1] - 1)], -1)
            have = (pages >= 0) & (pages < P)
            pages = np.where(have, pages, 0)
            see = np.broadcast_to(have, (n, L))
            if causal:
                see = see & (t <= p)
            if window:
                see = see & (t > p - window)
            see = np.repeat(see, G, 0)  # [n G, L]
            any_ = see.any(1, keepdims=True)
            for h in range(H):
                kk, vv = (decode8(c[pages, h, t % page], kind) * s[pages, h].astype(np.float64)[:, None]
                          for c, s in ((k_codes, k_scales), (v_codes, v_scales)))
                qq = q[first:first + n, h * G:(h + 1) * G].reshape(n * G, D)
                z = np.where(see, qq @ kk.T * scale, -np.inf)
                w = np.exp(z - np.where(any_, z.max(1, keepdims=True), 0.0))
                w /= np.where(any_, w.sum(1, keepdims=True), 1.0)
                to = np.s_[first:first + n, h * G:(h + 1) * G]
                o[to], av[to] = (w @ vv).reshape(n, G, D), (w @ np.abs(vv)).reshape(n, G, D)
                aqk[to] = np.where(see, np.abs(qq) @ np.abs(kk).T, 0.0).max(1).reshape(n, G) * abs(scale)
        first += n
    return o, av, aqk
