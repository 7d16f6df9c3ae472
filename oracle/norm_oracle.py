"""numpy fp64 oracle of the norm and dropout operators (test infrastructure only).

Dropout's keep decisions: Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
1, 2, 3", SC 2011), key = seed, counter = (column // 8, row, offset low, offset high); the words give eight 16-bit draws,
low half first; dropped where the draw is below round(65536 p)."""
import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=10):
    """counter: four uint64 arrays of 32-bit values, key: two ints; four uint64 arrays of 32-bit values."""
    a, b, c, d = (np.asarray(v, dtype=np.uint64) for v in counter)
    k0, k1 = key
    for _ in range(rounds):
        p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = ((q >> np.uint64(32)) ^ b ^ np.uint64(k0), q & M32, (p >> np.uint64(32)) ^ d ^ np.uint64(k1), p & M32)
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return a, b, c, d


def threshold(p):
    return int(np.rint(p * 65536.0))


def keep(rows, d, p, seed, offset, first_row=0):
    """(rows, d) bool; row r of the result is row first_row + r of the tensor."""
    t = threshold(p)
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    g = np.arange((d + 7) // 8, dtype=np.uint64)[None, :]
    r = np.arange(first_row, first_row + rows, dtype=np.uint64)[:, None]
    z = np.zeros((rows, g.shape[1]), dtype=np.uint64)
    w = philox4x32((z + g, z + r, z + np.uint64(offset & 0xFFFFFFFF), z + np.uint64(offset >> 32)), (seed & 0xFFFFFFFF, seed >> 32))
    draws = np.stack([h for v in w for h in (v & np.uint64(0xFFFF), v >> np.uint64(16))], axis=2).reshape(rows, -1)[:, :d]
    return draws >= np.uint64(t)


def scale(p):
    t = threshold(p)
    return 0.0 if t >= 65536 else 65536.0 / (65536.0 - t)


def norm_forward(v, w, b, eps, rms):
    """v (rows, d) fp64 -> y, xh, rstd (rows, 1)."""
    c = v if rms else v - v.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    xh = c * rstd
    y = xh if w is None else xh * w
    return (y if b is None else y + b), xh, rstd


def norm_backward(dy, xh, rstd, w, rms):
    """dv, dw, db of y = norm(v) * w + b."""
    g = dy if w is None else dy * w
    dv = g - xh * (g * xh).mean(1, keepdims=True)
    if not rms:
        dv = dv - g.mean(1, keepdims=True)
    return dv * rstd, (dy * xh).sum(0), dy.sum(0)
