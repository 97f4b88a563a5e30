"""Plain 64-bit integer forms of the ring products and of rotary positions, written from their formulas on numpy words."""
import numpy as np

DIGITS_LOW = np.uint64(0x7f7f7f7f7f7f7f80)    # every balanced byte digit is -128: sum of -128 * 256^i mod 2^64


def mask(bw):
    return np.uint64((1 << bw) - 1)


def words(seed, shape, bw=64):
    return np.random.default_rng(seed).integers(0, 1 << 64, shape, dtype=np.uint64) & mask(bw)


def product(x, w, bw, offsets=None, rows=None, share1=None, add=None, out=None):
    """out[r] = add[r] + W_g (x[t] + share1[t]); numpy's uint64 products and sums wrap modulo 2^64"""
    x = x if share1 is None else x + share1
    n = len(x) if rows is None else len(rows)
    out = np.zeros((n, w.shape[1]), np.uint64) if out is None else out.copy()
    off = [0, n] if offsets is None else offsets
    w = w.astype(np.int64).view(np.uint64)
    for g in range(w.shape[0]):
        for r in range(off[g], off[g + 1]):
            t = r if rows is None else rows[r]
            xr = x[t] if 0 <= t < len(x) else np.zeros_like(x[0])
            y = (w[g] * xr[None, :]).sum(axis=1, dtype=np.uint64)
            out[r] = (y if add is None else y + (add if add.ndim == 1 else add[r])) & mask(bw)
    return out


def coefficients(pos, phases, frac, amplitude=1.0):
    """round(amplitude 2^frac cos / sin(2 pi p f / 2^64)) in extended precision -> two uint64 arrays [tokens, pairs]"""
    turn = pos.astype(np.int64).view(np.uint64)[:, None] * np.array(phases, np.uint64)[None, :]
    angle = turn.astype(np.longdouble) * (np.longdouble("6.28318530717958647692528676655900576839") / np.longdouble(2) ** 64)
    whole = np.longdouble(amplitude) * np.longdouble(1 << frac)
    return tuple(np.rint(f(angle) * whole).astype(np.int64).view(np.uint64) for f in (np.cos, np.sin))


def rotary(x, pos, phases, frac, bw, interleaved=False, amplitude=1.0):
    """x uint64 [tokens, heads, dim] -> turned and scaled by 2^frac"""
    half = len(phases)
    c, s = coefficients(pos, phases, frac, amplitude)
    out = x << np.uint64(frac)
    for i in range(half):
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        out[:, :, p] = x[:, :, p] * c[:, i, None] - x[:, :, q] * s[:, i, None]
        out[:, :, q] = x[:, :, q] * c[:, i, None] + x[:, :, p] * s[:, i, None]
    return out & mask(bw)
