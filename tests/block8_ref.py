"""Plain evaluations of the 8-bit linear layer in 64 bits (numpy), matrices [n, rows] with dimension 0 along a row."""
import numpy as np

TOP = {"e4m3": 448.0, "e5m2": 57344.0}
LEAST = {"e4m3": -6, "e5m2": -14}                            # exponent of the smallest normal number
DIGITS = {"e4m3": 3, "e5m2": 2}


def _table(fmt):
    bias, digits = (7, 3) if fmt == "e4m3" else (15, 2)
    t = np.zeros(256)
    for c in range(256):
        e, m = (c & 0x7F) >> digits, c & ((1 << digits) - 1)
        v = m * 2.0 ** (1 - bias - digits) if e == 0 else (1 + m * 2.0 ** -digits) * 2.0 ** (e - bias)
        if fmt == "e4m3" and (c & 0x7F) == 0x7F:
            v = np.nan
        if fmt == "e5m2" and e == 31:
            v = np.inf if m == 0 else np.nan
        t[c] = -v if c & 0x80 else v
    return t


TABLE = {f: _table(f) for f in TOP}


def decode(codes, fmt):
    return TABLE[fmt][codes.view(np.uint8)]


def half_step(x, fmt):
    """Half the distance of neighbouring codes at x."""
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** LEAST[fmt])))
    return 2.0 ** (e - DIGITS[fmt] - 1)


def scales(x, block, fmt):
    n, rows = x.shape
    nb, rb = -(-n // 128), -(-rows // block)
    out = np.zeros((rb, nb))
    for i in range(rb):
        for j in range(nb):
            out[i, j] = max(np.abs(x[j * 128:(j + 1) * 128, i * block:(i + 1) * block]).max() / TOP[fmt], 2.0 ** -126)
    return out


def spread(scale, n, rows, block):
    """A scale for each element of [n, rows]."""
    return np.repeat(np.repeat(scale, block, 0)[:rows], 128, 1)[:, :n].T


def rms_norm(h, w, eps):
    y = h / np.sqrt((h * h).mean(0) + eps)
    return y if w is None else y * w.astype(np.float64)[:, None]


def rms_norm_grad(dy, h, w, eps, dres):
    """dh, dweight and for each the magnitudes that their terms had."""
    dy, h, w = dy.astype(np.float64), h.astype(np.float64), w.astype(np.float64)[:, None]
    r = 1 / np.sqrt((h * h).mean(0) + eps)
    g = dy * w
    dh = r * g - h * r ** 3 * (g * h).mean(0)
    mag = r * np.abs(g) + np.abs(h) * r ** 3 * np.abs(g * h).mean(0)
    if dres is not None:
        dh, mag = dh + dres.astype(np.float64), mag + np.abs(dres.astype(np.float64))
    return dh, (dy * h * r).sum(1), mag, np.abs(dy * h * r).sum(1)


def block_gemm(ca, sa, block_a, fa, cb, sb, block_b, fb):
    """c and the sum of its terms' magnitudes."""
    a = decode(ca, fa) * spread(sa.astype(np.float64), *ca.shape, block_a)
    b = decode(cb, fb) * spread(sb.astype(np.float64), *cb.shape, block_b)
    return a.T @ b, np.abs(a).T @ np.abs(b)
