"""The norms of the 8-bit linear layer over many rows: every block works through several times as many rows as its ring in
shared memory has places, so that places are filled again and their barriers come round; with residuals that are absent,
whole and off 16-byte boundaries.  Bounds as for few rows: a row's arithmetic does not depend on the others, and a
column's sum has one rounding more for each row."""
import numpy as np
import pytest

import block8_ref as ref
from solid_b200 import ops
from test_gpu_block8 import ACC, EPS, STEP, TINY, got, norm_bounds, roundings, upload, values

pytestmark = pytest.mark.gpu

# rows at once on 148 SMs: at most 16 blocks an SM with four places each (520), 4 with four (4096), 1 with two or three (16384)
SHAPES = [("half", 4096, 2400), ("half", 16384, 600), ("half", 520, 12000), ("half", 256, 8000), ("half", 1000, 6000), ("half", 1001, 2500),
          ("float", 4096, 1500), ("float", 8192, 600), ("float", 520, 10000), ("float", 9000, 500), ("float", 15000, 350), ("float", 4095, 500),
          ("double", 2048, 1500), ("double", 7500, 400), ("double", 1024, 3000)]


def residual(kind, rng, n, rows, dtype):
    """(numpy, tensor) of a residual: absent, beside x, or with rows off 16-byte boundaries."""
    if kind == "none":
        return None, None
    r = values(rng, n, rows, dtype)
    return r, upload(r, dtype, pad=0 if kind == "whole" else 1)


@pytest.mark.parametrize("kind", ["none", "whole", "padded"])
@pytest.mark.parametrize("dtype,n,rows", SHAPES)
def test_norm(gpu, dtype, n, rows, kind):
    rng = np.random.default_rng(n + rows)
    x, w = values(rng, n, rows, dtype), values(rng, n, 1, dtype)[:, 0]
    r, tr = residual(kind, rng, n, rows, dtype)
    hx = x.astype(np.float64) + (0 if r is None else r.astype(np.float64))
    want = ref.rms_norm(hx, w, EPS)
    tx, tw = upload(x, dtype), upload(w, dtype)
    out = ops.rms_norm(tx, tw, EPS, tr)
    y, h = (out, None) if r is None else out
    assert np.all(np.abs(got(y) - want) <= norm_bounds(dtype, n, want))
    if r is not None:
        assert np.all(np.abs(got(h) - hx) <= (STEP[dtype] + ACC[dtype]) * np.abs(hx) + TINY[dtype])
        again = ops.rms_norm(tx, tw, EPS, tr, dst=tx, h=tr)  # in the inputs' places
        assert again[0] is tx and again[1] is tr and np.array_equal(got(tx), got(y)) and np.array_equal(got(tr), got(h))


@pytest.mark.parametrize("kind", ["none", "whole", "padded"])
@pytest.mark.parametrize("dtype,n,rows", SHAPES)
def test_norm_to_codes(gpu, dtype, n, rows, kind):
    rng = np.random.default_rng(n + 2 * rows)
    fmt = "e5m2" if rows % 3 == 0 else "e4m3"
    x, w = values(rng, n, rows, dtype), values(rng, n, 1, dtype)[:, 0]
    r, tr = residual(kind, rng, n, rows, dtype)
    hx = x.astype(np.float64) + (0 if r is None else r.astype(np.float64))
    y = ref.rms_norm(hx, w, EPS)
    out = ops.rms_norm_quantize(upload(x, dtype), upload(w, dtype), EPS, tr, fmt)
    q, h = (out, None) if r is None else out
    if r is not None:
        assert np.all(np.abs(got(h) - hx) <= (STEP[dtype] + ACC[dtype]) * np.abs(hx) + TINY[dtype])
    nb = (n + 127) // 128
    full = np.zeros((nb * 128, rows))
    full[:n] = np.abs(y)
    want = np.maximum(full.reshape(nb, 128, rows).max(1).T / ref.TOP[fmt], 2.0 ** -126)
    scale, code = q.scales.numpy().astype(np.float64), ref.decode(q.codes.numpy(), fmt)
    slack = 2.0 ** -24 * (roundings(n) / 2 + 12)             # of y, as for few rows
    assert np.all(np.abs(scale - want) <= (slack + 2 * 2.0 ** -24) * want)
    exact = y / np.repeat(scale, 128, 1)[:, :n].T
    limit = ref.half_step(np.abs(exact) * (1 + 2.0 ** -20 + slack), fmt) + np.abs(exact) * (slack + 2.0 ** -21)
    assert np.all(np.abs(code - exact) <= limit)


@pytest.mark.parametrize("kind", ["none", "whole", "padded"])
@pytest.mark.parametrize("dtype,n,rows", SHAPES)
def test_gradient(gpu, dtype, n, rows, kind):
    rng = np.random.default_rng(n + 3 * rows)
    h, w = values(rng, n, rows, dtype), values(rng, n, 1, dtype)[:, 0]
    dy = (rng.standard_normal((n, rows)) * 0.01).astype(h.dtype)
    r, tr = residual(kind, rng, n, rows, dtype)
    dh, dw = ops.rms_norm_grad(upload(dy, dtype), upload(h, dtype), upload(w, dtype), EPS, tr)
    want, wantw, mag, magw = ref.rms_norm_grad(dy, h, w, EPS, r)
    assert np.all(np.abs(got(dh) - want) <= STEP[dtype] * np.abs(want) + TINY[dtype] + ACC[dtype] * (2 * roundings(n) + 16) * mag)
    assert np.all(np.abs(dw.numpy() - wantw) <= ACC[dtype] * (roundings(n) / 2 + rows + 16) * magw)


@pytest.mark.parametrize("n,rows", [(64, 40), (1000, 30), (1001, 30), (4096, 700), (16384, 400), (17000, 9)])
def test_gradient_of_what_is_not_finite(gpu, n, rows):
    """A NaN or an infinity in dy or h: its row of dh is not finite, the others have the bits that they have without it; the
    weights' gradient is lost where the row's own terms are."""
    rng = np.random.default_rng(n)
    h, dy, w = values(rng, n, rows, "float"), values(rng, n, rows, "float"), values(rng, n, 1, "float")[:, 0]
    clean, cleanw = (got(t) for t in ops.rms_norm_grad(upload(dy, "float"), upload(h, "float"), upload(w, "float"), EPS))
    for bad in (np.nan, np.inf, -np.inf):
        row, col = rows // 2, n // 3
        broken = dy.copy()
        broken[col, row] = bad
        dh, dw = (got(t) for t in ops.rms_norm_grad(upload(broken, "float"), upload(h, "float"), upload(w, "float"), EPS))
        rest = np.arange(rows) != row
        assert np.array_equal(dh[:, rest], clean[:, rest]) and not np.any(np.isfinite(dh[:, row]))
        assert not np.isfinite(dw[col]) and np.array_equal(np.delete(dw, col), np.delete(cleanw, col))
        broken = h.copy()
        broken[col, row] = bad
        dh, dw = (got(t) for t in ops.rms_norm_grad(upload(dy, "float"), upload(broken, "float"), upload(w, "float"), EPS))
        assert np.array_equal(dh[:, rest], clean[:, rest]) and np.isnan(dh[col, row]) and np.isnan(dw[col])
