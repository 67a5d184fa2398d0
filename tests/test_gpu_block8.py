"""The 8-bit linear layer against plain evaluations in 64 bits: rms_norm, rms_norm_quantize, rms_norm_grad,
block_quantize and block_gemm.

Roundings counted in the tolerances: half 2^-11 (and 2^-25 below its smallest normal number), float 2^-24, e4m3 2^-4,
e5m2 2^-3 of the value, each at most half a step.  A sum of n terms in 32 bits is off by at most about log2(n) + 16
roundings of the terms' magnitudes in the kernels' order (runs of at most 16 terms a thread, then trees and short chains
over warps); U(n) below counts them.
"""
import numpy as np
import pytest

import block8_ref as ref
from solid_b200 import Tensor, ops

pytestmark = pytest.mark.gpu

EPS = 1e-6
STEP = {"half": 2.0 ** -11, "float": 2.0 ** -24, "double": 2.0 ** -53}          # half a unit of the last place
TINY = {"half": 2.0 ** -25, "float": 2.0 ** -150, "double": 0.0}
ACC = {"half": 2.0 ** -24, "float": 2.0 ** -24, "double": 2.0 ** -53}           # of the arithmetic


def roundings(n):
    """Roundings on the longest path of a sum of n terms: 128 in a thread's own chain at most, the trees, and warps."""
    return min(n, 128) + 64


def upload(x, dtype, pad=0, turned=False):
    """[n, rows] numpy -> Tensor; pad: extra elements between rows; turned: contiguous along the rows' dimension."""
    if not pad and not turned:
        return Tensor.from_numpy(x, dtype)
    if turned:
        return upload(np.ascontiguousarray(x.T), dtype, pad).T
    n, rows = x.shape
    full = np.zeros((n + pad, rows), x.dtype)
    full[:n] = x
    return Tensor.from_numpy(full, dtype).slice(0, 0, n)


def values(rng, n, rows, dtype):
    x = rng.standard_normal((n, rows)) * np.exp(rng.standard_normal((n, 1)))
    return x.astype({"half": np.float16, "float": np.float32, "double": np.float64}[dtype])


def got(t):
    a = t.numpy()
    return a.view(np.float16) if t.dtype == "half" else a


def norm_bounds(dtype, n, want):
    """y = h r w: the sum's roundings enter r by half; the residual's addition, the square
    root, the quotient and two products add six."""
    return (STEP[dtype] + ACC[dtype] * (roundings(n) / 2 + 8)) * np.abs(want) + TINY[dtype]


SHAPES = [(1, 1), (7, 3), (64, 17), (128, 5), (129, 4), (256, 9), (1000, 7), (1024, 40), (1025, 3), (2048, 2), (2056, 3), (4096, 1),
          (4096, 300), (6144, 5), (8191, 2), (8192, 151), (8200, 2), (16384, 3), (16385, 2), (40000, 2)]


@pytest.mark.parametrize("dtype", ["half", "float", "double"])
@pytest.mark.parametrize("n,rows", SHAPES)
def test_rms_norm(gpu, dtype, n, rows):
    rng = np.random.default_rng(n * 7 + rows)
    x, r = values(rng, n, rows, dtype), values(rng, n, rows, dtype)
    w = (1 + 0.1 * rng.standard_normal(n)).astype(x.dtype)
    x[:, rows // 2] = 0                                      # a row of zeros beside its residual
    tx, tr, tw = upload(x, dtype), upload(r, dtype, pad=3), upload(w, dtype)
    y, h = ops.rms_norm(tx, tw, EPS, tr)
    hx = x.astype(np.float64) + r.astype(np.float64)
    want = ref.rms_norm(hx, w, EPS)
    assert np.all(np.abs(got(y) - want) <= norm_bounds(dtype, n, want))
    assert np.all(np.abs(got(h) - hx) <= (STEP[dtype] + ACC[dtype]) * np.abs(hx) + TINY[dtype])
    y = ops.rms_norm(tx, None, EPS)                          # no residual, no weights; one row is all zeros
    want = ref.rms_norm(x.astype(np.float64), None, EPS)
    assert np.all(np.abs(got(y) - want) <= norm_bounds(dtype, n, want))
    assert not np.any(got(y)[:, rows // 2])


@pytest.mark.parametrize("dtype", ["half", "float", "double"])
def test_rms_norm_strides_and_places(gpu, dtype):
    """Turned and padded operands, a result and h in place of the inputs, further dimensions, a stream of its own."""
    import torch
    rng = np.random.default_rng(5)
    n, rows = 520, 24
    x, r = values(rng, n, rows, dtype), values(rng, n, rows, dtype)
    w = (1 + 0.1 * rng.standard_normal(n)).astype(x.dtype)
    y0, h0 = ops.rms_norm(upload(x, dtype), upload(w, dtype), EPS, upload(r, dtype))
    y0, h0 = got(y0), got(h0)
    tol = 2 * norm_bounds(dtype, n, y0.astype(np.float64))   # two kernels, each within the bound of the same value
    for kind in (dict(pad=8), dict(pad=1), dict(turned=True), dict(turned=True, pad=5)):
        tx, tr = upload(x, dtype, **kind), upload(r, dtype, **kind)
        y, h = ops.rms_norm(tx, upload(w, dtype), EPS, tr, dst=tx, h=tr)
        assert y is tx and h is tr
        assert np.all(np.abs(got(y).astype(np.float64) - y0) <= tol) and np.array_equal(got(h), h0)
    s = torch.cuda.Stream()
    tx = Tensor.from_numpy(x.reshape(n, 4, 6, order="F"), dtype)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.rms_norm(tx, upload(w, dtype), EPS)
    torch.cuda.current_stream().wait_stream(s)
    assert y.size == [n, 4, 6]
    assert np.array_equal(got(y).reshape(n, rows, order="F"), got(ops.rms_norm(upload(x, dtype), upload(w, dtype), EPS)))


def check_blocks(q, x, block, fmt, slack):
    """Codes and scales of x (64 bits, [n, rows]).  slack: relative error of the values that were converted."""
    scale, code = q.scales.numpy().astype(np.float64), ref.decode(q.codes.numpy(), fmt)
    want = ref.scales(x, block, fmt)
    assert scale.shape == want.shape
    assert np.all(np.abs(scale - want) <= (slack + 2 * 2.0 ** -24) * want)
    n, rows = x.shape
    spread = ref.spread(scale, n, rows, block)
    # half a step of the format, plus what the value, its scale and the quotient were off by
    limit = ref.half_step(np.abs(x) / spread * (1 + 2.0 ** -20 + slack), fmt) + np.abs(x) / spread * (slack + 2.0 ** -21)
    assert np.all(np.abs(code - x / spread) <= limit)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["half", "float", "double"])
@pytest.mark.parametrize("n,rows", [(1, 1), (100, 3), (128, 20), (200, 5), (256, 4), (1000, 7), (1024, 9), (4096, 2), (8192, 150),
                                    (5000, 3), (16384, 2), (20001, 2)])
def test_rms_norm_quantize(gpu, dtype, fmt, n, rows):
    rng = np.random.default_rng(n + rows)
    x, r = values(rng, n, rows, dtype), values(rng, n, rows, dtype)
    w = (1 + 0.1 * rng.standard_normal(n)).astype(x.dtype)
    q, h = ops.rms_norm_quantize(upload(x, dtype), upload(w, dtype), EPS, upload(r, dtype, pad=1), fmt)
    hx = x.astype(np.float64) + r.astype(np.float64)
    y = ref.rms_norm(hx, w, EPS)
    # cancellation in x + r: the sum is rounded once in 32 bits, exact for halves
    check_blocks(q, y, 1, fmt, 2.0 ** -24 * (roundings(n) / 2 + 12))
    assert np.all(np.abs(got(h) - hx) <= (STEP[dtype] + ACC[dtype]) * np.abs(hx) + TINY[dtype])


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("dtype,fmt", [("half", "e4m3"), ("float", "e4m3"), ("float", "e5m2"), ("double", "e4m3")])
@pytest.mark.parametrize("n,rows,kind", [(1, 1, {}), (128, 128, {}), (256, 300, {}), (1000, 130, {}), (129, 257, dict(pad=1)),
                                         (300, 200, dict(turned=True)), (256, 384, dict(turned=True)), (77, 129, dict(turned=True, pad=1)),
                                         (4096, 3, {}), (3, 4096, {})])
def test_block_quantize(gpu, dtype, fmt, block, n, rows, kind):
    rng = np.random.default_rng(n + 3 * rows + block)
    x = values(rng, n, rows, dtype)
    x[: n // 2, 0] = 0
    q = ops.block_quantize(upload(x, dtype, **kind), block, fmt)
    check_blocks(q, x.astype(np.float64), block, fmt, 2.0 ** -24 if dtype == "double" else 0.0)


def test_block_quantize_special_values(gpu):
    """Zeros, subnormals, the largest numbers, and blocks that hold an infinity or a NaN."""
    x = np.zeros((512, 3), np.float32)
    x[0, 1] = 3.4e38; x[1, 1] = 1e30
    x[128, 1] = 1e-40; x[129, 1] = -2e-41
    x[256, 1] = np.inf; x[257, 1] = 1.0
    x[384, 1] = np.nan; x[385, 1] = 1.0
    for kind in ({}, dict(turned=True), dict(pad=1)):
        q = ops.block_quantize(upload(x, "float", **kind))
        s, c = q.scales.numpy(), ref.decode(q.codes.numpy(), "e4m3")
        assert np.all(s[0] == 2.0 ** -126) and not np.any(c[:, 0])
        assert c[0, 1] == 448 and s[1, 0] >= 3.3e38 / 448 and np.all(c[2:128, 1] == 0)
        # 1e-40 / 2^-126 = 0.0085 = 4.36 of the smallest code's 2^-9, 2e-41 is 0.87 of it
        assert s[1, 1] == 2.0 ** -126 and c[128, 1] == 4 / 512 and c[129, 1] == -1 / 512 and not np.any(c[130:256, 1])
        assert np.isinf(s[1, 2]) and np.isnan(c[256, 1]) and c[257, 1] == 0
        assert np.isnan(s[1, 3]) and np.all(np.isnan(c[384:, 1]))


@pytest.mark.parametrize("dtype", ["half", "float", "double"])
@pytest.mark.parametrize("n,rows", [(1, 1), (7, 3), (64, 170), (128, 33), (300, 20), (512, 1300), (1000, 77), (1024, 9), (2048, 40), (4096, 400),
                                    (5000, 3), (8192, 20), (8191, 5), (12000, 3), (16384, 2), (17000, 40)])
def test_rms_norm_grad(gpu, dtype, n, rows):
    rng = np.random.default_rng(3 * n + rows)
    h, dres = values(rng, n, rows, dtype), values(rng, n, rows, dtype)
    dy = (rng.standard_normal((n, rows)) * 0.01).astype(h.dtype)
    w = (1 + 0.1 * rng.standard_normal(n)).astype(h.dtype)
    for res, kind in ((dres, {}), (None, dict(pad=1))):
        dh, dw = ops.rms_norm_grad(upload(dy, dtype, **kind), upload(h, dtype, **kind), upload(w, dtype), EPS,
                                   None if res is None else upload(res, dtype, **kind))
        want, wantw, mag, magw = ref.rms_norm_grad(dy, h, w, EPS, res)
        bound = STEP[dtype] * np.abs(want) + TINY[dtype] + ACC[dtype] * (2 * roundings(n) + 16) * mag
        assert np.all(np.abs(got(dh) - want) <= bound)
        # a column's sum: rows in a chain within a block, then the blocks
        assert np.all(np.abs(dw.numpy() - wantw) <= ACC[dtype] * (roundings(n) / 2 + rows + 16) * magw)


def operand(rng, k, rows, block, fmt):
    """Codes of every finite value and scales over some octaves, as numpy and as Blocks with padded rows."""
    top = 0x7E if fmt == "e4m3" else 0x7B
    codes = (rng.integers(0, top + 1, (k, rows)) | (rng.integers(0, 2, (k, rows)) << 7)).astype(np.uint8)
    scales = np.exp2(rng.uniform(-4, 4, ((rows + block - 1) // block, (k + 127) // 128))).astype(np.float32)
    ld = (k + 15) // 16 * 16
    full = np.full((ld, rows), 0x7F, np.uint8)               # NaN codes behind the rows: they belong to nobody
    full[:k] = codes
    return codes, scales, ops.Blocks(Tensor.from_numpy(full, "uint8").slice(0, 0, k), Tensor.from_numpy(scales, "float"), fmt)


GEMM = [(1, 1, 1), (1, 1, 128), (128, 1, 128), (300, 1, 1000), (4096, 1, 4096), (129, 3, 256), (257, 16, 384), (512, 17, 640), (1000, 33, 512),
        (640, 64, 1500), (384, 100, 256), (128, 128, 128), (130, 129, 130), (300, 520, 700), (1024, 2048, 512), (2500, 2300, 260), (5, 700, 900)]


@pytest.mark.parametrize("m,n,k", GEMM)
@pytest.mark.parametrize("block_a,block_b,fa,fb,dtype", [(128, 1, "e4m3", "e4m3", "half"), (128, 1, "e4m3", "e4m3", "float"),
                                                         (1, 1, "e5m2", "e4m3", "float"), (128, 128, "e4m3", "e5m2", "float")])
def test_block_gemm(gpu, m, n, k, block_a, block_b, fa, fb, dtype):
    rng = np.random.default_rng(m + 3 * n + 5 * k)
    ca, sa, a = operand(rng, k, m, block_a, fa)
    cb, sb, b = operand(rng, k, n, block_b, fb)
    if dtype == "half":                                      # keep the results inside half's range
        sa *= 2.0 ** -14
        a = ops.Blocks(a.codes, Tensor.from_numpy(sa, "float"), fa)
    want, mag = ref.block_gemm(ca, sa, block_a, fa, cb, sb, block_b, fb)
    c = ops.block_gemm(a, b, dtype)
    assert c.size == [m, n]
    # products of codes are exact; 128 of them and their sums, two scales, then one addition for each block of 128
    tol = 2.0 ** -24 * (128 + 8 + k / 128) * mag + STEP[dtype] * np.abs(want) + TINY[dtype]
    assert np.all(np.abs(got(c) - want) <= tol)
    turned = ops.block_gemm(a, b, dtype, dst=Tensor.empty([n, m], dtype).T)      # rows of c contiguous instead
    assert np.all(np.abs(got(turned) - want) <= tol)


@pytest.mark.parametrize("m,n,k", [(1, 1, 5), (70, 3, 200), (200, 150, 333)])
def test_block_gemm_unaligned(gpu, m, n, k):
    """Codes off 16-byte boundaries, and a result with gaps whose other elements stay."""
    rng = np.random.default_rng(k)
    ca, sa, _ = operand(rng, k, m, 1, "e4m3")
    cb, sb, _ = operand(rng, k, n, 128, "e4m3")
    want, mag = ref.block_gemm(ca, sa, 1, "e4m3", cb, sb, 128, "e4m3")
    full = Tensor.from_numpy(np.full((m + 3, n), 7, np.float32), "float")
    a = ops.Blocks(upload(ca, "uint8", pad=1), Tensor.from_numpy(sa, "float"))
    b = ops.Blocks(upload(cb, "uint8", pad=3), Tensor.from_numpy(sb, "float"))
    c = ops.block_gemm(a, b, "float", dst=full.slice(0, 0, m))
    assert np.all(np.abs(c.numpy() - want) <= 2.0 ** -24 * (128 + 8 + k / 128) * mag + 2.0 ** -24 * np.abs(want))
    assert np.all(full.numpy()[m:] == 7)


def test_empty(gpu):
    e = Tensor.empty([0, 4], "half")
    assert ops.rms_norm(e).size == [0, 4]
    assert ops.rms_norm(Tensor.empty([4, 0], "half")).size == [4, 0]
    dh, dw = ops.rms_norm_grad(Tensor.empty([4, 0], "half"), Tensor.empty([4, 0], "half"))
    assert dh.size == [4, 0] and np.array_equal(dw.numpy(), np.zeros(4, np.float32))
    q = ops.block_quantize(Tensor.empty([0, 4], "half"))
    c = ops.block_gemm(q, q, "float")                        # a depth of zero: sums of nothing
    assert np.array_equal(c.numpy(), np.zeros((4, 4), np.float32))
