"""The 8-bit linear layer at the ends of what it accepts: places that a caller's own allocator gives, numbers near the ends
of their type's range."""
import numpy as np
import pytest

import block8_ref as ref
from solid_b200 import Tensor, ops
from solid_b200._lib import Matrix
from test_gpu_block8 import ACC, EPS, STEP, got, operand, roundings, upload, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["half", "float", "double"])
@pytest.mark.parametrize("n,rows", [(40, 100), (264, 30), (1024, 300), (4096, 200), (8192, 5), (16384, 3), (17001, 4)])
def test_scratch_at_any_element(gpu, dtype, n, rows):
    """The gradient's buffer at every place of an arena that its alignment allows: the same bits, and nothing behind its end."""
    import torch
    from solid_b200 import _lib
    lib, rng = _lib.get(), np.random.default_rng(n)
    es, ws = {"half": (2, 4), "float": (4, 4), "double": (8, 8)}[dtype]
    dy, h, w = (upload(values(rng, *s, dtype), dtype) for s in ((n, rows), (n, rows), (n, 1)))
    want, wantw = ops.rms_norm_grad(dy, h, w.as_strided([n], [es]), EPS)
    size = lib.rms_norm_grad_buffer_size(dtype, n, rows, 0)
    for place in range(0, 32, ws):
        arena = torch.full((place + size + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        dh, dw = Tensor.empty([n, rows], dtype), Tensor.empty([n], "double" if dtype == "double" else "float")
        lib.rms_norm_grad(dtype, n, rows, Matrix(dy.ptr, es, es * n), Matrix(h.ptr, es, es * n), w.ptr, EPS, None,
                          Matrix(dh.ptr, es, es * n), dw.ptr, arena.data_ptr() + place, torch.cuda.current_stream().cuda_stream)
        assert np.array_equal(got(dh), got(want)) and np.array_equal(dw.numpy(), wantw.numpy())
        around = arena.cpu().numpy()
        assert np.all(around[:place] == 0xA5) and np.all(around[place + size:] == 0xA5)


@pytest.mark.parametrize("dtype", ["float", "double"])
@pytest.mark.parametrize("exponent", [50, -43])
@pytest.mark.parametrize("n,rows,pad", [(64, 20, 0), (77, 9, 1), (1000, 30, 0), (1001, 5, 1), (4096, 400, 0), (8192, 20, 0), (16384, 2, 0), (17000, 4, 0)])
def test_gradient_of_large_and_small_rows(gpu, dtype, exponent, n, rows, pad):
    """Rows of 1e15 and of 1e-13 with eps 0: r^3 is beyond the range of 32 bits, the gradient is not.  The bounds are those
    of ordinary rows: a power of two changes no rounding."""
    rng = np.random.default_rng(n)
    h = values(rng, n, rows, dtype) * (np.float32 if dtype == "float" else np.float64)(2.0 ** exponent)
    dy, w = (values(rng, n, rows, dtype) * h.dtype.type(0.01)), values(rng, n, 1, dtype)[:, 0]
    dh, dw = ops.rms_norm_grad(upload(dy, dtype, pad), upload(h, dtype, pad), upload(w, dtype), 0.0)
    want, wantw, mag, magw = ref.rms_norm_grad(dy, h, w, 0.0, None)
    assert np.all(np.abs(got(dh) - want) <= STEP[dtype] * np.abs(want) + ACC[dtype] * (2 * roundings(n) + 16) * mag)
    assert np.all(np.abs(dw.numpy() - wantw) <= ACC[dtype] * (roundings(n) / 2 + rows + 16) * magw)


EXPONENTS = np.array([-149, -140, -126, -110, -91, -89, -60, -20, 0, 20, 60, 87, 89, 100, 119, 127])


@pytest.mark.parametrize("m,n,k", [(300, 1, 1000), (129, 3, 256), (512, 17, 640), (640, 64, 1500), (384, 100, 256), (128, 128, 128), (130, 129, 130),
                                   (300, 520, 700), (1024, 2048, 512), (2500, 2300, 260)])
@pytest.mark.parametrize("block_a,block_b,fa,fb", [(128, 1, "e4m3", "e4m3"), (1, 1, "e5m2", "e4m3"), (128, 128, "e5m2", "e5m2"), (1, 128, "e4m3", "e5m2")])
@pytest.mark.parametrize("aligned", [True, False])
def test_scales_of_the_whole_range(gpu, m, n, k, block_a, block_b, fa, fb, aligned):
    """Scales from the smallest float to the largest on either side: wherever the terms' magnitudes fit a float, the product
    is as good as with ordinary scales, also where the two scales' own product is infinite or zero; zero codes give zero.

    The bound is the ordinary one, and for what lands among the subnormals 2^-149 for each addition and 2^-149 for a term
    that is rounded there."""
    if not aligned and m * n > 100000:
        pytest.skip("the plain kernel has no tiles of other sizes")
    rng = np.random.default_rng(m + n + k)

    def side(rows, block, fmt):
        codes, scales, _ = operand(rng, k, rows, block, fmt)
        codes[:, rng.integers(0, rows, rows // 8)] = 0
        e = EXPONENTS[rng.integers(0, len(EXPONENTS), scales.shape)]
        scales = np.ldexp(1 + rng.integers(0, 1 << 23, scales.shape) * 2.0 ** -23, e).astype(np.float32)
        ld = (k + 15) // 16 * 16 + (0 if aligned else 1)
        full = np.full((ld, rows), 0x7F, np.uint8)
        full[:k] = codes
        return codes, scales, ops.Blocks(Tensor.from_numpy(full, "uint8").slice(0, 0, k), Tensor.from_numpy(scales, "float"), fmt)

    ca, sa, a = side(m, block_a, fa)
    cb, sb, b = side(n, block_b, fb)
    want, mag = ref.block_gemm(ca, sa, block_a, fa, cb, sb, block_b, fb)
    c = got(ops.block_gemm(a, b, "float"))
    fits = mag < 2.0 ** 127
    assert np.any(fits)
    tol = 2.0 ** -24 * (128 + 8 + k / 128) * mag + 2.0 ** -149 * (2 * (k // 128) + 4)
    assert np.all(np.isfinite(c[fits])) and np.all(np.abs(c - want)[fits] <= tol[fits])


@pytest.mark.parametrize("m,n,k", [(300, 1, 1000), (129, 3, 256), (512, 17, 640), (640, 64, 1500), (384, 100, 256), (128, 128, 128), (130, 129, 130),
                                   (300, 520, 700), (1024, 2048, 512), (2500, 2300, 260)])
@pytest.mark.parametrize("block_a,block_b", [(128, 1), (1, 1), (128, 128), (1, 128)])
@pytest.mark.parametrize("aligned", [True, False])
def test_scales_that_cancel(gpu, m, n, k, block_a, block_b, aligned):
    """In each depth block one side's scales are as large as the other's are small, or both far from one: the results are
    ordinary numbers, with the ordinary bound.  A row of zeros meets scales whose product is infinite."""
    if not aligned and m * n > 100000:
        pytest.skip("the plain kernel has no tiles of other sizes")
    rng = np.random.default_rng(m + 2 * n + k)
    nb = (k + 127) // 128
    ea = EXPONENTS[rng.integers(0, len(EXPONENTS), nb)]
    eb = np.clip(rng.choice([-30, 0, 30], nb) - ea, -146, 124)

    def side(rows, block, e):
        codes, scales, _ = operand(rng, k, rows, block, "e5m2")
        codes[:, rng.integers(0, rows, rows // 8)] = 0
        scales = np.ldexp(1 + rng.integers(0, 1 << 23, scales.shape) * 2.0 ** -23, np.minimum(e[None] + rng.integers(-3, 3, scales.shape), 127)).astype(np.float32)
        scales[0, 0], codes[:128, :block] = 2.0 ** 127, 0    # a zero part under the largest scale
        ld = (k + 15) // 16 * 16 + (0 if aligned else 1)
        full = np.full((ld, rows), 0x7F, np.uint8)
        full[:k] = codes
        return codes, scales, ops.Blocks(Tensor.from_numpy(full, "uint8").slice(0, 0, k), Tensor.from_numpy(scales, "float"), "e5m2")

    ca, sa, a = side(m, block_a, ea)
    cb, sb, b = side(n, block_b, eb)
    want, mag = ref.block_gemm(ca, sa, block_a, "e5m2", cb, sb, block_b, "e5m2")
    assert np.all(mag < 2.0 ** 127)
    for dtype in ("float", "half"):
        c = got(ops.block_gemm(a, b, dtype))
        tol = 2.0 ** -24 * (128 + 8 + k / 128) * mag + 2.0 ** -149 * (2 * nb + 4)
        if dtype == "half":
            tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
            fits = np.abs(want) + tol < 65504
            assert np.all(np.isinf(c[np.abs(want) - tol > 65536]))
        else:
            fits = np.full(want.shape, True)
        assert np.all(np.abs(c - want)[fits] <= tol[fits])


@pytest.mark.parametrize("m,n,k", [(300, 200, 1000), (300, 200, 1001), (640, 3, 515), (1024, 600, 270)])
def test_turned_codes_reach_the_tensor_cores(gpu, m, n, k):
    """Codes that are contiguous along the rows' dimension are laid out again with rows on 16-byte boundaries, whatever the
    depth: the same bits as from codes that lay so from the start."""
    rng = np.random.default_rng(k)
    a, b = ops.block_quantize(upload(values(rng, k, m, "half"), "half"), 128), ops.block_quantize(upload(values(rng, k, n, "half"), "half"))
    turned = [ops.Blocks(ops.clone(q.codes.T).T, q.scales, q.format) for q in (a, b)]
    assert all(t.codes.strides[0] != 1 for t in turned)
    assert all(ops._blocks_view(t, "a")[1].ld % 16 == 0 for t in turned)
    assert np.array_equal(got(ops.block_gemm(*turned, "float")), got(ops.block_gemm(a, b, "float")))


@pytest.mark.parametrize("m,n,k", [(300, 1, 1000), (512, 17, 640), (130, 129, 130), (300, 520, 700), (1024, 2048, 512)])
@pytest.mark.parametrize("block_a,block_b", [(128, 1), (1, 1), (1, 128)])
@pytest.mark.parametrize("large", [False, True])
def test_small_scales(gpu, m, n, k, block_a, block_b, large):
    """One side's scales are those that a padded batch has beside ordinary ones (2^-126, and up to 2^-91), the other's at most
    one, but for a single large one: floats keep their bits where they are ordinary, halves are as near as with any scales.
    An infinite code keeps its infinity."""
    rng = np.random.default_rng(m + 3 * n + k)

    def side(rows, block, low, high):
        codes, scales, _ = operand(rng, k, rows, block, "e5m2")
        scales = np.ldexp(1 + rng.integers(0, 1 << 23, scales.shape) * 2.0 ** -23, rng.integers(low, high, scales.shape)).astype(np.float32)
        return codes, scales

    def blocks(codes, scales):                             # with padded rows: the plain kernel is not meant
        full = np.full(((k + 15) // 16 * 16, codes.shape[1]), 0x7F, np.uint8)
        full[:k] = codes
        return ops.Blocks(Tensor.from_numpy(full, "uint8").slice(0, 0, k), Tensor.from_numpy(scales, "float"), "e5m2")

    ca, sa = side(m, block_a, -20, 0)
    cb, sb = side(n, block_b, -126, -90)
    ordinary = rng.random(sb.shape) < 0.1
    sb[ordinary] = 2.0 ** -rng.integers(1, 9, ordinary.sum())
    sb[rng.random(sb.shape) < 0.3] = 2.0 ** -126
    if large:
        sa[-1, 0] = 2.0 ** 60
    want, mag = ref.block_gemm(ca, sa, block_a, "e5m2", cb, sb, block_b, "e5m2")
    a, b = blocks(ca, sa), blocks(cb, sb)
    tol = 2.0 ** -24 * (128 + 8 + k / 128) * mag + 2.0 ** -149 * (2 * (k // 128) + 4)
    assert np.all(np.abs(got(ops.block_gemm(a, b, "float")) - want) <= tol)
    c = got(ops.block_gemm(a, b, "half"))
    halves = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -100
    fits = np.abs(want) + halves < 65504
    assert np.all(np.abs(c - want)[fits] <= halves[fits])

    ca[5, 0], cb[5] = 0x7C, 0x3C                           # infinity times one in every column, whatever the scales
    sb[:, 0] = 2.0 ** -126
    a, b = blocks(ca, sa), blocks(cb, sb)
    others, mag = ref.block_gemm(np.where(ca == 0x7C, 0, ca), sa, block_a, "e5m2", cb, sb, block_b, "e5m2")
    for dtype in ("half", "float"):
        c = got(ops.block_gemm(a, b, dtype))
        fits = (np.abs(others) + 2.0 ** -24 * (128 + 8 + k / 128) * mag < 65504) | (dtype == "float")
        assert np.all(c[0] == np.inf) and np.all(np.isfinite(c[1:][fits[1:]]))


@pytest.mark.parametrize("dtype", ["half", "float"])
def test_padded_batch(gpu, dtype):
    """A batch whose last tokens are zeros: their products are zeros, the others' and the weights' gradient are those of the
    batch without them, to the last bit."""
    rng = np.random.default_rng(7)
    k, m, used, n = 520, 700, 384, 768
    w, x, dy = values(rng, k, m, "half"), values(rng, k, n, "half"), values(rng, m, n, "half")
    x[:, used:], dy[:, used:] = 0, 0

    def layer(tokens):
        tx, ty = upload(x[:, :tokens], "half"), upload(dy[:, :tokens], "half")
        y = ops.block_gemm(ops.block_quantize(upload(w, "half"), 128), ops.block_quantize(tx), dtype)
        return got(y), got(ops.block_gemm(ops.block_quantize(tx.T), ops.block_quantize(ty.T), dtype))

    y, dw = layer(n)
    y0, dw0 = layer(used)
    assert np.all(y[:, used:] == 0) and np.array_equal(y[:, :used], y0)
    assert np.array_equal(dw, dw0)
