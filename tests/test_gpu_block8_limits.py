"""The 8-bit linear layer at the ends of what it accepts: places that a caller's own allocator gives, numbers near the ends
of their type's range."""
import numpy as np
import pytest

import block8_ref as ref
from solid_b200 import Tensor, ops
from solid_b200._lib import Matrix
from test_gpu_block8 import ACC, EPS, STEP, got, roundings, upload, values

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
