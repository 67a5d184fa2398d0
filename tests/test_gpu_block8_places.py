"""Where the 8-bit linear layer's C functions read and write: places that a caller's own allocator gives."""
import numpy as np
import pytest

from solid_b200 import Tensor, ops
from solid_b200._lib import Matrix
from test_gpu_block8 import EPS, got, upload, values

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
