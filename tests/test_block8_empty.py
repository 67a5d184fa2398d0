"""Matrices without elements in the 8-bit linear layer: allocators give no address for them, and none is needed."""
import ctypes as C

import numpy as np
import pytest

from solid_b200 import Tensor, _lib, ops
from solid_b200._lib import BlocksView, Matrix


def test_no_address_no_call():
    """Nothing to do: no device is needed either."""
    lib = _lib.get()
    m, v, v128 = C.byref(Matrix(None, 2, 2)), C.byref(BlocksView(None, 16, None, 4, 4, 1, 0)), C.byref(BlocksView(None, 16, None, 4, 4, 128, 0))
    for n, rows in ((0, 4), (4, 0), (0, 0)):
        lib.rms_norm("half", n, rows, m, m, None, 1e-6, m, m)
        lib.rms_norm_quantize("half", n, rows, m, None, None, 1e-6, None, v)
        lib.block_quantize("half", n, rows, m, v)
        lib.block_quantize("half", n, rows, m, v128)
    lib.rms_norm_grad("half", 0, 4, m, m, None, 1e-6, None, m, None, None)
    lib.block_gemm("half", 0, 4, 4, v, C.byref(BlocksView(1 << 20, 16, 1 << 20, 4, 4, 1, 0)), m)
    lib.block_gemm("half", 4, 0, 4, C.byref(BlocksView(1 << 20, 16, 1 << 20, 4, 4, 1, 0)), v, m)


@pytest.mark.gpu
def test_tensors_of_no_bytes(gpu):
    """Tensors over storages of no bytes, as a batch without tokens comes from torch."""
    import torch

    def none(size, dtype):
        return Tensor(torch.empty(0, dtype=torch.uint8, device="cuda"), dtype, size)

    w = Tensor.from_numpy(np.ones(256, np.float16), "half")
    y, h = ops.rms_norm(none([256, 0], "half"), w, 1e-6, none([256, 0], "half"))
    assert y.size == [256, 0] and h.size == [256, 0]
    q, h = ops.rms_norm_quantize(none([256, 0], "half"), w, 1e-6, none([256, 0], "half"))
    assert q.codes.size == [256, 0] and q.scales.size == [0, 2]
    dh, dw = ops.rms_norm_grad(none([256, 0], "half"), none([256, 0], "half"), w)
    assert dh.size == [256, 0] and np.array_equal(dw.numpy(), np.zeros(256, np.float32))
    for block in (1, 128):
        q = ops.block_quantize(none([256, 0], "float"), block)
        assert q.codes.size == [256, 0] and q.scales.size == [0, 2]
    eight = ops.block_quantize(Tensor.from_numpy(np.ones((256, 8), np.float32), "float"))
    tokens = ops.Blocks(none([256, 0], "uint8"), none([0, 2], "float"))
    assert ops.block_gemm(eight, tokens).size == [8, 0]
    assert ops.block_gemm(tokens, eight, dst=none([0, 8], "float")).size == [0, 8]
    deep = ops.Blocks(none([0, 3], "uint8"), none([3, 0], "float"))
    assert np.array_equal(ops.block_gemm(deep, deep, "float").numpy(), np.zeros((3, 3), np.float32))
