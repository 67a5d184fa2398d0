"""What the entry points of the 8-bit linear layer refuse, before any CUDA call: no device needed."""
import ctypes as C

import pytest

from solid_b200 import _lib
from solid_b200._lib import BlocksView, Matrix, SolidError

P = 1 << 20                                              # an address: nothing here gets as far as reading it


def matrix(ptr=P, s0=4, s1=64):
    return C.byref(Matrix(ptr, s0, s1))


def view(codes=P, ld=128, scales=P, ss0=4, ss1=64, block=1, fmt=0):
    return C.byref(BlocksView(codes, ld, scales, ss0, ss1, block, fmt))


def test_types():
    lib = _lib.get()
    for dtype in ("int32", "uint8", "chalf", "cfloat", "bool"):
        with pytest.raises(SolidError, match="half, float or double"):
            lib.rms_norm(dtype, 16, 4, matrix(), None, None, 1e-6, None, matrix())
        with pytest.raises(SolidError, match="half, float or double"):
            lib.rms_norm_grad(dtype, 16, 4, matrix(), matrix(), None, 1e-6, None, matrix(), None, P)
        with pytest.raises(SolidError, match="half, float or double"):
            lib.block_quantize(dtype, 16, 4, matrix(), view())
    for dtype in ("double", "int8", "uint8"):
        with pytest.raises(SolidError, match="half or float"):
            lib.block_gemm(dtype, 4, 4, 4, view(), view(), matrix())


def test_missing_and_misaligned_matrices():
    lib = _lib.get()
    with pytest.raises(SolidError, match="missing matrix x"):
        lib.rms_norm("float", 16, 4, None, None, None, 1e-6, None, matrix())
    with pytest.raises(SolidError, match="missing matrix y"):
        lib.rms_norm("float", 16, 4, matrix(), None, None, 1e-6, None, matrix(ptr=None))
    with pytest.raises(SolidError, match="residual must be aligned"):
        lib.rms_norm("float", 16, 4, matrix(), matrix(ptr=P + 2), None, 1e-6, None, matrix())
    with pytest.raises(SolidError, match="x must be aligned"):
        lib.rms_norm("float", 16, 4, matrix(s1=66), None, None, 1e-6, None, matrix())
    with pytest.raises(SolidError, match="weights must be aligned"):
        lib.rms_norm("float", 16, 4, matrix(), None, P + 1, 1e-6, None, matrix())
    with pytest.raises(SolidError, match="missing scratch buffer"):
        lib.rms_norm_grad("float", 16, 4, matrix(), matrix(), None, 1e-6, None, matrix(), P, None)
    with pytest.raises(SolidError, match="dweight and buffer must be aligned"):
        lib.rms_norm_grad("half", 16, 4, matrix(), matrix(), None, 1e-6, None, matrix(), P + 2, P)
    with pytest.raises(SolidError, match="missing matrix c"):
        lib.block_gemm("float", 4, 4, 4, view(), view(), None)
    with pytest.raises(SolidError, match="c must be aligned"):
        lib.block_gemm("float", 4, 4, 4, view(), view(), matrix(ptr=P + 2))


@pytest.mark.parametrize("eps", [-1e-6, float("nan")])
def test_eps(eps):
    with pytest.raises(SolidError, match="eps"):
        _lib.get().rms_norm("float", 16, 4, matrix(), None, None, eps, None, matrix())


def test_codes_and_scales():
    lib = _lib.get()
    for bad, text in ((dict(codes=None), "missing codes"), (dict(scales=None), "missing codes or scales"), (dict(fmt=2), "8-bit format"),
                      (dict(block=64), "1 or 128 rows"), (dict(scales=P + 2), "scales of .* must be aligned"),
                      (dict(ss1=6), "scales of .* must be aligned")):
        for call in (lambda: lib.block_quantize("half", 16, 4, matrix(), view(**bad)),
                     lambda: lib.block_gemm("half", 4, 4, 4, view(), view(**bad), matrix()),
                     lambda: lib.block_gemm("half", 4, 4, 4, view(**bad), view(), matrix()),
                     lambda: lib.rms_norm_quantize("half", 16, 4, matrix(), None, None, 1e-6, None, view(**bad))):
            with pytest.raises(SolidError, match=text):
                call()
    with pytest.raises(SolidError, match="block 1"):
        lib.rms_norm_quantize("half", 16, 4, matrix(), None, None, 1e-6, None, view(block=128))


def test_sizes():
    lib = _lib.get()
    with pytest.raises(SolidError, match="too large"):
        lib.rms_norm("half", 1 << 41, 4, matrix(), None, None, 1e-6, None, matrix())
    with pytest.raises(SolidError, match="too large"):
        lib.block_quantize("half", 1 << 39, 1 << 39, matrix(), view())
    with pytest.raises(SolidError, match="too large"):
        lib.block_gemm("half", 4, 4, 1 << 41, view(), view(), matrix())


def test_nothing_to_do():
    """No element: no launch, whatever the addresses."""
    lib = _lib.get()
    lib.rms_norm("half", 0, 4, matrix(), None, None, 1e-6, None, matrix())
    lib.rms_norm("half", 4, 0, matrix(), None, None, 1e-6, None, matrix())
    lib.block_quantize("half", 4, 0, matrix(), view())
    lib.block_gemm("half", 0, 4, 4, view(), view(), matrix())


def test_python_layer():
    import torch
    from solid_b200 import Tensor, ops

    def host(size, dtype, device="cpu"):
        return Tensor(torch.zeros(1 << 16, dtype=torch.uint8), dtype, size)

    with pytest.raises(TypeError, match="not available"):
        ops.rms_norm(host([4, 4], "int32"))
    with pytest.raises(ValueError, match="at least one dimension"):
        ops.rms_norm(host([], "half"))
    with pytest.raises(ValueError, match=r"size \[4\]"):
        ops.rms_norm(host([4, 4], "half"), host([5], "half"))
    with pytest.raises(ValueError, match="no residual"):
        ops.rms_norm(host([4, 4], "half"), h=host([4, 4], "half"))
    with pytest.raises(ValueError, match="size of h"):
        ops.rms_norm_grad(host([4, 3], "half"), host([4, 4], "half"))
    with pytest.raises(ValueError, match="8-bit format"):
        ops.rms_norm_quantize(host([4, 4], "half"), format="e3m4")
    with pytest.raises(ValueError, match="1 or 128 rows"):
        ops.block_quantize(host([4, 4], "half"), 64)
    good = ops.Blocks(host([256, 130], "uint8"), host([130, 2], "float"))
    with pytest.raises(TypeError, match="half or float"):
        ops.block_gemm(good, good, "double")
    with pytest.raises(ValueError, match="do not belong"):
        ops.block_gemm(good, ops.Blocks(host([256, 130], "uint8"), host([3, 2], "float")))
    with pytest.raises(ValueError, match="depths"):
        ops.block_gemm(good, ops.Blocks(host([255, 130], "uint8"), host([2, 2], "float")))
    with pytest.raises(TypeError, match="codes are uint8"):
        ops.block_gemm(good, ops.Blocks(host([256, 130], "int8"), host([2, 2], "float")))
    with pytest.raises(ValueError, match="the result has size"):
        ops.block_gemm(good, good, dst=host([130, 129], "half"))
