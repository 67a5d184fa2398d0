"""Operands and results of different types in the 8-bit linear layer: what is refused, before any CUDA call."""
import pytest

import torch

from solid_b200 import Tensor, ops


def host(size, dtype):
    return Tensor(torch.zeros(1 << 16, dtype=torch.uint8), dtype, size)


@pytest.mark.parametrize("wide", ["float", "double"])
@pytest.mark.parametrize("narrow", ["half", "chalf"])
def test_a_result_with_more_bits_than_its_tensor(wide, narrow):
    """A float or double result would be flushed and rounded away from zero on its way into halves."""
    x, out = host([4, 3], "half"), host([4, 3], narrow)
    with pytest.raises(TypeError, match="the norm is of type %s" % wide):
        ops.rms_norm(host([4, 3], wide), dst=out)
    with pytest.raises(TypeError, match="the norm is of type %s" % wide):
        ops.rms_norm(x, host([4], wide), dst=out)
    with pytest.raises(TypeError, match="the sum is of type %s" % wide):
        ops.rms_norm(x, None, 1e-6, host([4, 3], wide), h=out)
    with pytest.raises(TypeError, match="the sum is of type %s" % wide):
        ops.rms_norm_quantize(x, host([4], wide), 1e-6, x, h=out)
    with pytest.raises(TypeError, match="the gradient is of type %s" % wide):
        ops.rms_norm_grad(host([4, 3], wide), x, dst=out)
    with pytest.raises(TypeError, match="the gradient is of type %s" % wide):
        ops.rms_norm_grad(x, x, dres=host([4, 3], wide), dst=out)


@pytest.mark.parametrize("other", ["cfloat", "chalf", "cdouble"])
def test_complex_operands(other):
    x = host([4, 3], "half")
    for call in (lambda: ops.rms_norm(x, host([4], other)), lambda: ops.rms_norm(x, residual=host([4, 3], other)),
                 lambda: ops.rms_norm_quantize(x, residual=host([4, 3], other)), lambda: ops.rms_norm_grad(host([4, 3], other), x)):
        with pytest.raises(TypeError, match="not available for type c"):
            call()


def test_a_float_product_into_complex_halves():
    codes = ops.Blocks(host([256, 4], "uint8"), host([4, 2], "float"))
    with pytest.raises(TypeError, match="the product is of type float"):
        ops.block_gemm(codes, codes, "float", dst=host([4, 4], "chalf"))
