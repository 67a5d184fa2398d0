"""Operands of different types in the 8-bit linear layer: they meet in their common type, nothing is narrowed on the way.
Numbers are compared with 64-bit evaluations of the values that the tensors hold; the bounds are those of one type, with
the common type in its place, since widening is exact."""
import numpy as np
import pytest

import block8_ref as ref
from solid_b200 import Tensor, ops
from test_gpu_block8 import ACC, EPS, STEP, TINY, check_blocks, got, norm_bounds, roundings, upload, values

pytestmark = pytest.mark.gpu

ORDER = ["half", "float", "double"]


def widest(*types):
    return max((t for t in types if t), key=ORDER.index)


@pytest.mark.parametrize("n,rows", [(64, 5), (1000, 7), (4096, 3)])
@pytest.mark.parametrize("tx,tr,tw", [("half", "float", "half"), ("half", "float", "float"), ("float", "half", "half"), ("half", None, "float"),
                                      ("half", "half", "double"), ("double", "half", "float"), ("float", "float", "half")])
def test_norm(gpu, tx, tr, tw, n, rows):
    rng = np.random.default_rng(n)
    x = values(rng, n, rows, tx)
    r = values(rng, n, rows, tr) if tr else None
    w = values(rng, n, 1, tw)[:, 0]
    x[:, 0] *= x.dtype.type(2.0 ** -12)                      # subnormal halves among them
    w[0] = w.dtype.type(3e-6)
    if tr:
        r[:, 0] *= r.dtype.type(2.0 ** -12)
        if tr != "half":
            r[3, 1] = 1e6                                    # beyond the range of halves
    t = widest(tx, tr, tw)
    hx = x.astype(np.float64) + (r.astype(np.float64) if tr else 0)
    want = ref.rms_norm(hx, w, EPS)
    tensors = upload(x, tx), upload(w, tw), EPS, upload(r, tr) if tr else None
    out = ops.rms_norm(*tensors)
    y, h = out if tr else (out, None)
    assert y.dtype == t and np.all(np.abs(got(y) - want) <= norm_bounds(t, n, want))
    if tr:
        assert h.dtype == t and np.all(np.abs(got(h) - hx) <= (STEP[t] + ACC[t]) * np.abs(hx) + TINY[t])
    out = ops.rms_norm_quantize(*tensors)
    q, h = out if tr else (out, None)
    check_blocks(q, want, 1, "e4m3", 2.0 ** -24 * (roundings(n) / 2 + 12))
    if tr:
        assert h.dtype == t and np.all(np.abs(got(h) - hx) <= (STEP[t] + ACC[t]) * np.abs(hx) + TINY[t])


@pytest.mark.parametrize("size", [2e-5, 1e-7])
@pytest.mark.parametrize("n,rows", [(64, 5), (1000, 30), (4096, 3)])
@pytest.mark.parametrize("tg,th,tw,tr", [("float", "half", "half", None), ("float", "half", "half", "half"), ("half", "float", "half", None),
                                         ("half", "half", "float", "float"), ("double", "half", "float", "half")])
def test_gradient(gpu, tg, th, tw, tr, n, rows, size):
    """Gradients below the smallest normal half, beside a norm of ordinary numbers."""
    rng = np.random.default_rng(n + rows)
    h, w = values(rng, n, rows, th), values(rng, n, 1, tw)[:, 0]
    dy = (rng.standard_normal((n, rows)) * size).astype(values(rng, 1, 1, tg).dtype)
    res = (rng.standard_normal((n, rows)) * size).astype(values(rng, 1, 1, tr).dtype) if tr else None
    t = widest(tg, th, tw, tr)
    dh, dw = ops.rms_norm_grad(upload(dy, tg), upload(h, th), upload(w, tw), EPS, upload(res, tr) if tr else None)
    want, wantw, mag, magw = ref.rms_norm_grad(dy, h, w, EPS, res)
    assert dh.dtype == t and dw.dtype == ("double" if t == "double" else "float")
    assert np.any(wantw) and np.any(dw.numpy())
    assert np.all(np.abs(got(dh) - want) <= STEP[t] * np.abs(want) + TINY[t] + ACC[t] * (2 * roundings(n) + 16) * mag)
    assert np.all(np.abs(dw.numpy() - wantw) <= ACC[t] * (roundings(n) / 2 + rows + 16) * magw)


def test_from_the_product_into_the_gradient(gpu):
    """A product in 32 bits goes into the gradient as it is: the same numbers as from a float h."""
    rng = np.random.default_rng(2)
    n, m, rows = 256, 384, 40
    w, dy, h = (values(rng, *s, "half") for s in ((n, m), (m, rows), (n, rows)))
    dx = ops.block_gemm(ops.block_quantize(upload(w, "half").T, 128), ops.block_quantize(upload((dy * np.float16(1e-3)), "half")), "float")
    a, b = ops.rms_norm_grad(dx, upload(h, "half")), ops.rms_norm_grad(dx, upload(h.astype(np.float32), "float"))
    assert [np.array_equal(p.numpy(), q.numpy()) for p, q in zip(a, b)] == [True, True]


@pytest.mark.parametrize("dtype", ["half", "float", "double"])
def test_byte_swapped_and_unaligned(gpu, dtype):
    """Bytes in the other order and elements off their own boundaries, small numbers among them: what the plain ones give."""
    import torch
    rng = np.random.default_rng(8)
    n, rows = 264, 9
    x, r, w = values(rng, n, rows, dtype), values(rng, n, rows, dtype), values(rng, n, 1, dtype)[:, 0]
    x[:, 2] *= x.dtype.type(2.0 ** -15)
    r[:, 2] *= r.dtype.type(2.0 ** -15)

    def swapped(a):
        return ops.byteswap(upload(a, dtype))

    def unaligned(a):
        raw = torch.from_numpy(np.concatenate([np.zeros(1, np.uint8), np.asfortranarray(a).reshape(-1, order="F").view(np.uint8)])).cuda()
        return Tensor(raw, dtype, a.shape, None, 1)

    def all_of(form):
        y, h = ops.rms_norm(form(x), form(w), EPS, form(r))
        q, h8 = ops.rms_norm_quantize(form(x), form(w), EPS, form(r))
        dh, dw = ops.rms_norm_grad(form(r), form(x), form(w), EPS, form(r))
        c = ops.block_quantize(form(x), 128)
        return [t.numpy().tobytes() for t in (y, h, q.codes, q.scales, h8, dh, dw, c.codes, c.scales)]

    plain = all_of(lambda a: upload(a, dtype))
    assert all_of(swapped) == plain
    assert all_of(unaligned) == plain


@pytest.mark.parametrize("dtype,into", [("half", "float"), ("half", "double"), ("float", "double")])
def test_into_a_tensor_of_more_bits(gpu, dtype, into):
    rng = np.random.default_rng(4)
    n, rows = 100, 6
    x, r = values(rng, n, rows, dtype), values(rng, n, rows, dtype)
    y, h = ops.rms_norm(upload(x, dtype), None, EPS, upload(r, dtype))
    wide, wideh = Tensor.empty([n, rows], into), Tensor.empty([n, rows], into)
    a, b = ops.rms_norm(upload(x, dtype), None, EPS, upload(r, dtype), dst=wide, h=wideh)
    assert a is wide and b is wideh
    assert np.array_equal(got(a), got(y).astype(got(a).dtype)) and np.array_equal(got(b), got(h).astype(got(b).dtype))


@pytest.mark.parametrize("m,n,k", [(7, 3, 40), (300, 200, 512), (640, 40, 1000)])
@pytest.mark.parametrize("size", [1.0, 300.0, 2.0 ** -22])
def test_product_follows_its_result(gpu, m, n, k, size):
    """Without a type, dst says how many bits are kept; halves are rounded to nearest even from the 32-bit sums, subnormals
    among them (size 2^-22), numbers above 65504 stay finite in a float or double (size 300)."""
    rng = np.random.default_rng(m)
    a = ops.block_quantize(upload((values(rng, k, m, "float") * np.float32(size)), "float"), 128)
    b = ops.block_quantize(upload((values(rng, k, n, "float") * np.float32(size if size > 1 else 1)), "float"))
    c32 = ops.block_gemm(a, b, "float").numpy()
    with np.errstate(over="ignore"):
        c16 = c32.astype(np.float16)                         # numpy rounds to nearest even with subnormals
    if size > 1:
        assert np.any(np.abs(c32) > 65504)
    if size < 1:
        assert np.any((np.abs(c32) < 2.0 ** -15) & (c16 != 0))
    for into, dtype, want in (("float", None, c32), ("double", None, c32), ("float", "float", c32), ("double", "float", c32),
                              ("half", None, c16), ("half", "half", c16), ("half", "float", c16), ("float", "half", c16)):
        full = Tensor.from_numpy(np.full((m + 1, n), 7, {"half": np.float16, "float": np.float32, "double": np.float64}[into]), into)
        for dst in (Tensor.empty([m, n], into), Tensor.empty([n, m], into).T, full.slice(0, 1, m + 1)):
            c = ops.block_gemm(a, b, dtype, dst=dst)
            assert c is dst and np.array_equal(got(c), want.astype(got(c).dtype))
        assert np.all(got(full)[0] == 7)
    out = Tensor(Tensor.empty([m, n], "half").storage, "half", [m, n], None, 0, True)
    assert np.array_equal(got(ops.block_gemm(a, b, "float", dst=out)), c16)      # bytes in the other order
    assert ops.block_gemm(a, b).dtype == "half" and np.array_equal(got(ops.block_gemm(a, b)), c16)
