"""The 8-bit linear layer as it is used: norm, conversion, product and their gradients in a row; captured and replayed;
on several streams; at far addresses; inside larger tensors.  Numbers are checked against 64-bit evaluations with bounds
that count half a step of every conversion."""
import numpy as np
import pytest

import block8_ref as ref
from solid_b200 import Tensor, ops

pytestmark = pytest.mark.gpu

EPS = 1e-6


def got(t):
    a = t.numpy()
    return a.view(np.float16) if t.dtype == "half" else a


def half(rng, *size, scale=1.0):
    return (rng.standard_normal(size) * scale).astype(np.float16)


def conversion_error(x, block):
    """What e4m3 codes may be off by: half a step, 2^-4 of a normal code and 2^-10 of the scale below those; and 2^-20 for
    the scale and the quotient, which are rounded in 32 bits."""
    s = ref.spread(ref.scales(x, block, "e4m3"), *x.shape, block)
    return np.abs(x) * (2.0 ** -4 + 2.0 ** -20) + s * 2.0 ** -10


def product_error(a, ea, b, eb):
    return ea.T @ np.abs(b) + np.abs(a).T @ eb + ea.T @ eb


def layer(x, r, g, w, dy, dres):
    q, h = ops.rms_norm_quantize(x, g, EPS, r)
    y = ops.block_gemm(ops.block_quantize(w, 128), q, "float")
    xn = ops.rms_norm(h, g, EPS)
    dx = ops.block_gemm(ops.block_quantize(w.T, 128), ops.block_quantize(dy))
    dw = ops.block_gemm(ops.block_quantize(xn.T), ops.block_quantize(dy.T), "float")
    dh, dg = ops.rms_norm_grad(dx, h, g, EPS, dres)
    return y, h, dw, dx, dh, dg


def inputs(rng, k, m, tokens):
    arrays = (half(rng, k, tokens), half(rng, k, tokens), (1 + half(rng, k, scale=0.1)).astype(np.float16),
              half(rng, k, m, scale=k ** -0.5), half(rng, m, tokens, scale=0.1), half(rng, k, tokens, scale=0.1))
    return arrays, [Tensor.from_numpy(a, "half") for a in arrays]


@pytest.mark.parametrize("k,m,tokens", [(256, 384, 1), (512, 640, 33), (1000, 300, 200), (1536, 1024, 700)])
def test_layer_and_its_gradients(gpu, k, m, tokens):
    rng = np.random.default_rng(k + tokens)
    (x, r, g, w, dy, dres), tensors = inputs(rng, k, m, tokens)
    y, h, dw, dx, dh, dg = layer(*tensors)
    x, r, w, dy, dres = (a.astype(np.float64) for a in (x, r, w, dy, dres))
    hx = x + r
    xn = ref.rms_norm(hx, g, EPS)
    small = 2.0 ** -15                                       # sums in 32 bits, and the norm of h rounded to half (2^-11 each of two)
    ew, en, ed = conversion_error(w, 128), conversion_error(xn, 1), conversion_error(dy, 1)
    assert np.all(np.abs(got(y) - w.T @ xn) <= product_error(w, ew, xn, en) * (1 + small) + small * (np.abs(w).T @ np.abs(xn)))
    wt = np.ascontiguousarray(w.T)
    want = wt.T @ dy
    assert np.all(np.abs(got(dx) - want) <= (product_error(wt, conversion_error(wt, 128), dy, ed) + 2.0 ** -11 * np.abs(want)) * (1 + small) +
                  small * (np.abs(wt).T @ np.abs(dy)) + 2.0 ** -25)
    # xn is rounded to half, from an h that was rounded to half
    nt, dt_ = np.ascontiguousarray(xn.T), np.ascontiguousarray(dy.T)
    en = conversion_error(nt, 1) * (1 + 2.0 ** -9) + np.abs(nt) * 2.0 ** -9
    assert dw.size == [k, m]
    assert np.all(np.abs(got(dw) - nt.T @ dt_) <= product_error(nt, en, dt_, conversion_error(dt_, 1)) * (1 + small) +
                  small * (np.abs(nt).T @ np.abs(dt_)))
    # the norm's gradient at the stored h, from the stored dx
    want, wantg, mag, magg = ref.rms_norm_grad(got(dx), got(h), g, EPS, dres)
    assert np.all(np.abs(got(dh) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -16 * mag)
    assert np.all(np.abs(got(dg) - wantg) <= 2.0 ** -16 * magg)


def test_norm_gradient_against_differences(gpu):
    """Central differences of the norm itself, in double: a step of 1e-4 leaves a third-order term of about 1e-8 and a
    rounding of 2^-53 / 1e-4 = 1e-12 of the sum's magnitude."""
    rng = np.random.default_rng(3)
    n, rows, step = 40, 3, 1e-4
    h, dy, w = rng.standard_normal((n, rows)), rng.standard_normal((n, rows)), 1 + 0.1 * rng.standard_normal(n)

    def loss(h, w):
        return float((dy * ops.rms_norm(Tensor.from_numpy(h), Tensor.from_numpy(w), EPS).numpy()).sum())

    dh, dw = ops.rms_norm_grad(Tensor.from_numpy(dy), Tensor.from_numpy(h), Tensor.from_numpy(w), EPS)
    dh, dw = dh.numpy(), dw.numpy()
    for i, row in [(0, 0), (7, 1), (39, 2), (20, 0)]:
        up, down = h.copy(), h.copy()
        up[i, row] += step; down[i, row] -= step
        assert abs((loss(up, w) - loss(down, w)) / (2 * step) - dh[i, row]) <= 1e-6
        up, down = w.copy(), w.copy()
        up[i] += step; down[i] -= step
        assert abs((loss(h, up) - loss(h, down)) / (2 * step) - dw[i]) <= 1e-6


def test_same_bits_every_time(gpu):
    rng = np.random.default_rng(4)
    for k, m, tokens in ((4096, 512, 1), (2048, 768, 48), (1024, 600, 300)):
        _, tensors = inputs(rng, k, m, tokens)
        first = [got(t).tobytes() for t in layer(*tensors)]
        for _ in range(3):
            assert [got(t).tobytes() for t in layer(*tensors)] == first


def test_captured_and_replayed_on_two_streams(gpu):
    """Two graphs of the whole layer replayed side by side, with new inputs in the same places: what the calls give."""
    import torch
    rng = np.random.default_rng(6)
    sizes = (1024, 512, 40), (1000, 300, 600)
    held = [inputs(rng, *s)[1] for s in sizes]
    graphs, outs = [], []
    for tensors in held:
        layer(*tensors)                                      # outside first, as capture asks
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(*tensors))
        graphs.append(g)
    for again in range(3):
        for s, tensors in zip(sizes, held):
            for t, new in zip(tensors, inputs(rng, *s)[1]):
                t.storage.copy_(new.storage)
        want = [[got(t).tobytes() for t in layer(*tensors)] for tensors in held]
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert [[got(t).tobytes() for t in o] for o in outs] == want


def test_streams_at_once(gpu):
    import torch
    rng = np.random.default_rng(8)
    held = [inputs(rng, 1536, 640, 100 + i)[1] for i in range(3)]
    want = [[got(t).tobytes() for t in layer(*tensors)] for tensors in held]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in held], []
    for _ in range(5):
        for tensors, s in zip(held, streams):
            with torch.cuda.stream(s):
                outs.append(layer(*tensors))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert [got(t).tobytes() for t in o] == want[i % 3]


@pytest.mark.parametrize("m,n,k", [(260, 300, 384), (512, 700, 300), (640, 9, 512), (200, 64, 256)])
@pytest.mark.parametrize("dtype", ["half", "float"])
@pytest.mark.parametrize("turned", [False, True])
def test_product_inside_a_larger_tensor(gpu, m, n, k, dtype, turned):
    """What lies around the result stays, whole lines or not."""
    rng = np.random.default_rng(m)
    a, b = half(rng, k, m), half(rng, k, n)
    qa, qb = ops.block_quantize(Tensor.from_numpy(a, "half"), 128), ops.block_quantize(Tensor.from_numpy(b, "half"))
    want = got(ops.block_gemm(qa, qb, dtype))
    for before, after in ((8, 8), (3, 2)):
        rows, cols = before + (n if turned else m) + after, 2 + (m if turned else n) + 1
        full = Tensor.from_numpy(np.full((rows, cols), 5, np.float16 if dtype == "half" else np.float32), dtype)
        inner = full.slice(0, before, rows - after).slice(1, 2, cols - 1)
        c = ops.block_gemm(qa, qb, dtype, dst=inner.T if turned else inner)
        assert np.array_equal(got(c), want)
        around = got(full).copy()
        around[before:rows - after, 2:cols - 1] = 5
        assert np.all(around == 5)


def test_far_rows(gpu):
    """Rows more than 4 GB apart."""
    import torch
    rng = np.random.default_rng(9)
    far = (1 << 32) + 4096
    room = torch.zeros(far + (1 << 16), dtype=torch.uint8, device="cuda")
    n = 1024
    x = half(rng, n, 2)
    t = Tensor(room, "half", [n, 2], [2, far], 256)
    ops.copy(Tensor.from_numpy(x, "half"), t)
    near = Tensor.from_numpy(x, "half")
    assert np.array_equal(got(ops.rms_norm(t)), got(ops.rms_norm(near)))
    for f in (lambda v: ops.block_quantize(v), lambda v: ops.block_quantize(v, 128), lambda v: ops.block_quantize(v.T)):
        p, q = f(t), f(near)
        assert np.array_equal(p.codes.numpy(), q.codes.numpy()) and np.array_equal(p.scales.numpy(), q.scales.numpy())
    y = ops.rms_norm(near, dst=t)
    assert np.array_equal(got(y), got(ops.rms_norm(near)))
    dh, dw = ops.rms_norm_grad(t, t)
    eh, ew = ops.rms_norm_grad(ops.clone(t), ops.clone(t))
    assert np.array_equal(got(dh), got(eh)) and np.array_equal(dw.numpy(), ew.numpy())
    q = ops.block_quantize(near)
    codes = Tensor(room, "uint8", [n, 2], [1, far], 4096)
    ops.copy(q.codes, codes)
    b = ops.block_quantize(Tensor.from_numpy(half(rng, n, 70), "half"))
    assert np.array_equal(got(ops.block_gemm(ops.Blocks(codes, q.scales), b)), got(ops.block_gemm(q, b)))


def test_operands_of_any_strides(gpu):
    """Scales with the blocks' index running fastest, rows in reverse order, a residual that is the same for all rows,
    weights with gaps: what plain copies of them give."""
    rng = np.random.default_rng(12)
    n, rows, m = 520, 70, 200
    x, w = half(rng, n, rows), half(rng, n, m)
    tx = Tensor.from_numpy(x, "half")
    back = tx.slice(1, rows - 1, -1, -1)
    assert back.size == [n, rows] and np.array_equal(got(back), x[:, ::-1])
    one = Tensor.from_numpy(half(rng, n, 1), "half")
    gaps = Tensor.from_numpy(half(rng, 2 * n), "half").slice(0, 0, 2 * n, 2)
    y, h = ops.rms_norm(back, gaps, EPS, one)
    want, wanth = ops.rms_norm(ops.clone(back), ops.clone(gaps), EPS, ops.clone(one.broadcast_to([n, rows])))
    assert np.array_equal(got(y), got(want)) and np.array_equal(got(h), got(wanth))
    q, qb = ops.block_quantize(ops.clone(back)), ops.block_quantize(back)
    assert np.array_equal(q.codes.numpy(), qb.codes.numpy()) and np.array_equal(q.scales.numpy(), qb.scales.numpy())
    qw = ops.block_quantize(Tensor.from_numpy(w, "half"), 128)
    c = got(ops.block_gemm(qw, q))
    turned = ops.Blocks(q.codes, ops.clone(q.scales.T).T, q.format)
    assert turned.scales.strides != q.scales.strides
    assert np.array_equal(got(ops.block_gemm(qw, turned)), c)
    # rows of the codes in reverse order: no tensor map takes them, the plain kernel does (other order of the same sums)
    codes = ops.clone(q.codes)
    reverse = ops.Blocks(codes.slice(1, rows - 1, -1, -1), q.scales.slice(0, rows - 1, -1, -1), q.format)
    a, b = (ref.decode(t.codes.numpy(), "e4m3") * ref.spread(t.scales.numpy().astype(np.float64), *t.codes.size, k) for t, k in ((qw, 128), (q, 1)))
    assert np.all(np.abs(got(ops.block_gemm(qw, reverse))[:, ::-1] - a.T @ b) <= 2.0 ** -24 * 136 * (np.abs(a).T @ np.abs(b)) + 2.0 ** -11 * np.abs(a.T @ b) + 2.0 ** -25)


@pytest.mark.parametrize("tokens", [1, 40, 200, 600])
def test_what_is_not_finite_stays_in_its_row(gpu, tokens):
    """A token with an infinity and one with a NaN: their results are NaN, all others what they are without them; results
    beyond the range of halves are infinite."""
    rng = np.random.default_rng(tokens)
    k, m = 512, 640
    x, w = half(rng, k, tokens), half(rng, k, m)
    qw = ops.block_quantize(Tensor.from_numpy(w, "half"), 128)
    clean = got(ops.block_gemm(qw, ops.block_quantize(Tensor.from_numpy(x, "half")), "float"))
    bad = sorted({0, tokens - 1})
    x[7, bad[0]], x[300, bad[-1]] = np.inf, np.nan
    c = got(ops.block_gemm(qw, ops.block_quantize(Tensor.from_numpy(x, "half")), "float"))
    assert np.all(np.isnan(c[:, bad]))
    good = [t for t in range(tokens) if t not in bad]
    assert np.array_equal(c[:, good], clean[:, good])
    y = got(ops.rms_norm(Tensor.from_numpy(x, "half")))
    assert np.all(np.isnan(y[300, bad[-1]])) and np.all(np.isfinite(y[:, good]))
    big = np.full((k, tokens), 3e4, np.float16)
    ones = ops.block_quantize(Tensor.from_numpy(np.ones((k, m), np.float16), "half"), 128)
    assert np.all(np.isposinf(got(ops.block_gemm(ones, ops.block_quantize(Tensor.from_numpy(big, "half"))))))
