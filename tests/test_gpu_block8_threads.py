"""The 8-bit linear layer called by several host threads at once, each on a stream of its own."""
import threading

import numpy as np
import pytest

from solid_b200 import Tensor, ops
from solid_b200._lib import BlocksView, Matrix
from test_gpu_block8 import EPS, got, upload, values

pytestmark = pytest.mark.gpu

CALLS = 4000


def run_together(workers):
    errors, start = [], threading.Barrier(len(workers))

    def body(f):
        try:
            start.wait()
            f()
        except Exception as e:                               # handed to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=body, args=(f,)) for f in workers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


@pytest.mark.parametrize("dtype", ["half", "float"])
@pytest.mark.parametrize("op", ["norm", "codes", "gradient"])
def test_long_and_short_rows(gpu, op, dtype):
    """Rows of different lengths take the same kernel with different amounts of shared memory; the library's calls follow
    each other as closely as they can, without Python's part between them."""
    import torch
    from solid_b200 import _lib
    lib, rng = _lib.get(), np.random.default_rng(1)
    es = 2 if dtype == "half" else 4
    workers, checks = [], []
    for n, rows in ((8192, 150), (2056, 150), (8192, 150), (2056, 150)):
        x, r, w = upload(values(rng, n, rows, dtype), dtype), upload(values(rng, n, rows, dtype), dtype), upload(values(rng, n, 1, dtype)[:, 0], dtype)
        stream = torch.cuda.Stream()
        mx, mr = Matrix(x.ptr, es, es * n), Matrix(r.ptr, es, es * n)
        out, out2 = Tensor.empty([n, rows], dtype), Tensor.empty([n, rows], dtype)
        mo, mo2 = Matrix(out.ptr, es, es * n), Matrix(out2.ptr, es, es * n)
        if op == "norm":
            def call(args=(dtype, n, rows, mx, mr, w.ptr, EPS, mo2, mo, stream.cuda_stream)):
                lib.rms_norm(*args)
            want = ops.rms_norm(x, w, EPS, r)
            checks.append((out, want[0], out2, want[1]))
        elif op == "codes":
            codes, scales = Tensor.empty([n, rows], "uint8"), Tensor.empty([rows, (n + 127) // 128], "float")

            def call(args=(dtype, n, rows, mx, mr, w.ptr, EPS, mo2, BlocksView(codes.ptr, n, scales.ptr, 4, 4 * rows, 1, 0), stream.cuda_stream)):
                lib.rms_norm_quantize(*args)
            want = ops.rms_norm_quantize(x, w, EPS, r)
            checks.append((codes, want[0].codes, scales, want[0].scales))
        else:
            dw = Tensor.empty([n], "float")
            buffer = torch.empty(lib.rms_norm_grad_buffer_size(dtype, n, rows, 0), dtype=torch.uint8, device="cuda")

            def call(args=(dtype, n, rows, mx, mr, w.ptr, EPS, mx, mo, dw.ptr, buffer.data_ptr(), stream.cuda_stream), keep=buffer):
                lib.rms_norm_grad(*args)
            want = ops.rms_norm_grad(x, r, w, EPS, x)
            checks.append((out, want[0], dw, want[1]))

        def worker(call=call, keep=(x, r, w, out, out2)):
            torch.cuda.set_device(0)
            for _ in range(CALLS):
                call()
        workers.append(worker)
    torch.cuda.synchronize()
    run_together(workers)
    torch.cuda.synchronize()
    for a, b, c, d in checks:
        assert np.array_equal(got(a), got(b)) and np.array_equal(got(c), got(d))


def test_the_layer_in_several_threads(gpu):
    """Whole calls of the Python layer, decode and batch sizes beside each other: what they give alone."""
    import torch
    rng = np.random.default_rng(3)
    workers, outs, wants = [], [], []

    def layer(x, r, w, g):
        q, h = ops.rms_norm_quantize(x, g, EPS, r)
        y = ops.block_gemm(ops.block_quantize(w, 128), q, "float")
        dh, dg = ops.rms_norm_grad(h, r, g, EPS)
        return y, h, dh, dg

    for k, m, tokens in ((1024, 300, 1), (4096, 512, 300), (640, 700, 160), (2048, 256, 64)):
        t = [upload(values(rng, *s, "half"), "half") for s in ((k, tokens), (k, tokens), (k, m))] + [upload(values(rng, k, 1, "half")[:, 0], "half")]
        wants.append([got(v).tobytes() for v in layer(*t)])
        stream, mine = torch.cuda.Stream(), []
        outs.append(mine)

        def worker(t=t, stream=stream, mine=mine):
            torch.cuda.set_device(0)
            with torch.cuda.stream(stream):
                for _ in range(50):
                    mine[:] = layer(*t)
                stream.synchronize()
        workers.append(worker)
    torch.cuda.synchronize()
    run_together(workers)
    for mine, want in zip(outs, wants):
        assert [got(v).tobytes() for v in mine] == want
