"""Operations on device tensors with Ocean's names and argument meaning, dispatching
through the Solid function tables exactly as Ocean's GPU module does
(src/core/gpu/op/tensor_{unary,binary,copy,fill,reduce_all,reduce_axis}_gpu.c of the
reference): same-dtype elementwise kernels, conversion only in copy, global
reductions returning host scalars, axis reductions writing device tensors.

The mixed-dtype rules applied before dispatch mirror the interface layer
(src/core/generic/tensor_op.c:141-186): operands are brought to a common type,
broadcast with zero strides, and byte-swapped or unaligned operands are
normalised by a converting copy -- except where a fused entry point accepts them
directly.
"""
from __future__ import annotations

import builtins as _py
import struct
from typing import NamedTuple

import numpy as np

from . import _lib
from . import _ocean
from . import dtypes as dt
from . import oplist as ol
from .tensor import Tensor


def _stream(t: Tensor) -> int:
    import torch
    return torch.cuda.current_stream(t.storage.device).cuda_stream


def _lib_for(t: Tensor):
    import torch
    torch.cuda.set_device(t.storage.device)              # Solid reads launch parameters from the current device
    return _lib.get()


def _dispatch(name: str, *args):
    """Call OcTensorGPU_<name> of the Ocean-level dispatch library; tensors become views on the
    current torch stream of their device."""
    import ctypes as C
    oc = _ocean.get()
    conv, keep = [], []
    for a in args:
        if isinstance(a, Tensor):
            v = oc.view(a, _stream(a)); keep.append(v); conv.append(C.byref(v))
        else:
            conv.append(a)
    oc._check(oc.fn(name)(*conv), name)


def scalar_bytes(value, dtype: str) -> bytes:
    """Python number -> the bytes of a solid_scalar member of `dtype` (half uses the library's own rounding)."""
    if dtype == "bool":
        return struct.pack("<B", 1 if value else 0)
    if dtype in dt.UINT or dtype in dt.SINT:
        return np.array(value).astype(dt.NUMPY[dtype]).tobytes()
    if dtype == "float":
        return struct.pack("<f", float(value))
    if dtype == "double":
        return struct.pack("<d", float(value))
    if dtype == "half":
        return _half_bits(float(value)).tobytes()
    c = complex(value)
    if dtype == "cfloat":
        return struct.pack("<ff", c.real, c.imag)
    if dtype == "cdouble":
        return struct.pack("<dd", c.real, c.imag)
    if dtype == "chalf":
        return _half_bits(c.real).tobytes() + _half_bits(c.imag).tobytes()
    raise KeyError(dtype)


def _half_bits(x: float) -> np.ndarray:
    """float -> binary16 bits, rounding half away from zero on the dropped mantissa bits
    (solid/src/base/generic/half.c:101-149)."""
    raw = np.array([x], dtype=np.float32).view(np.uint32)[0]
    d, e, s = int(raw & 0x7FFFFF), int((raw >> 23) & 0xFF), int((raw >> 16) & 0x8000)
    if e < 112:
        h = 0
    elif e > 143:
        h = 0x7F00 if (e == 255 and d) else (s | 0x7C00)
    else:
        h = (((e - 112) << 10) | (d >> 13) | s) + (1 if (d & 0x1FFF) >= 0x1000 else 0)
    return np.array([h & 0xFFFF], dtype=np.uint16)


# ---------------------------------------------------------------------------
# copy / convert
# ---------------------------------------------------------------------------
def copy(src: Tensor, dst: Tensor) -> Tensor:
    """dst[...] = src with type conversion, byte-order handling and any alignment."""
    _dispatch("copy", src, dst)
    return dst


def cast(src: Tensor, dtype: str) -> Tensor:
    return copy(src, Tensor.empty(src.size, dtype, src.storage.device))


def clone(src: Tensor) -> Tensor:
    return copy(src, Tensor.empty(src.size, src.dtype, src.storage.device))


def byteswap(t: Tensor) -> Tensor:
    """Reverse the stored bytes in place and flip the flag, so the logical values are unchanged."""
    _dispatch("byteswapNoFlag", t)
    t.byteswapped = not t.byteswapped
    return t


def fill(t: Tensor, value) -> Tensor:
    import ctypes as C
    sv = _ocean.get().scalar(scalar_bytes(value, t.dtype), t.dtype)
    _dispatch("fill", t, C.byref(sv))
    return t


def fill_nan(t: Tensor, value) -> Tensor:
    import ctypes as C
    sv = _ocean.get().scalar(scalar_bytes(value, t.dtype), t.dtype)
    _dispatch("fillNaN", t, C.byref(sv))
    return t


def masked_fill(t: Tensor, mask: Tensor, value) -> Tensor:
    import ctypes as C
    m = mask.broadcast_to(t.size)
    sv = _ocean.get().scalar(scalar_bytes(value, t.dtype), t.dtype)
    _dispatch("maskedFill", t, m, C.byref(sv))
    return t


# ---------------------------------------------------------------------------
# elementwise
# ---------------------------------------------------------------------------
_RANK = {n: i for i, n in enumerate(dt.NAMES)}


def common_type(a: str, b: str) -> str:
    """Smallest type that holds both (order of the type table; a signed/unsigned
    pair of equal width moves to the next wider signed type, integers with a
    floating type take the floating type)."""
    if a == b:
        return a
    ca, cb = a in dt.COMPLEX, b in dt.COMPLEX
    fa, fb = a in dt.GROUPS["float"], b in dt.GROUPS["float"]
    if fa or fb:
        width = max(dt.SIZE[dt.elem_type(x)] for x in (a, b) if x in dt.GROUPS["float"])
        for x in (a, b):
            if x not in dt.GROUPS["float"] and dt.SIZE[x] >= 4:
                width = max(width, 8 if dt.SIZE[x] >= 4 and width < 8 and dt.SIZE[x] > 2 else width)
        base = {2: "half", 4: "float", 8: "double"}[width]
        return {"half": "chalf", "float": "cfloat", "double": "cdouble"}[base] if (ca or cb) else base
    if a == "bool":
        return b
    if b == "bool":
        return a
    sa, sb = a in dt.SINT, b in dt.SINT
    if sa == sb:
        return a if dt.SIZE[a] >= dt.SIZE[b] else b
    s, u = (a, b) if sa else (b, a)
    if dt.SIZE[s] > dt.SIZE[u]:
        return s
    return {1: "int16", 2: "int32", 4: "int64", 8: "double"}[dt.SIZE[u]]


def _prepared(t: Tensor, dtype: str, size) -> Tensor:
    """Operand as the elementwise kernels require it: common dtype, native byte order, aligned."""
    aligned = t.ptr % t.elemsize == 0 and _py.all(s % t.elemsize == 0 for s in t.strides)
    if t.dtype != dtype or t.byteswapped or not aligned:
        t = cast(t, dtype)
    return t.broadcast_to(size)


def _broadcast_size(*tensors):
    nd = max(t.ndims for t in tensors)
    size = [1] * nd
    for t in tensors:
        own = [1] * (nd - t.ndims) + t.size
        for i, s in enumerate(own):
            if s != 1:
                if size[i] != 1 and size[i] != s:
                    raise ValueError("incompatible sizes")
                size[i] = s
    return size


def unary(name: str, src: Tensor, dst: Tensor | None = None) -> Tensor:
    if src.dtype not in dt.GROUPS[ol.UNARY_OPS[name]]:
        raise TypeError("%s is not available for type %s" % (name, src.dtype))
    x = _prepared(src, src.dtype, src.size)
    if name in ("isinf", "isnan", "isfinite", "isposinf", "isneginf"):
        rtype = "bool"
    elif name == "absolute":
        rtype = dt.elem_type(src.dtype)
    else:
        rtype = src.dtype
    out = dst if (dst is not None and dst.dtype == rtype and not dst.byteswapped) else Tensor.empty(src.size, rtype, src.storage.device)
    _dispatch(_ocean.ocean_name(name), x, out)
    if dst is not None and out is not dst:
        copy(out, dst)
        return dst
    return out


def binary(name: str, a: Tensor, b: Tensor, dst: Tensor | None = None) -> Tensor:
    size = _broadcast_size(a, b)
    # shifts keep the type of the shifted tensor (the count is cast to int8); every other
    # operation works in the common type of both operands
    ctype = a.dtype if name in ("bitshift_left", "bitshift_right") else common_type(a.dtype, b.dtype)
    if name == "power" and a.dtype in dt.GROUPS["integer_bool"] and b.dtype in dt.GROUPS["integer_bool"]:
        ctype = a.dtype                                  # integer base with an integer exponent (cast to int16)
    if ctype not in dt.GROUPS[ol.BINARY_OPS[name]]:
        raise TypeError("%s is not available for type %s" % (name, ctype))
    x = _prepared(a, ctype, size)
    if name in ("bitshift_left", "bitshift_right"):
        y = _prepared(b, "int8", size)
    elif name == "power" and ctype in dt.GROUPS["integer_bool"]:
        y = _prepared(b, "int16", size)
    else:
        y = _prepared(b, ctype, size)
    rtype = "bool" if name in ol.COMPARE_OPS else ctype
    out = dst if (dst is not None and dst.dtype == rtype and not dst.byteswapped and dst.size == size) \
        else Tensor.empty(size, rtype, a.storage.device)
    _dispatch(_ocean.ocean_name(name), x, y, out)
    if dst is not None and out is not dst:
        copy(out, dst)
        return dst
    return out


def scalar_op(name: str, a: Tensor, value, dst: Tensor | None = None) -> Tensor:
    """Tensor (op) Python scalar in the tensor's own type with the scalar passed by value (Ocean's
    addScalar, subtractScalar, multiplyScalar, bitwise{And,Or,Xor}Scalar without the 0-d device tensor)."""
    if name not in ol.SCALAR_OPS or a.dtype not in dt.GROUPS[ol.SCALAR_OPS[name]]:
        raise TypeError("%s with a scalar is not available for type %s" % (name, a.dtype))
    x = _native(a)
    out = dst if (dst is not None and dst.dtype == a.dtype and not dst.byteswapped and dst.size == a.size) \
        else Tensor.empty(a.size, a.dtype, a.storage.device)
    sv = _ocean.get().scalar(scalar_bytes(value, a.dtype), a.dtype)
    import ctypes as C
    _dispatch(_ocean.ocean_name(name) + "Scalar" if name != "multiply" else "multiplyScalar", x, C.byref(sv), out)
    if dst is not None and out is not dst:
        copy(out, dst)
        return dst
    return out


def add(a, b, dst=None):
    return binary("add", a, b, dst)


def subtract(a, b, dst=None):
    return binary("subtract", a, b, dst)


def scale(a, b, dst=None):
    """Elementwise product (Ocean's `scale`; `*` is matrix multiplication there)."""
    return binary("multiply", a, b, dst)


def divide(a, b, dst=None):
    return binary("divide", a, b, dst)


for _n in ol.UNARY_OPS:
    if _n not in globals():
        globals()[_n] = (lambda n: (lambda src, dst=None: unary(n, src, dst)))(_n)
del _n


def axpy(a, x: Tensor, y: Tensor, dst: Tensor | None = None) -> Tensor:
    """a*x + y in the element type with the product rounded first (fused multiplyScalar + add)."""
    size = _broadcast_size(x, y)
    xx, yy = _prepared(x, x.dtype, size), _prepared(y, x.dtype, size)
    out = dst or Tensor.empty(size, x.dtype, x.storage.device)
    _lib_for(out).axpy(x.dtype, size, scalar_bytes(a, x.dtype), xx.strides, xx.ptr, yy.strides, yy.ptr,
                       out.strides, out.ptr, _stream(out))
    return out


def multiply_add(a: Tensor, b: Tensor, c: Tensor, dst: Tensor, ctype: str | None = None) -> Tensor:
    """dst = a*b + c in one kernel, operands in their own dtype / byte order / alignment.
    `ctype` defaults to the type Ocean would promote (a, b, c) to."""
    ctype = ctype or common_type(common_type(a.dtype, b.dtype), c.dtype)
    if ctype in dt.COMPLEX:
        raise TypeError("multiply_add computes in float or double")
    ctype = "double" if ctype not in ("float", "half") else "float"
    size = dst.size
    ops_ = [(t.broadcast_to(size)) for t in (a, b, c)] + [dst]
    _lib_for(dst).mixed_multiply_add(size, [(t.ptr, t.strides, t.dtype, t.byteswapped) for t in ops_], ctype, _stream(dst))
    return dst


# ---------------------------------------------------------------------------
# reductions
# ---------------------------------------------------------------------------
_scratch = {}


def _scratch_buffer(device, nbytes: int):
    import torch
    key = (device, )
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _scratch[key] = buf
    return buf


def _native(t: Tensor) -> Tensor:
    aligned = t.ptr % t.elemsize == 0 and _py.all(s % t.elemsize == 0 for s in t.strides)
    return clone(t) if (t.byteswapped or not aligned) else t


def reduce_all(name: str, t: Tensor, bounds=(), p=None):
    """Global reduction; returns a numpy scalar of the result type (on the host, like Ocean)."""
    import ctypes as C
    t = _native(t)
    oc = _ocean.get()
    oname = _ocean.ocean_name(name)
    if name in ol.REDUCE_BOOL_OPS:
        r = C.c_int(0)
        _dispatch(oname, t, C.byref(r))
        return np.uint8(r.value)
    if name in ol.REDUCE_BOUND1_OPS or name in ol.REDUCE_BOUND2_OPS:
        r = C.c_int(0)
        sv = [oc.scalar(scalar_bytes(b, t.dtype), t.dtype) for b in bounds]
        _dispatch(oname, t, *[C.byref(v) for v in sv], C.byref(r))
        return np.uint8(r.value)
    if name in ol.REDUCE_U64_OPS:
        r = C.c_uint64(0)
        _dispatch(oname, t, C.byref(r))
        return np.uint64(r.value)
    res = _ocean.ScalarView()
    if name in ol.REDUCE_NORM_OPS:
        _dispatch(oname, t, C.c_double(p), C.byref(res))
    else:
        _dispatch(oname, t, C.byref(res))
    rtype = dt.NAMES[res.dtype]
    raw = bytes(C.string_at(C.addressof(res.value), 16))
    return np.frombuffer(raw[: dt.SIZE[rtype]], dtype=dt.NUMPY[rtype])[0]


def reduce_axis(name: str, t: Tensor, axes, dst: Tensor | None = None, p=None, keepdims: bool = False) -> Tensor:
    import ctypes as C
    t = _native(t)
    axes = sorted({a % t.ndims for a in ([axes] if isinstance(axes, int) else axes)})
    keep = [i for i in range(t.ndims) if i not in axes]
    rtype = ol.reduce_result_type("axis_" + name, t.dtype)
    osize = [t.size[i] for i in keep]
    out = dst if dst is not None else Tensor.empty(osize, rtype, t.storage.device)
    ax = (C.c_int * max(len(axes), 1))(*axes)
    oname = _ocean.ocean_name("axis_" + name)
    if p is None:
        _dispatch(oname, t, C.c_int(len(axes)), ax, out)
    else:
        _dispatch(oname, t, C.c_double(p), C.c_int(len(axes)), ax, out)
    if keepdims:
        size = [1 if i in axes else t.size[i] for i in range(t.ndims)]
        return Tensor(out.storage, out.dtype, size, None, out.offset)
    return out


def _reduction(name):
    def run(t: Tensor, axes=None, dst=None, keepdims=False):
        if axes is None:
            return reduce_all(name, t)
        return reduce_axis(name, t, axes, dst, keepdims=keepdims)
    run.__name__ = name
    return run


sum = _reduction("sum")
prod = _reduction("prod")
any = _reduction("any")
all = _reduction("all")
nnz = _reduction("nnz")
maximum = _reduction("maximum")
minimum = _reduction("minimum")
sum_abs = _reduction("sum_abs")
maximum_abs = _reduction("maximum_abs")
minimum_abs = _reduction("minimum_abs")
norm2 = _reduction("norm2")


def norm(t: Tensor, p=2, axes=None, dst=None):
    """p-norm with Ocean's special cases (src/core/interface/tensor_itf.c:5405-5447):
    p=0 counts non-zeros, 1 sums magnitudes, inf takes the largest magnitude, 2 is norm2."""
    name, kw = {0: ("nnz", {}), 1: ("sum_abs", {}), 2: ("norm2", {}), float("inf"): ("maximum_abs", {})}.get(p, ("norm", {"p": float(p)}))
    if axes is None:
        return reduce_all(name, t, **kw)
    return reduce_axis(name, t, axes, dst, **kw)


def axpy_sums(a, x: Tensor, y: Tensor, z: Tensor | None = None, sums=None):
    """Fused z = a*x + y with sum(z) and sum(z*z) left on the device: returns (z, sums) where
    sums is a 2-element torch tensor {sum(z), sum(z*z)} of the element type.  Contiguous float/double."""
    import torch
    if not (x.is_contiguous() and y.is_contiguous()) or x.dtype not in ("float", "double") or x.dtype != y.dtype:
        raise TypeError("axpy_sums takes contiguous float or double tensors of one type")
    lib = _lib_for(x)
    z = z or Tensor.empty(x.size, x.dtype, x.storage.device)
    tdt = torch.float32 if x.dtype == "float" else torch.float64
    if sums is None:
        sums = torch.empty(2, dtype=tdt, device=x.storage.device)
    part = _scratch_buffer(x.storage.device, lib.axpy_sums_buffer_size(x.device_index, x.nelem))
    lib.axpy_sums(x.dtype, x.nelem, scalar_bytes(a, x.dtype), x.ptr, y.ptr, z.ptr, sums.data_ptr(), part.data_ptr(), _stream(x))
    return z, sums


# ----------------------------------------------------------------------------
# indexed access (Ocean's tensor[index] with integer index lists)
# ----------------------------------------------------------------------------
def _index_view(t: Tensor, positions):
    """OcIndexView for `t` and one entry per dimension: None (every position, by stride) or a sequence of integer
    positions (negative ones count from the end).  Returns the view, the selection shape and the objects to keep."""
    import ctypes as C
    oc = _ocean.get()
    if len(positions) != t.ndims:
        raise ValueError("one index entry per dimension is needed")
    ix = _ocean.IndexView()
    ix.view = oc.view(t, _stream(t))
    ix.ndims = t.ndims
    keep, shape = [], []
    for d, pos in enumerate(positions):
        if pos is None:
            ix.size[d] = t.size[d]; shape.append(t.size[d])
            continue
        p = np.asarray(pos, dtype=np.int64).reshape(-1)
        p = np.where(p < 0, p + t.size[d], p)
        if p.size and (p.min() < 0 or p.max() >= t.size[d]):
            raise IndexError("index out of range in dimension %d" % d)
        table = Tensor.from_numpy(p * t.strides[d], "int64", t.storage.device)
        tv = oc.view(table, _stream(t))
        keep += [table, tv]
        ix.offsets[d] = C.pointer(tv)
        ix.size[d] = p.size; shape.append(int(p.size))
    return ix, shape, keep


def take(t: Tensor, positions, dst: Tensor | None = None) -> Tensor:
    """dst = t[positions] (outer product of the per-dimension index lists)."""
    import ctypes as C
    t = _native(t)
    ix, shape, keep = _index_view(t, positions)
    out = dst if dst is not None else Tensor.empty(shape, t.dtype, t.storage.device)
    _dispatch("getIndex", C.byref(ix), out)
    return out


def put(t: Tensor, positions, src: Tensor) -> Tensor:
    """t[positions] = src (positions must not repeat)."""
    import ctypes as C
    ix, shape, keep = _index_view(t, positions)
    _dispatch("setIndex", C.byref(ix), _native(src) if src.dtype == t.dtype else cast(src, t.dtype))
    return t


def fill_at(t: Tensor, positions, value) -> Tensor:
    """t[positions] = value."""
    import ctypes as C
    ix, shape, keep = _index_view(t, positions)
    sv = _ocean.get().scalar(scalar_bytes(value, t.dtype), t.dtype)
    _dispatch("fillIndex", C.byref(ix), C.byref(sv))
    return t


# ----------------------------------------------------------------------------
# the 8-bit linear layer: norm, conversion to 8 bits with scales, product
# ----------------------------------------------------------------------------
# A matrix [n, rows] is column-major like every tensor: a row (a token) is n elements side by side, and dimension 0 is
# the one that a norm or a block of 128 runs along.  Further dimensions count as rows.  Half, float and double; results
# are rounded once, to nearest even, with subnormals.  Operands of different types are widened to their common type, which
# is the results' type too.  The copy family's conversion to half is never used here: it rounds as the reference's CPU code
# does, and turns what is below 2^-15 into zero.
class Blocks(NamedTuple):
    """8-bit floating-point codes with scales: element (i, row) stands for codes[i, row] * scales[row // block, i // 128].

    codes    uint8 tensor [n, rows], stride 1 along dimension 0 (rows on 16-byte boundaries reach the tensor cores)
    scales   float tensor [rows, ceil(n / 128)], or [ceil(rows / 128), ceil(n / 128)] where 128 rows share a scale
    format   "e4m3" or "e5m2"
    """
    codes: Tensor
    scales: Tensor
    format: str = "e4m3"


def _format(name: str) -> int:
    if name not in _lib.FORMATS:
        raise ValueError("unknown 8-bit format %r: e4m3 or e5m2" % (name,))
    return _lib.FORMATS[name]


def _as_rows(t: Tensor):
    """(rows, stride of a row) of a tensor whose dimensions 1.. step evenly, None where they do not."""
    rows, step = 1, 0
    for s, st in zip(t.size[1:], t.strides[1:]):
        if s == 1:
            continue
        if rows == 1:
            step = st
        elif st != step * rows:
            return None
        rows *= s
    return (0 if 0 in t.size[1:] else rows), step


# A single token's call is a few microseconds of work on the GPU, so the host's part is kept as short: matrices that
# the kernels take as they are pass one test, everything else goes the general way through _prepared and clone.
def _row_operand(t: Tensor, dtype: str, size, device, what: str):
    """An operand as the kernels take it, the number of its rows, and its Matrix: of the given type, native, aligned, its
    rows a step apart."""
    if t.storage.device != device:
        raise ValueError("%s is on another device" % what)
    if t.dtype == dtype and len(size) == 2 and t.size == size and not t.byteswapped:
        s0, s1 = t.strides
        p = t.storage.data_ptr() + t.offset
        if not (p | s0 | s1) & (dt.SIZE[dtype] - 1):
            return t, size[1], _lib.Matrix(p, s0, s1)
    t = _prepared(t, dtype, size)
    r = _as_rows(t)
    if r is None:
        t = clone(t)
        r = _as_rows(t)
    return t, r[0], _lib.Matrix(t.ptr, t.strides[0], r[1])


def _layer_type(what: str, x: Tensor, *others) -> str:
    """The common type of an operator's operands (None: absent).  Widening a half or a float is exact."""
    if x.dtype not in ("half", "float", "double"):
        raise TypeError("%s is not available for type %s" % (what, x.dtype))
    dtype = x.dtype
    for t in others:
        if t is not None and t.dtype != dtype:
            dtype = common_type(dtype, t.dtype)
    if dtype not in ("half", "float", "double"):
        raise TypeError("%s is not available for type %s" % (what, dtype))
    return dtype


def _takes(dst: Tensor | None, dtype: str, what: str):
    """Refuses a tensor of halves for a result that has more bits: the copy to half would flush and round otherwise."""
    if dst is not None and dst.dtype in ("half", "chalf") and dtype != "half":
        raise TypeError("%s is of type %s and cannot go into a tensor of type %s" % (what, dtype, dst.dtype))


def _row_input(x: Tensor, dtype: str, what: str):
    if not x.size:
        raise ValueError("%s needs at least one dimension" % what)
    return _row_operand(x, dtype, x.size, x.storage.device, "the input")


def _view(storage, dtype: str, size, strides, offset: int = 0) -> Tensor:
    """A tensor of fields that are known to be right."""
    t = Tensor.__new__(Tensor)
    t.storage, t.dtype, t.size, t.strides, t.offset, t.byteswapped = storage, dtype, size, strides, offset, False
    return t


def _new(storage, size, dtype: str):
    """A new column-major tensor beside `storage`, and its Matrix."""
    es = dt.SIZE[dtype]
    strides, step = [], es
    for s in size:
        strides.append(step)
        step *= s
    t = _view(storage.new_empty(step if step > 16 else 16), dtype, list(size), strides)
    return t, _lib.Matrix(t.storage.data_ptr(), es, es * size[0])


def _norm_weight(weight, x: Tensor):
    """The weights as the kernels take them (contiguous, in the type of x, which is the operands' common one) and their address."""
    if weight is None:
        return None, None
    if weight.size != x.size[:1]:
        raise ValueError("the weights need size [%d]" % x.size[0])
    if weight.storage.device != x.storage.device:
        raise ValueError("weight is on another device")
    es = dt.SIZE[x.dtype]
    p = weight.storage.data_ptr() + weight.offset
    if weight.dtype == x.dtype and weight.strides[0] == es and not weight.byteswapped and p % es == 0:
        return weight, p
    w = clone(_prepared(weight, x.dtype, weight.size))
    return w, w.storage.data_ptr()


def _result(dst, size, dtype: str, storage):
    """Where a kernel writes, and its Matrix: dst itself where the kernel can, else a new tensor that is copied there."""
    if dst is not None:
        if dst.size != size:
            raise ValueError("the result has size %s, not %s" % (size, dst.size))
        if dst.storage.device != storage.device:
            raise ValueError("the result is on another device")
        r = _as_rows(dst)
        if dst.dtype == dtype and not dst.byteswapped and r is not None and \
                dst.ptr % dst.elemsize == 0 and _py.all(s % dst.elemsize == 0 for s in dst.strides) and \
                _py.all(st != 0 or s <= 1 for s, st in zip(dst.size, dst.strides)):
            return dst, _lib.Matrix(dst.ptr, dst.strides[0], r[1])
    return _new(storage, size, dtype)


def _delivered(out: Tensor, dst) -> Tensor:
    return out if dst is None or out is dst else copy(out, dst)


def _here(device):
    """The library with the tensors' device current, and that device's current stream."""
    import torch
    if torch.cuda.current_device() != device.index:
        torch.cuda.set_device(device)
    return _lib.get(), torch._C._cuda_getCurrentRawStream(device.index)


def rms_norm(x: Tensor, weight: Tensor | None = None, eps: float = 1e-6, residual: Tensor | None = None,
             dst: Tensor | None = None, h: Tensor | None = None):
    """Root-mean-square norm along dimension 0: y = x * weight / sqrt(mean(x^2) + eps).

    With a residual the sum h = x + residual is normalised (before it is rounded) and returned too: (y, h).  dst and h
    say where y and h go; h may be the residual's own tensor, dst that of x.  y and h have the operands' common type:
    halves beside float weights or a float residual give floats."""
    dtype = _layer_type("rms_norm", x, weight, residual)
    _takes(dst, dtype, "the norm")
    x, rows, mx, res, mr, w, pw, total, mh = _norm_operands(x, weight, residual, h, dtype, "rms_norm")
    out, my = _result(dst, x.size, x.dtype, x.storage)
    lib, stream = _here(x.storage.device)
    lib.rms_norm(x.dtype, x.size[0], rows, mx, mr, pw, eps, mh, my, stream)
    y = _delivered(out, dst)
    return y if total is None else (y, _delivered(total, h))


def _norm_operands(x, weight, residual, h, dtype, what):
    """What rms_norm and rms_norm_quantize share.  The tensors are returned beside their addresses to keep them alive."""
    _takes(h, dtype, "the sum")
    x, rows, mx = _row_input(x, dtype, what)
    w, pw = _norm_weight(weight, x)
    if residual is None:
        if h is not None:
            raise ValueError("h is x + residual: there is no residual")
        return x, rows, mx, None, None, w, pw, None, None
    res, _, mr = _row_operand(residual, x.dtype, x.size, x.storage.device, "residual")
    total, mh = _result(h, x.size, x.dtype, x.storage)
    return x, rows, mx, res, mr, w, pw, total, mh


def _empty_blocks(n: int, rows: int, block: int, format: str, storage):
    """Room for codes (rows padded to 16 bytes) with the scales behind them, and its BlocksView."""
    ld = (n + 15) // 16 * 16
    rb, nb = (rows + block - 1) // block, (n + 127) // 128
    room = storage.new_empty(ld * rows + 4 * rb * nb // 16 * 16 + 16)
    p = room.data_ptr()
    return Blocks(_view(room, "uint8", [n, rows], [1, ld]), _view(room, "float", [rb, nb], [4, 4 * rb], ld * rows), format), \
        _lib.BlocksView(p, ld, p + ld * rows, 4, 4 * rb, block, _lib.FORMATS[format])


def _blocks_view(b: Blocks, what: str):
    """(codes, BlocksView) of a caller's codes and scales, checked against each other."""
    codes, scales = b.codes, b.scales
    if codes.dtype != "uint8" or scales.dtype != "float" or scales.byteswapped:
        raise TypeError("%s: codes are uint8, scales native floats" % what)
    if len(codes.size) != 2 or len(scales.size) != 2:
        raise ValueError("%s: codes and scales are matrices" % what)
    if scales.storage.device != codes.storage.device:
        raise ValueError("%s: codes and scales are on different devices" % what)
    n, rows = codes.size
    nb = (n + 127) // 128
    if scales.size == [rows, nb]:
        block = 1
    elif scales.size == [(rows + 127) // 128, nb]:
        block = 128
    else:
        raise ValueError("%s: scales of size %s do not belong to codes of size %s" % (what, scales.size, codes.size))
    fmt = _format(b.format)
    if n > 1 and codes.strides[0] != 1:                    # rows on 16-byte boundaries, for the tensor cores
        ld = (n + 15) // 16 * 16
        codes = copy(codes, _view(codes.storage.new_empty(ld * rows), "uint8", [n, rows], [1, ld]))
    return codes, _lib.BlocksView(codes.storage.data_ptr() + codes.offset, codes.strides[1],
                                  scales.storage.data_ptr() + scales.offset, scales.strides[0], scales.strides[1], block, fmt)


def rms_norm_quantize(x: Tensor, weight: Tensor | None = None, eps: float = 1e-6, residual: Tensor | None = None,
                      format: str = "e4m3", h: Tensor | None = None):
    """rms_norm whose y is returned as Blocks, a scale for 128 elements of each row; with a residual (Blocks, h)."""
    _format(format)
    dtype = _layer_type("rms_norm_quantize", x, weight, residual)
    x, rows, mx, res, mr, w, pw, total, mh = _norm_operands(x, weight, residual, h, dtype, "rms_norm_quantize")
    out, view = _empty_blocks(x.size[0], rows, 1, format, x.storage)
    lib, stream = _here(x.storage.device)
    lib.rms_norm_quantize(x.dtype, x.size[0], rows, mx, mr, pw, eps, mh, view, stream)
    return out if total is None else (out, _delivered(total, h))


def rms_norm_grad(dy: Tensor, h: Tensor, weight: Tensor | None = None, eps: float = 1e-6, dres: Tensor | None = None,
                  dst: Tensor | None = None):
    """Gradient of rms_norm at h (the input, or x + residual): returns (dh, dweight).

    dres, the gradient that reaches h past the norm, is added to dh.  dh has the operands' common type, dweight the work type
    of that (half: float)."""
    if dy.size != h.size or (dres is not None and dres.size != h.size):
        raise ValueError("gradients have the size of h, %s" % h.size)
    dtype = _layer_type("rms_norm_grad", h, dy, weight, dres)
    _takes(dst, dtype, "the gradient")
    h, rows, mh = _row_input(h, dtype, "rms_norm_grad")
    device, n = h.storage.device, h.size[0]
    dy, _, mg = _row_operand(dy, dtype, h.size, device, "dy")
    w, pw = _norm_weight(weight, h)
    mr = None
    if dres is not None:
        dres, _, mr = _row_operand(dres, dtype, h.size, device, "dres")
    out, mo = _result(dst, h.size, dtype, h.storage)
    dweight, md = _new(h.storage, [n], "double" if dtype == "double" else "float")
    lib, stream = _here(device)
    # a buffer of its own for each call: calls on several streams and captured graphs share nothing
    buf = h.storage.new_empty(lib.rms_norm_grad_buffer_size(dtype, n, rows, device.index))
    lib.rms_norm_grad(dtype, n, rows, mg, mh, pw, eps, mr, mo, md.ptr, buf.data_ptr(), stream)
    return _delivered(out, dst), dweight


def block_quantize(x: Tensor, block: int = 1, format: str = "e4m3") -> Blocks:
    """8-bit codes of a matrix [n, rows] with a scale for 128 elements of dimension 0 by `block` (1 or 128) rows.

    In 32 bits: scale = max(largest magnitude * (1 / largest code), 2^-126); code = x * (1 / scale) to nearest even.
    Strides are free: block_quantize(x.T) gives the codes of the transposed matrix."""
    _format(format)
    if block not in (1, 128):
        raise ValueError("a scale belongs to 1 or 128 rows")
    x, rows, mx = _row_input(x, _layer_type("block_quantize", x), "block_quantize")
    out, view = _empty_blocks(x.size[0], rows, block, format, x.storage)
    lib, stream = _here(x.storage.device)
    lib.block_quantize(x.dtype, x.size[0], rows, mx, view, stream)
    return out


def block_gemm(a: Blocks, b: Blocks, dtype: str | None = None, dst: Tensor | None = None) -> Tensor:
    """Product of 8-bit matrices with scales: c[m, n] = sum over k of a[k, m] b[k, n], half or float.

    Without a dtype the result has the type of dst (float where that is neither half nor float), and is half without dst.
    A float result for a tensor of halves is rounded once, by the product itself.

    A linear layer with weights W [K, M] and tokens X [K, N] (both Blocks): y = block_gemm(W, X).  Its gradients:
    dX = block_gemm(block_quantize(w.T, 128), block_quantize(dy)), and dW = block_gemm(block_quantize(x.T),
    block_quantize(dy.T), "float"), a matrix [K, M]."""
    if dtype is None:
        dtype = "half" if dst is None or dst.dtype in ("half", "chalf") else "float"
    if dtype not in ("half", "float"):
        raise TypeError("block_gemm gives half or float, not %s" % dtype)
    if dst is not None and dst.dtype == "half":
        dtype = "half"
    _takes(dst, dtype, "the product")
    ka, va = _blocks_view(a, "a")
    kb, vb = _blocks_view(b, "b")
    k, m = ka.size
    device = ka.storage.device
    if kb.size[0] != k:
        raise ValueError("block_gemm: depths %d and %d differ" % (k, kb.size[0]))
    if kb.storage.device != device:
        raise ValueError("block_gemm: operands on different devices")
    n = kb.size[1]
    out, mc = _result(dst, [m, n], dtype, ka.storage)
    lib, stream = _here(device)
    lib.block_gemm(dtype, m, n, k, va, vb, mc, stream)
    return _delivered(out, dst)
