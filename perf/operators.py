"""Cases of the 8-bit linear layer: the norm in front of it, the conversion to 8 bits with scales, and the product.

Matrices are column-major in the framework: a token is a column with its features side by side, so a torch tensor
[tokens, features] in C order is the framework's tensor of size [features, tokens].  Codes are held in uint8 tensors,
scales in float tensors of size [tokens, blocks], the token's index running fastest.
"""
import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
BLOCK = 128
TYPES = {"half": torch.float16, "float": torch.float32}
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "e5m2": (torch.float8_e5m2, 57344.0)}
LARGEST = 8192                                     # rows of the largest square product


def listed():
    return [
        # decoding: the norm of one token in front of a layer, the residual added on the way
        {"name": "norm one token", "op": "norm", "type": "half", "n": 4096, "rows": 1, "residual": True},
        # prefill or a training step: every token of a batch
        {"name": "norm 8192 tokens", "op": "norm", "type": "half", "n": 4096, "rows": 8192, "residual": True},
        # a decode batch straight into the 8-bit layer
        {"name": "norm to 8 bits, 16 tokens", "op": "norm8", "type": "half", "n": 8192, "rows": 16, "residual": True, "format": "e4m3"},
        # prefill into the 8-bit layer
        {"name": "norm to 8 bits, 4096 tokens", "op": "norm8", "type": "half", "n": 8192, "rows": 4096, "residual": True, "format": "e4m3"},
        # the norm's backward pass, the residual stream's gradient added
        {"name": "norm gradient 4096 tokens", "op": "grad", "type": "half", "n": 4096, "rows": 4096, "residual": True},
        # the same for a ragged batch in 32 bits
        {"name": "norm gradient ragged", "op": "grad", "type": "float", "n": 1000, "rows": 777, "residual": False},
        # a weight matrix after an optimiser's step: square blocks
        {"name": "weights to 8 bits", "op": "to8", "type": "float", "n": 8192, "rows": 4096, "block": 128, "across": False, "format": "e4m3"},
        # an output gradient for the weights' gradient: blocks along the tokens, codes of the transposed matrix
        {"name": "gradient across to 8 bits", "op": "to8", "type": "half", "n": 4096, "rows": 4096, "block": 1, "across": True, "format": "e5m2"},
        # decoding: one token through a layer
        {"name": "product one token", "op": "product", "m": 4096, "n": 1, "k": 4096, "block": 128, "type": "half", "formats": "e4m3 e4m3"},
        # a decode batch
        {"name": "product 64 tokens", "op": "product", "m": 8192, "n": 64, "k": 8192, "block": 128, "type": "half", "formats": "e4m3 e4m3"},
        # the weights' gradient of a ragged layer: both sides scaled along the tokens, 32-bit sums out
        {"name": "product weight gradient", "op": "product", "m": 4096, "n": 2000, "k": 5000, "block": 1, "type": "float", "formats": "e5m2 e4m3"},
        # prefill or training: many tokens through a large layer
        {"name": "product 8192 tokens", "op": "product", "m": 8192, "n": 8192, "k": 8192, "block": 128, "type": "half", "formats": "e4m3 e4m3"},
    ]


def draw(rng):
    def size(low, high):
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        if rng.random() < 0.5:                     # half of them are whole vectors, the others whatever comes
            v = max(1, v // 16 * 16) if v >= 16 else v
        return min(max(v, low), high)

    op = rng.choice(["norm", "norm8", "grad", "to8", "product", "product"])
    kind = rng.choice(["half", "float"])
    form = rng.choice(["e4m3", "e4m3", "e5m2"])
    if op == "product":
        m, n, k = size(128, LARGEST), size(1, LARGEST), size(128, LARGEST)
        return {"op": op, "m": m, "n": n, "k": k, "block": rng.choice([1, 128, 128]), "type": kind, "formats": form + " e4m3"}
    n = size(64, 16384)
    case = {"op": op, "type": kind, "n": n, "rows": size(1, min(16384, (1 << 25) // n))}
    if op == "to8":
        case.update(block=rng.choice([1, 128]), across=rng.choice([True, False]), format=form)
    else:
        case.update(residual=rng.choice([True, False]))
        if op == "norm8":
            case.update(format=form)
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def held(x):
    """A matrix [rows, n] as a program holds it: the torch view, and the bytes that the framework's tensor stands on."""
    rows, n = x.shape
    size = x.element_size()
    name = {torch.float16: "half", torch.float32: "float"}.get(x.dtype, "uint8")
    flat = x.as_strided((rows * x.stride(0),), (1,)).view(torch.uint8)
    return {"torch": x, "flat": flat, "type": name, "size": [n, rows], "strides": [size, size * x.stride(0)]}


def features(g, rows, n, kind):
    """Activations: some features are many times larger than the others, as in a residual stream."""
    spread = torch.exp(1.2 * torch.randn(n, generator=g, device="cuda"))
    return held((torch.randn(rows, n, generator=g, device="cuda") * spread).to(TYPES[kind]))


def with_scales(x, form, per_rows):
    """Codes (rows padded to whole 16 bytes) and scales of x [rows, n], one scale for 128 features by `per_rows` rows."""
    code, top = CODES[form]
    rows, n = x.shape
    nb, rb = blocks(n), -(-rows // per_rows)
    full = torch.zeros(rb * per_rows, nb * BLOCK, device="cuda")
    full[:rows, :n] = x
    tiles = full.view(rb, per_rows, nb, BLOCK)
    scale = (tiles.abs().amax((1, 3)) / top).clamp_min(2.0 ** -126)
    codes = torch.zeros(rows, (n + 15) // 16 * 16, device="cuda", dtype=code)
    codes[:, :n] = (tiles / scale[:, None, :, None]).view(rb * per_rows, nb * BLOCK)[:rows, :n].to(code)
    return held(codes[:, :n]), held(scale.t().contiguous())


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        fa, fb = case["formats"].split()
        # weights of a layer (or, with a scale for each row, output gradients), and activations
        a = torch.randn(m, k, generator=g, device="cuda") * (k ** -0.5)
        b = features(g, n, k, "float")["torch"]
        a, sa = with_scales(a, fa, case["block"])
        b, sb = with_scales(b, fb, 1)
        return {"case": case, "a": a, "sa": sa, "b": b, "sb": sb}
    rows, n, kind = case["rows"], case["n"], case["type"]
    state = {"case": case, "x": features(g, rows, n, kind)}
    if op == "to8":
        return state
    state["w"] = held((1 + 0.1 * torch.randn(1, n, generator=g, device="cuda")).to(TYPES[kind]))
    state["w"].update(size=[n], strides=state["w"]["strides"][:1])
    if case["residual"]:
        state["r"] = features(g, rows, n, kind)
    if op == "grad":
        state["dy"] = held((1e-2 * torch.randn(rows, n, generator=g, device="cuda")).to(TYPES[kind]))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return framework(state)
    case = state["case"]
    op = case["op"]
    if op == "product":
        a = state["a"]["torch"].float() * spread_scales(state["sa"]["torch"], case["block"], *state["a"]["torch"].shape)
        b = state["b"]["torch"].float() * spread_scales(state["sb"]["torch"], 1, *state["b"]["torch"].shape)
        return (b @ a.t()).to(TYPES[case["type"]])
    if op == "to8":
        x = state["x"]["torch"].float()
        return codes_of(x.t() if case["across"] else x, case["format"], case["block"])
    x, w = state["x"]["torch"].float(), state["w"]["torch"].float()
    if op == "grad":
        g = state["dy"]["torch"].float() * w
        r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
        dh = r * g - x * (r * r * r * (g * x).mean(1, keepdim=True))
        if "r" in state:
            dh = dh + state["r"]["torch"].float()
        dw = (state["dy"]["torch"].float() * x * r).sum(0)
        return dh.to(TYPES[case["type"]]), dw
    h = x + state["r"]["torch"].float() if "r" in state else x
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * w
    out = [y.to(TYPES[case["type"]])] if op == "norm" else codes_of(y, case["format"], 1)
    return out + [h.to(TYPES[case["type"]])] if "r" in state else out


def spread_scales(scale, per_rows, rows, n):
    """scales [blocks, row blocks] -> one for each element of [rows, n]."""
    return scale.t().repeat_interleave(per_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :n]


def codes_of(x, form, per_rows):
    code, top = CODES[form]
    rows, n = x.shape
    nb, rb = blocks(n), -(-rows // per_rows)
    tiles = torch.nn.functional.pad(x, (0, nb * BLOCK - n, 0, rb * per_rows - rows)).view(rb, per_rows, nb, BLOCK)
    scale = (tiles.abs().amax((1, 3)) / top).clamp_min(2.0 ** -126)
    q = (tiles * (1 / scale)[:, None, :, None]).clamp(-top, top)
    return [q.view(rb * per_rows, nb * BLOCK)[:rows, :n].to(code), scale.t().contiguous()]


def framework(state):
    if "solid_b200" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "ocean-tensor-package_b200"))
    from solid_b200 import Tensor, ops

    def tensor(key):
        h = state.get(key)
        return None if h is None else Tensor(h["flat"], h["type"], h["size"], h["strides"])

    def matrix(t, kind):
        """The framework's tensor [n, rows] as torch's [rows, n]."""
        v = t.storage.view(kind)
        step = t.elemsize
        return v.as_strided((t.size[1], t.size[0]), (t.strides[1] // step, 1), t.offset // step)

    case = state["case"]
    op = case["op"]
    if op == "product":
        fa, fb = case["formats"].split()
        # the columns of the first operand become the rows of c, whose index runs fastest: a token's outputs side by side
        c = ops.block_gemm(ops.Blocks(tensor("a"), tensor("sa"), fa), ops.Blocks(tensor("b"), tensor("sb"), fb), case["type"])
        return matrix(c, TYPES[case["type"]])
    if op == "to8":
        x = tensor("x")
        q = ops.block_quantize(x.T if case["across"] else x, case["block"], case["format"])
        return [matrix(q.codes, CODES[case["format"]][0]), matrix(q.scales, torch.float32)]
    if op == "grad":
        dh, dw = ops.rms_norm_grad(tensor("dy"), tensor("x"), tensor("w"), EPS, tensor("r"))
        return matrix(dh, TYPES[case["type"]]), dw.storage.view(torch.float32)[:case["n"]]
    if op == "norm":
        out = ops.rms_norm(tensor("x"), tensor("w"), EPS, tensor("r"))
        return [matrix(t, TYPES[case["type"]]) for t in (out if "r" in state else (out,))]
    out = ops.rms_norm_quantize(tensor("x"), tensor("w"), EPS, tensor("r"), case["format"])
    q = out[0] if "r" in state else out
    got = [matrix(q.codes, CODES[case["format"]][0]), matrix(q.scales, torch.float32)]
    return got + [matrix(out[1], TYPES[case["type"]])] if "r" in state else got


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = 2 if case["type"] == "half" else 4
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = blocks(k) * (n + -(-m // case["block"]))
        return {"bytes": m * k + n * k + 4 * scales + m * n * size, "flops": 2.0 * m * n * k}
    n, rows = case["n"], case["rows"]
    e = n * rows
    if op == "to8":
        along, other = (rows, n) if case["across"] else (n, rows)
        return {"bytes": e * (size + 1) + 4 * blocks(along) * -(-other // case["block"]), "flops": 3.0 * e}
    extra = 1 if case["residual"] else 0
    if op == "grad":
        return {"bytes": e * size * (3 + extra) + n * (size + 4), "flops": 10.0 * e}
    moved = e * size * (1 + 2 * extra) + n * size
    if op == "norm":
        return {"bytes": moved + e * size, "flops": 5.0 * e}
    return {"bytes": moved + e + 4 * rows * blocks(n), "flops": 8.0 * e}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def wide(key):
        return s[key]["torch"].to(torch.float64)

    if op == "product":
        total = torch.zeros(case["n"], case["m"], dtype=torch.float64, device="cuda")
        a, b, sa, sb = wide("a"), wide("b"), wide("sa"), wide("sb")
        row = torch.arange(case["m"], device="cuda") // case["block"]
        for i in range(blocks(case["k"])):
            part = slice(i * BLOCK, (i + 1) * BLOCK)
            total += (b[:, part] @ a[:, part].t()) * sb[i][:, None] * sa[i][row][None, :]
        return total

    def to_codes(x, per_rows):
        rows, n = x.shape
        top, least, digits = (448.0, -6, 3) if case["format"] == "e4m3" else (57344.0, -14, 2)
        r, c = torch.arange(rows, device="cuda") // per_rows, torch.arange(n, device="cuda") // BLOCK
        most = torch.zeros(int(r[-1]) + 1, int(c[-1]) + 1, dtype=torch.float64, device="cuda")
        most = most.view(-1).scatter_reduce(0, (r[:, None] * most.shape[1] + c[None, :]).view(-1), x.abs().reshape(-1), "amax").view_as(most)
        scale = torch.maximum(most / top, torch.tensor(2.0 ** -126, dtype=torch.float64, device="cuda"))
        q = x / scale[r][:, c]
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** least))) - digits)
        return [torch.round(q / step) * step, scale.t()]

    if op == "to8":
        x = wide("x")
        return to_codes(x.t() if case["across"] else x, case["block"])
    h = wide("x")
    if op == "grad":
        dy, w = wide("dy"), wide("w")
        n = case["n"]
        length = torch.sqrt((h ** 2).sum(1) / n + EPS)
        unit = h / length[:, None]
        dunit = dy * w
        dh = (dunit - unit * ((dunit * unit).sum(1) / n)[:, None]) / length[:, None]
        return (dh + wide("r") if case["residual"] else dh), (dy * unit).sum(0)
    if case["residual"]:
        h = h + wide("r")
    y = h / torch.sqrt((h ** 2).sum(1, keepdim=True) / case["n"] + EPS) * wide("w")
    out = [y] if op == "norm" else to_codes(y, 1)
    return out + [h] if case["residual"] else out
