"""The operators of a model's feed-forward layer, case by case, for timing them.

  norm      GpuRuntime.rms_norm: root-mean-square norm with the residual's addition, its output in 16 bits or
            in 8 bits with a scale for each block of 128
  norm_bwd  GpuRuntime.rms_norm_backward: the gradients of its input and its weight
  quantize  GpuRuntime.fp8_quantize: 8 bits with a scale for each block of 128 or of 128 x 128, optionally the
            transposed matrix in the same pass
  gemm      GpuRuntime.fp8_gemm: the product of two such matrices
  gated     GpuRuntime.gated_linear: act(x Wg^T) * (x Wu^T), and (train) with GpuRuntime.gated_linear_backward
            behind it, which gives the gradients of x and of both weights

`draw` covers the same ranges: 1 to 16384 rows, widths of 64 to 16384, sizes that are multiples of 128, of 8, or
odd, padded leading dimensions, both 8-bit types and block shapes, both layouts of the projections' weights,
their halves in one tensor or apart.
"""
import math
import os
import sys

import torch

own = False
_runtime = None
_F8 = {"e4m3": (torch.float8_e4m3fn, 448.0), "e5m2": (torch.float8_e5m2, 57344.0)}
_FLOAT = {"bf16": torch.bfloat16, "f32": torch.float32}
_LEAST = 2.0 ** -100   # a block's largest magnitude counts as at least this


def _t0g():
    path = os.path.join(os.getcwd(), "t0-gpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import t0g
    return t0g


def _rt():
    """The process's runtime handle, opened once, as a program keeps it."""
    global _runtime
    if _runtime is None:
        _runtime = _t0g().GpuRuntime.new(0)
    return _runtime


def _norm(name, rows, width, x="bf16", residual=True, y="bf16", pad=0):
    """y: "bf16", "f32", or "e4m3" or "e5m2" for 8 bits with scales.  The sum with the residual goes out too."""
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "x": x, "residual": residual, "y": y, "pad": pad}


def _norm_bwd(name, rows, width, x="bf16", dsum=True, pad=0):
    """dsum: a gradient that reaches the sum past the norm."""
    return {"name": name, "kind": "norm_bwd", "rows": rows, "width": width, "x": x, "dsum": dsum, "pad": pad}


def _quantize(name, rows, width, x="bf16", q="e4m3", block="row", both=False, pad=0):
    return {"name": name, "kind": "quantize", "rows": rows, "width": width, "x": x, "q": q, "block": block, "both": both,
            "pad": pad}


def _gemm(name, m, n, k, a="e4m3", b="e4m3", block="tile", out="bf16", pad=0):
    """block: what B has a scale for, "row" (1 x 128) or "tile" (128 x 128).  A has one for each 1 x 128."""
    return {"name": name, "kind": "gemm", "m": m, "n": n, "k": k, "a": a, "b": b, "block": block, "out": out, "pad": pad}


def _gated(name, rows, features, width, train, layout="NT", act="silu", apart=False, pad=0):
    return {"name": name, "kind": "gated", "rows": rows, "features": features, "width": width, "train": train,
            "layout": layout, "act": act, "apart": apart, "pad": pad}


def listed():
    return [
        # one token's norm while an answer is decoded: launches decide
        _norm("norm_1x4096", 1, 4096),
        # a long prompt's norm in front of an 8-bit projection
        _norm("norm_8192x4096_e4m3", 8192, 4096, y="e4m3"),
        # a training step's backward pass through the norm and the residual stream
        _norm_bwd("norm_bwd_8192x4096", 8192, 4096),
        # a decoding batch's activations
        _quantize("quantize_16x4096", 16, 4096),
        # a training step's gradients, for the product with the weights and the one with the inputs
        _quantize("quantize_8192x11008_both", 8192, 11008, both=True),
        # one token through an 8-bit projection: the weight is read once
        _gemm("gemm_1x11008x4096", 1, 11008, 4096),
        # a ragged batch and a projection whose rows are not aligned
        _gemm("gemm_777x5001x1023", 777, 5001, 1023, out="f32"),
        # a weight's gradient: both operands with a scale for each 1 x 128
        _gemm("gemm_4096x11008x8192_row", 4096, 11008, 8192, b="e4m3", block="row", out="f32"),
        # the largest projection of a long prompt
        _gemm("gemm_8192x8192x8192", 8192, 8192, 8192),
        # one token through both projections
        _gated("gated_1x11008x4096", 1, 11008, 4096, False),
        # a ragged prompt, weights stored [width][features], rows that are not aligned
        _gated("gated_1000x2731x1023_nn", 1000, 2731, 1023, False, "NN"),
        # a training step of the layer
        _gated("gated_2048x11008x4096_train", 2048, 11008, 4096, True),
    ]


def _size(rng, lo, hi, step):
    """An integer spread over the logarithm of [lo, hi], a multiple of `step` (1: odd)."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    if step == 1:
        return min(hi - 1 + hi % 2, max(lo, int(v)) | 1)
    return min(hi, max(step, int(v / step + 0.5) * step))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_bwd", "quantize", "gemm", "gemm", "gemm", "gated", "gated", "gated"])
    pad = rng.choice([0, 0, 16, 3])
    while True:
        rows = _size(rng, 1, 16384, rng.choice([1, 1, 8, 128]))
        width = _size(rng, 64, 16384, rng.choice([1, 8, 128, 128]))
        other = _size(rng, 64, 16384, rng.choice([1, 8, 128, 128]))
        train = kind == "gated" and rng.random() < 0.5
        if kind in ("gemm", "gated"):
            if 1 << 20 <= rows * width * other * (1 if kind == "gemm" else 6 if train else 2) <= 1 << 39:
                break
        elif rows * width <= 8192 * 11008:
            break
    x, f8 = rng.choice(["bf16", "bf16", "f32"]), rng.choice(["e4m3", "e4m3", "e5m2"])
    if kind == "norm":
        c = _norm("", rows, width, x, rng.random() < 0.7, rng.choice(["bf16", "bf16", "f32", f8, f8]), pad)
    elif kind == "norm_bwd":
        c = _norm_bwd("", rows, width, x, rng.random() < 0.7, pad)
    elif kind == "quantize":
        c = _quantize("", rows, width, x, f8, rng.choice(["row", "row", "tile"]), rng.random() < 0.5, pad)
    elif kind == "gemm":
        c = _gemm("", rows, other, width, f8, rng.choice(["e4m3", "e4m3", "e5m2"]), rng.choice(["row", "tile"]),
                  rng.choice(["bf16", "bf16", "f32"]), pad)
    else:
        c = _gated("", rows, other, width, train, rng.choice(["NT", "NT", "NN"]), rng.choice(["silu", "silu", "gelu"]),
                   rng.random() < 0.3, pad)
    c.pop("name")
    return c


def _blocks(n):
    return (n + 127) // 128


def _quantized(v, q, block):
    """v in 8 bits and its scales, [blocks of the columns][rows, or blocks of the rows]."""
    dtype, most = _F8[q]
    rows, cols = v.shape
    high = 128 if block == "tile" else 1
    padded = torch.zeros((-(-rows // high) * high, _blocks(cols) * 128), dtype=v.dtype, device=v.device)
    padded[:rows, :cols] = v
    tiles = padded.reshape(-1, high, _blocks(cols), 128)
    scale = tiles.abs().amax(dim=(1, 3), keepdim=True).clamp(min=_LEAST) / most
    return (tiles / scale).reshape(padded.shape)[:rows, :cols].to(dtype), scale[:, 0, :, 0].t()


def _values(q, scale, block, real):
    """What 8-bit values and their scales stand for."""
    s = scale.t().to(real).repeat_interleave(128, dim=1)[:, :q.shape[1]]
    if block == "tile":
        s = s.repeat_interleave(128, dim=0)[:q.shape[0]]
    return q.to(real) * s


def _inputs(case, seed):
    """The case's input tensors, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pad = case["pad"]

    def normal(r, c, scale, dtype="bf16"):
        return torch.randn((r, c + pad), generator=g, device="cuda").mul_(scale).to(_FLOAT[dtype])[:, :c]

    def eight(r, c, scale, q, block):
        """A quantized matrix of which a few columns are much larger than the others, as activations have them."""
        v = torch.randn((r, c), generator=g, device="cuda").mul_(scale)
        v *= torch.where(torch.rand(c, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        v, s = _quantized(v, q, block)
        held = torch.zeros((r, c + pad), dtype=torch.uint8, device="cuda")
        held[:, :c] = v.view(torch.uint8)
        return held.view(_F8[q][0])[:, :c], s.contiguous()

    kind = case["kind"]
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        s = dict(zip(("a", "a_scales"), eight(m, k, 1.0, case["a"], "row")))
        s["b"], s["b_scales"] = eight(n, k, k ** -0.5, case["b"], case["block"])
        return s
    rows, width = case["rows"], case["width"]
    if kind == "gated":
        f = case["features"]
        s = {"x": normal(rows, width, 1.0)}
        if case["layout"] == "NT":
            both = normal(2 * f, width, width ** -0.5)
            s["wg"], s["wu"] = both[:f], both[f:]
        else:
            both = normal(width, 2 * f, width ** -0.5)
            s["wg"], s["wu"] = both[:, :f], both[:, f:]
        if case["apart"]:
            s["wg"], s["wu"] = (w.contiguous() for w in (s["wg"], s["wu"]))
        if case["train"]:
            s["dh"] = normal(rows, f, 1.0)
        return s
    s = {"x": normal(rows, width, 2.0, case["x"])}
    if kind == "quantize":
        return s
    s["weight"] = (1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(torch.bfloat16)
    if kind == "norm" and case["residual"]:
        s["residual"] = normal(rows, width, 2.0, case["x"])
    if kind == "norm_bwd":
        s["dy"] = normal(rows, width, 1.0)
        if case["dsum"]:
            s["dsum"] = normal(rows, width, 1.0, case["x"])
    return s


_EPS = 1e-6


def _empty(*shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["names"] = case, ()
    if own:
        _outputs(s)
        s["rt"] = _rt()
        s["calls"] = _calls(s)
    torch.cuda.synchronize()   # the runtime's stream is its own: the inputs are there before it is used
    return s


def _outputs(s):
    """The buffers that a program keeps for the outputs; s["names"]: those that run() returns."""
    case, kind = s["case"], s["case"]["kind"]
    if kind == "gemm":
        s["c"] = _empty(case["m"], case["n"], dtype=_FLOAT[case["out"]])
        s["names"] = ("c",)
        return
    rows, width = case["rows"], case["width"]
    if kind == "gated":
        f = case["features"]
        s["h"] = _empty(rows, f, dtype=torch.bfloat16)
        s["names"] = ("h",)
        if case["train"]:
            s["gate"], s["up"] = _empty(rows, f, dtype=torch.bfloat16), _empty(rows, f, dtype=torch.bfloat16)
            s["dx"] = _empty(rows, width, dtype=torch.bfloat16)
            s["dwg"], s["dwu"] = (_empty(*s["wg"].shape, dtype=torch.bfloat16) for _ in range(2))
            s["names"] = ("h", "dx", "dwg", "dwu")
    elif kind == "norm_bwd":
        s["dx"], s["dw"] = _empty(rows, width, dtype=_FLOAT[case["x"]]), _empty(width, dtype=torch.float32)
        s["names"] = ("dx", "dw")
    elif kind == "norm":
        if case["residual"]:
            s["sum"] = _empty(rows, width, dtype=_FLOAT[case["x"]])
            s["names"] += ("sum",)
        if case["y"] in _FLOAT:
            s["y"] = _empty(rows, width, dtype=_FLOAT[case["y"]])
            s["names"] += ("y",)
        else:
            s["q"], s["scales"] = _empty(rows, width, dtype=_F8[case["y"]][0]), _empty(_blocks(width), rows, dtype=torch.float32)
            s["names"] += ("q", "scales")
    else:
        high = _blocks(rows) if case["block"] == "tile" else rows
        f8 = _F8[case["q"]][0]
        s["q"], s["scales"] = _empty(rows, width, dtype=f8), _empty(_blocks(width), high, dtype=torch.float32)
        s["names"] = ("q", "scales")
        if case["both"]:
            wide = _blocks(width) if case["block"] == "tile" else width
            s["qt"], s["scales_t"] = _empty(width, rows, dtype=f8), _empty(_blocks(rows), wide, dtype=torch.float32)
            s["names"] += ("qt", "scales_t")


def _calls(s):
    """The calls of one pass: methods of the runtime and their descriptors."""
    t0g, case, kind, rt = _t0g(), s["case"], s["case"]["kind"], s["rt"]
    of = {"bf16": t0g.BF16, "f32": t0g.F32, "e4m3": t0g.E4M3, "e5m2": t0g.E5M2}
    blocks = {"row": t0g.BLOCK_ROW, "tile": t0g.BLOCK_TILE}

    def p(name):
        return s[name].data_ptr() if s.get(name) is not None else 0

    def ld(name):
        return s[name].stride(0) if s.get(name) is not None else 0

    if kind == "gemm":
        return [(rt.fp8_gemm, t0g.fp8_gemm_desc(
            p("a"), p("a_scales"), p("b"), p("b_scales"), p("c"), case["m"], case["n"], case["k"], lda=ld("a"), ldb=ld("b"),
            a_dtype=of[case["a"]], b_dtype=of[case["b"]], b_block=blocks[case["block"]], out_dtype=of[case["out"]]))]
    rows, width = case["rows"], case["width"]
    if kind == "gated":
        same = dict(transpose=case["layout"], activation=case["act"], ldx=ld("x"), ldw=ld("wg"))
        calls = [(rt.gated_linear, t0g.gated_linear_desc(p("x"), p("wg"), p("wu"), p("h"), rows, case["features"], width,
                                                         gate=p("gate"), up=p("up"), **same))]
        if case["train"]:
            calls.append((rt.gated_linear_backward, t0g.gated_linear_backward_desc(
                p("dh"), p("x"), p("wg"), p("wu"), rows, case["features"], width, gate=p("gate"), up=p("up"), dx=p("dx"),
                dwg=p("dwg"), dwu=p("dwu"), lddh=ld("dh"), **same)))
        return calls
    if kind == "quantize":
        return [(rt.fp8_quantize, t0g.fp8_quantize_desc(
            p("x"), p("q"), p("scales"), rows, width, qt=p("qt"), scales_t=p("scales_t"), ldx=ld("x"), x_dtype=of[case["x"]],
            q_dtype=of[case["q"]], block=blocks[case["block"]]))]
    if kind == "norm":
        eight = case["y"] not in _FLOAT
        return [(rt.rms_norm, t0g.rms_norm_desc(
            p("x"), p("weight"), rows, width, eps=_EPS, residual=p("residual"), sum=p("sum"), y=p("y"), q=p("q"),
            scales=p("scales"), ldx=ld("x"), ldr=ld("residual"), x_dtype=of[case["x"]], residual_dtype=of[case["x"]],
            sum_dtype=of[case["x"]], y_dtype=t0g.BF16 if eight else of[case["y"]], q_dtype=of[case["y"]] if eight else t0g.E4M3))]
    return [(rt.rms_norm_backward, t0g.rms_norm_backward_desc(
        p("dy"), p("x"), p("weight"), rows, width, eps=_EPS, dsum=p("dsum"), dx=p("dx"), dw=p("dw"), lddy=ld("dy"), ldx=ld("x"),
        ldds=ld("dsum"), x_dtype=of[case["x"]], dsum_dtype=of[case["x"]], dx_dtype=of[case["x"]]))]


def _act(name, g):
    """The activation and its derivative."""
    k = 1.702 if name == "gelu" else 1.0
    sig = 1.0 / (1.0 + torch.exp(-k * g))
    return g * sig, sig + k * g * sig * (1.0 - sig)


def run(s):
    if own:
        for call, desc in s["calls"]:
            call(desc)
        return {n: s[n] for n in s["names"]}
    case, kind, real = s["case"], s["case"]["kind"], torch.float32
    if kind == "gemm":
        a, b = _values(s["a"], s["a_scales"], "row", real), _values(s["b"], s["b_scales"], case["block"], real)
        return {"c": (a @ b.t()).to(_FLOAT[case["out"]])}
    x = s["x"].to(real)
    if kind == "gated":
        wg, wu = s["wg"].to(real), s["wu"].to(real)
        nt = case["layout"] == "NT"
        g, u = (x @ (w.t() if nt else w) for w in (wg, wu))
        a, slope = _act(case["act"], g)
        out = {"h": (a * u).to(torch.bfloat16)}
        if case["train"]:
            dh = s["dh"].to(real)
            dg, du = dh * u * slope, dh * a
            out["dx"] = (dg @ (wg if nt else wg.t()) + du @ (wu if nt else wu.t())).to(torch.bfloat16)
            out["dwg"], out["dwu"] = ((d.t() @ x if nt else x.t() @ d).to(torch.bfloat16) for d in (dg, du))
        return out
    if kind == "quantize":
        q, scales = _quantized(x, case["q"], case["block"])
        out = {"q": q, "scales": scales}
        if case["both"]:
            out["qt"], out["scales_t"] = _quantized(x.t(), case["q"], case["block"])
        return out
    w = s["weight"].to(real)
    if kind == "norm":
        out = {}
        if "residual" in s:
            x = x + s["residual"].to(real)
            out["sum"] = x.to(s["x"].dtype)
        y = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + _EPS) * w
        if case["y"] in _FLOAT:
            out["y"] = y.to(_FLOAT[case["y"]])
        else:
            out["q"], out["scales"] = _quantized(y, case["y"], "row")
        return out
    rate = 1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + _EPS)
    dy = s["dy"].to(real)
    unit, dn = x * rate, dy * w
    dx = rate * (dn - unit * (dn * unit).mean(dim=1, keepdim=True))
    if "dsum" in s:
        dx = dx + s["dsum"].to(real)
    return {"dx": dx.to(s["x"].dtype), "dw": (dy * unit).sum(dim=0)}


def work(case):
    kind = case["kind"]
    size = {"bf16": 2.0, "f32": 4.0, "e4m3": 1.0, "e5m2": 1.0}
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4.0 * _blocks(k) * (m + (n if case["block"] == "row" else _blocks(n)))
        return {"bytes": float(m) * k + float(n) * k + size[case["out"]] * m * n + scales, "flops": 2.0 * m * n * k}
    rows, width = case["rows"], case["width"]
    t = float(rows) * width
    if kind == "gated":
        f = case["features"]
        nbytes = 2.0 * (t + 2.0 * f * width + rows * f)
        if case["train"]:   # dh, dx, dwg, dwu
            nbytes += 2.0 * (rows * f + t + 2.0 * f * width)
        return {"bytes": nbytes, "flops": 4.0 * t * f * (3 if case["train"] else 1)}
    if kind == "quantize":
        blocks = _blocks(width) * (_blocks(rows) if case["block"] == "tile" else rows)
        nbytes = t * (size[case["x"]] + 1.0) + 4.0 * blocks
        if case["both"]:
            nbytes += t + 4.0 * _blocks(rows) * (_blocks(width) if case["block"] == "tile" else width)
        return {"bytes": nbytes, "flops": 2.0 * t}
    if kind == "norm":
        nbytes = t * (size[case["x"]] * (3 if case["residual"] else 1) + size[case["y"]]) + 2.0 * width
        return {"bytes": nbytes + (0.0 if case["y"] in _FLOAT else 4.0 * rows * _blocks(width)), "flops": 4.0 * t}
    return {"bytes": t * (2.0 + size[case["x"]] * (3 if case["dsum"] else 2)) + 6.0 * width, "flops": 9.0 * t}


def _exact_quantized(v, q, block):
    """Block by block of 128 columns, from v in 64 bits."""
    dtype, most = _F8[q]
    rows, cols = v.shape
    high = 128 if block == "tile" else 1
    out, scales = torch.empty((rows, cols), dtype=dtype, device="cuda"), []
    band = torch.arange(rows, device="cuda") // high
    for c in range(0, cols, 128):
        part = v[:, c:c + 128]
        top = torch.zeros(int(band[-1]) + 1, dtype=torch.float64, device="cuda")
        top.scatter_reduce_(0, band, part.abs().max(dim=1)[0], "amax")
        s = torch.clamp(top, min=_LEAST) / most
        out[:, c:c + 128] = (part / s[band][:, None]).to(dtype)
        scales.append(s)
    return out, torch.stack(scales)


def exact(case, seed):
    """From the definitions; long products in blocks of the rows."""
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        c = torch.zeros((m, n), dtype=torch.float64, device="cuda")
        for b in range(_blocks(k)):   # the definition's sum over the blocks of k
            cols = slice(128 * b, min(k, 128 * b + 128))
            left = s["a"][:, cols].double() * s["a_scales"][b].double()[:, None]
            each = s["b_scales"][b].double()
            if case["block"] == "tile":
                each = each[torch.arange(n, device="cuda") // 128]
            right = (s["b"][:, cols].double() * each[:, None]).t().contiguous()
            c += left @ right
        return {"c": c}
    x = s["x"].double()
    rows, width = x.shape
    if kind == "gated":
        nt = case["layout"] == "NT"
        wg, wu = ((w if nt else w.t()).double().contiguous() for w in (s["wg"], s["wu"]))   # [features][width]
        out = {"h": torch.empty((rows, case["features"]), dtype=torch.float64, device="cuda")}
        if case["train"]:
            out["dx"] = torch.empty_like(x)
            out["dwg"], out["dwu"] = torch.zeros_like(wg), torch.zeros_like(wu)
        k = 1.702 if case["act"] == "gelu" else 1.0
        for r in range(0, rows, 2048):
            part = slice(r, r + 2048)
            g, u = x[part] @ wg.t().contiguous(), x[part] @ wu.t().contiguous()
            sig = torch.sigmoid(k * g)
            out["h"][part] = g * sig * u
            if case["train"]:
                dh = s["dh"][part].double()
                dg = dh * u * (sig + g * k * torch.sigmoid(-k * g) * sig)
                du = dh * g * sig
                out["dx"][part] = dg @ wg + du @ wu
                out["dwg"] += dg.t().contiguous() @ x[part]
                out["dwu"] += du.t().contiguous() @ x[part]
        if case["train"] and not nt:
            out["dwg"], out["dwu"] = out["dwg"].t().contiguous(), out["dwu"].t().contiguous()
        return out
    if kind == "quantize":
        out = dict(zip(("q", "scales"), _exact_quantized(x, case["q"], case["block"])))
        if case["both"]:
            out["qt"], out["scales_t"] = _exact_quantized(x.t(), case["q"], case["block"])
        return out
    w = s["weight"].double()
    if kind == "norm":
        out = {}
        if "residual" in s:
            x = x + s["residual"].double()
            out["sum"] = x
        y = x * w[None, :] / (torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / width + _EPS) ** 0.5
        if case["y"] in _FLOAT:
            out["y"] = y
        else:
            out["q"], out["scales"] = _exact_quantized(y, case["y"], "row")
        return out
    # the Jacobian of y_j = w_j x_j / r with r = sqrt(mean x^2 + eps), row by row of it
    r = (torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / width + _EPS) ** 0.5
    dy = s["dy"].double()
    along = (dy * w * x).sum(dim=1, keepdim=True)
    dx = dy * w / r - x * along / (width * r ** 3)
    if "dsum" in s:
        dx = dx + s["dsum"].double()
    return {"dx": dx, "dw": (dy * x / r).sum(dim=0)}
