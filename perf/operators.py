"""The losses of a projection onto a vocabulary, case by case, for timing them.

  ce       GpuRuntime.linear_cross_entropy: softmax cross entropy of x W^T, the loss of every row, its
           log-sum-exp, and (grad "x", "w" or "xw") the gradients
  distill  GpuRuntime.linear_distill: the divergence from a teacher of whom the top logits are known,
           optionally with the labels' cross entropy in the same pass (log-sum-exp of the logits over the
           temperature)

Sizes are rows x vocabulary x width.  `draw` covers the same ranges: 1 to 8192 rows, 256 to 131072
tokens, widths of 64 to 4096, both layouts of the weight, padded leading dimensions, ignored rows, 1 to
256 teacher entries of which some are missing, and sizes that are multiples of 64, of 8, or odd.
"""
import math
import os
import sys

import torch

own = False
_runtime = None


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


def _ce(name, rows, vocab, width, grad, layout="NT", pad=0, ignored=0.0):
    return {"name": name, "kind": "ce", "rows": rows, "vocab": vocab, "width": width, "grad": grad, "layout": layout,
            "pad": pad, "ignored": ignored, "scale": 1.0}


def _distill(name, rows, vocab, width, top, temperature, labels, grad="xw", layout="NT", pad=0, ignored=0.0, narrow=False):
    """narrow: the teacher's logits in bf16 and 32-bit tokens, else f32 and 64-bit ones."""
    return {"name": name, "kind": "distill", "rows": rows, "vocab": vocab, "width": width, "grad": grad, "layout": layout,
            "pad": pad, "ignored": ignored, "scale": 1.0, "top": top, "temperature": temperature, "labels": labels,
            "narrow": narrow}


def listed():
    return [
        # one token's log-probability: the weight is read once
        _ce("score_1x32000x2048", 1, 32000, 2048, ""),
        # the tokens of a decoding batch scored against a large vocabulary
        _ce("score_16x131072x4096", 16, 131072, 4096, ""),
        # a ragged prompt scored by a head whose rows are not 16-byte aligned
        _ce("score_777x50001x1023", 777, 50001, 1023, ""),
        # a small classifier's step: launches decide
        _ce("ce_64x1000x256", 64, 1000, 256, "xw"),
        # fine-tuning on short answers: many ignored prompt tokens, the weight stored [width][vocabulary]
        _ce("ce_512x32000x1024_nn", 512, 32000, 1024, "xw", "NN", 0, 0.4),
        # an ordinary training step
        _ce("ce_2048x32000x4096", 2048, 32000, 4096, "xw", "NT", 0, 0.05),
        # a frozen head: only the hidden states' gradient, padded rows
        _ce("ce_4096x50304x2048_dx", 4096, 50304, 2048, "x", "NT", 64, 0.1),
        # the largest training step: the logits would take 4.3 GB
        _ce("ce_8192x131072x4096", 8192, 131072, 4096, "xw", "NT", 0, 0.02),
        # a short distillation step
        _distill("distill_32x32000x1024_k8", 32, 32000, 1024, 8, 1.0, False, narrow=True),
        # an odd vocabulary, labels missing in places
        _distill("distill_1000x50001x768_k50", 1000, 50001, 768, 50, 2.0, True, "xw", "NT", 8, 0.1),
        # distillation and labels in one pass, two temperatures
        _distill("distill_2048x32000x2048_k64", 2048, 32000, 2048, 64, 2.0, True, "xw", "NT", 0, 0.05),
        # many teacher entries over a large vocabulary, no labels
        _distill("distill_4096x131072x2048_k128", 4096, 131072, 2048, 128, 1.0, False, "xw", "NT", 0, 0.02),
    ]


def _size(rng, lo, hi, step):
    """An integer spread over the logarithm of [lo, hi], a multiple of `step` (1: odd)."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    if step == 1:
        return min(hi - 1 + hi % 2, max(lo, int(v)) | 1)
    return min(hi, max(step, int(v / step + 0.5) * step))


def draw(rng):
    kind = rng.choice(["ce", "ce", "ce", "distill", "distill"])
    while True:
        rows = _size(rng, 1, 8192, rng.choice([1, 1, 8, 64]))
        vocab = _size(rng, 256, 131072, rng.choice([1, 8, 64, 64]))
        width = _size(rng, 64, 4096, rng.choice([1, 8, 64, 64]))
        if 1 << 20 <= rows * vocab * width <= 1 << 41:
            break
    grad = rng.choice(["", "x", "xw", "xw"])
    layout, pad = rng.choice(["NT", "NT", "NN"]), rng.choice([0, 0, 8, 24])
    ignored = rng.choice([0.0, 0.05, 0.5])
    if kind == "ce":
        c = _ce("", rows, vocab, width, grad, layout, pad, ignored)
        c["scale"] = rng.choice([1.0, 1.0, 0.5])
    else:
        c = _distill("", rows, vocab, width, _size(rng, 1, 256, rng.choice([1, 8])), rng.choice([1.0, 2.0, 4.0]),
                     rng.random() < 0.5, grad, layout, pad, ignored, rng.random() < 0.5)
    c.pop("name")
    return c


def _inputs(case, seed):
    """The case's input tensors, from the seed alone: hidden states of unit size, a weight that gives logits of
    deviation 2.5 (a trained head's are peaked), labels that favour the frequent (low) tokens."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, width, pad = case["rows"], case["vocab"], case["width"], case["pad"]

    def normal(r, c, scale):
        t = torch.randn((r, c + pad), generator=g, device="cuda")
        return t.mul_(scale).to(torch.bfloat16)[:, :c]

    def unit(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    s = {"x": normal(rows, width, 1.0)}
    w = (vocab, width) if case["layout"] == "NT" else (width, vocab)
    s["w"] = normal(*w, 2.5 * width ** -0.5)
    out = unit(rows) < case["ignored"]
    if case["kind"] == "ce" or case["labels"]:
        y = torch.clamp((unit(rows).double() ** 3 * vocab).long(), max=vocab - 1)
        s["labels"] = torch.where(out, torch.full_like(y, -100), y)
    # a row's weight in the loss, as a mask of lengths or a sampled weight gives it
    s["dloss"] = 0.5 + unit(rows)
    if case["kind"] == "distill":
        top = min(case["top"], vocab)
        # distinct tokens of every row, in no order; the teacher's logits descend
        gap = 1 + (unit(rows, top).double() * (vocab // top)).long().clamp_(max=vocab // top - 1)
        tokens = (gap.cumsum(1) - 1)[:, torch.argsort(unit(top))]
        gone = (unit(rows, top) < 0.03) | out[:, None]   # entries that a shorter list pads, and rows without a teacher
        s["tokens"] = torch.where(gone, torch.full_like(tokens, -1), tokens)
        s["teacher"] = torch.sort(3.0 * torch.randn((rows, top), generator=g, device="cuda"), dim=1, descending=True)[0]
        if case["narrow"]:
            s["teacher"], s["tokens"] = s["teacher"].to(torch.bfloat16), s["tokens"].int()
    return s


_LABEL_WEIGHT, _DISTILL_WEIGHT = 0.25, 0.75


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    rows, vocab, width, grad = case["rows"], case["vocab"], case["width"], case["grad"]
    s["loss"], s["lse"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    s["dx"] = torch.empty((rows, width), dtype=torch.bfloat16, device="cuda") if "x" in grad else None
    s["dw"] = torch.empty(s["w"].shape, dtype=torch.bfloat16, device="cuda") if "w" in grad else None
    s["mean"] = 1.0 / rows
    if own:
        t0g = _t0g()

        def p(name):
            return s[name].data_ptr() if s.get(name) is not None else 0

        head = dict(transpose=case["layout"], lse=p("lse"), dx=p("dx"), dw=p("dw"), dloss=p("dloss"), loss_scale=s["mean"],
                    logit_scale=case["scale"], ldx=s["x"].stride(0), ldw=s["w"].stride(0))
        if case["kind"] == "ce":
            s["desc"] = t0g.linear_ce_desc(p("x"), p("w"), p("labels"), p("loss"), rows, vocab, width, **head)
        else:
            both = case["labels"]
            s["desc"] = t0g.linear_distill_desc(
                p("x"), p("w"), p("teacher"), p("tokens"), p("loss"), rows, vocab, width, s["tokens"].shape[1],
                temperature=case["temperature"], labels=p("labels"), label_weight=_LABEL_WEIGHT if both else 0.0,
                distill_weight=_DISTILL_WEIGHT if both else 1.0, teacher_dtype=t0g.BF16 if case["narrow"] else t0g.F32,
                token_type=t0g.I32 if case["narrow"] else t0g.I64, **head)
        s["rt"] = _rt()
    torch.cuda.synchronize()   # the runtime's stream is its own: the inputs are there before it is used
    return s


def _loss(s, real):
    """The losses and gradients from elementary operations in the type `real`."""
    case, vocab = s["case"], s["case"]["vocab"]
    x, w = s["x"].to(real), s["w"].to(real)
    wt = w.t() if case["layout"] == "NT" else w
    z = (x @ wt) * case["scale"]
    top = z.max(dim=1, keepdim=True)[0]
    zero = torch.zeros((), dtype=real, device=z.device)

    def softmax(t):
        e = torch.exp((z - top) / t)
        total = e.sum(dim=1, keepdim=True)
        return e / total, (top / t + torch.log(total))[:, 0]

    p, lse = softmax(1.0)
    rate = s["dloss"].to(real) * s["mean"] * case["scale"]
    loss, used, grad = zero, torch.zeros(len(z), dtype=torch.bool, device=z.device), None
    if "labels" in s:
        a = _LABEL_WEIGHT if case["kind"] == "distill" else 1.0
        y = s["labels"]
        has = (y >= 0) & (y < vocab)
        at = torch.where(has, y, torch.zeros_like(y))[:, None]
        loss = torch.where(has, a * (lse - z.gather(1, at)[:, 0]), zero)
        used = has
        if case["grad"]:
            c = torch.where(has, a * rate, zero)[:, None]
            grad = (p * c).scatter_add_(1, at, -c)
    if case["kind"] == "distill":
        b, t = (_DISTILL_WEIGHT if "labels" in s else 1.0), case["temperature"]
        i = s["tokens"].long()
        has = (i >= 0) & (i < vocab)
        at = torch.where(has, i, torch.zeros_like(i))
        u = torch.where(has, s["teacher"].to(real) / t, zero - math.inf)
        some = has.any(dim=1)
        u = torch.where(some[:, None], u, torch.zeros_like(u))
        u = u - u.max(dim=1, keepdim=True)[0]
        log_q = u - torch.log(torch.exp(u).sum(dim=1, keepdim=True))
        q = torch.where(has, torch.exp(log_q), zero)
        pt, lse = softmax(t)
        each = torch.where(has, q * (log_q - z.gather(1, at) / t + lse[:, None]), zero)
        loss = loss + b * t * t * each.sum(dim=1)
        used = used | some
        if case["grad"]:
            c = torch.where(some, b * t * rate, zero)[:, None]
            more = (pt * c).scatter_add_(1, at, -c * q)
            grad = more if grad is None else grad + more
    out = {"loss": loss, "lse": torch.where(used, lse, zero)}
    if "x" in case["grad"]:
        out["dx"] = grad @ wt.t()
    if "w" in case["grad"]:
        out["dw"] = grad.t() @ x if case["layout"] == "NT" else x.t() @ grad
    return out


def run(s):
    if not own:
        return {k: v.to(torch.bfloat16) if k in ("dx", "dw") else v for k, v in _loss(s, torch.float32).items()}
    if s["case"]["kind"] == "ce":
        s["rt"].linear_cross_entropy(s["desc"])
    else:
        s["rt"].linear_distill(s["desc"])
    return {k: s[k] for k in ("loss", "lse", "dx", "dw") if s[k] is not None}


def work(case):
    t, v, d, grad = case["rows"], case["vocab"], case["width"], case["grad"]
    tvd = float(t) * v * d
    nbytes = 2.0 * (t * d + v * d) + 8.0 * t + 8.0 * t
    if case["kind"] == "distill":
        nbytes += (6.0 if case["narrow"] else 12.0) * min(case["top"], v) * t
    return {"bytes": nbytes + 2.0 * t * d * ("x" in grad) + 2.0 * v * d * ("w" in grad),
            "flops": 2 * tvd * (1 + len(grad))}


def exact(case, seed):
    """From the definition, row block by row block: the logits' gradient is written out entry by entry."""
    s = _inputs(case, seed)
    t, v, kind = case["rows"], case["vocab"], case["kind"]
    w = s["w"].double()
    if case["layout"] == "NN":
        w = w.t().contiguous()   # [vocabulary][width]
    loss, lse = torch.zeros(t, dtype=torch.float64, device="cuda"), torch.zeros(t, dtype=torch.float64, device="cuda")
    dx = torch.zeros((t, case["width"]), dtype=torch.float64, device="cuda")
    dw = torch.zeros((v, case["width"]), dtype=torch.float64, device="cuda")
    block = max(1, min(t, (1 << 28) // v))
    tau = case.get("temperature", 1.0)
    a = 0.0 if "labels" not in s else (1.0 if kind == "ce" else _LABEL_WEIGHT)
    b = 0.0 if kind == "ce" else (_DISTILL_WEIGHT if "labels" in s else 1.0)
    for r0 in range(0, t, block):
        r = slice(r0, min(t, r0 + block))
        x = s["x"][r].double()
        n = len(x)
        z = (x @ w.t().contiguous()) * case["scale"]
        every = torch.arange(n, device="cuda")
        rate = s["dloss"][r].double() / t * case["scale"]
        g = torch.zeros_like(z)
        used = torch.zeros(n, dtype=torch.bool, device="cuda")
        if a:
            y = s["labels"][r]
            ok = every[(y >= 0) & (y < v)]
            logp = torch.log_softmax(z[ok], dim=1)
            loss[r0 + ok] += -a * logp[torch.arange(len(ok), device="cuda"), y[ok]]
            g[ok] += a * rate[ok][:, None] * torch.exp(logp)
            g[ok, y[ok]] -= a * rate[ok]
            used[ok] = True
        if b:
            i = s["tokens"][r].long()
            rows, cols = torch.nonzero((i >= 0) & (i < v), as_tuple=True)
            tokens = i[rows, cols]
            weight = torch.zeros(i.shape, dtype=torch.float64, device="cuda")
            weight[rows, cols] = torch.exp((s["teacher"][r].double()[rows, cols] - s["teacher"][r].double().max()) / tau)
            q = weight / weight.sum(dim=1, keepdim=True).clamp(min=1e-300)
            ok = every[weight.sum(dim=1) > 0]
            used[ok] = True
            logp = torch.log_softmax(z / tau, dim=1)
            kl = torch.zeros(n, dtype=torch.float64, device="cuda")
            kl.index_add_(0, rows, q[rows, cols] * (torch.log(q[rows, cols]) - logp[rows, tokens]))
            loss[r] += b * tau * tau * kl
            g[ok] += b * tau * rate[ok][:, None] * torch.exp(logp[ok])
            g[rows, tokens] -= b * tau * rate[rows] * q[rows, cols]
            del logp
        lse[r] = torch.where(used, torch.logsumexp(z / tau, dim=1), torch.zeros_like(lse[r]))
        if "x" in case["grad"]:
            dx[r] = g @ w
        if "w" in case["grad"]:
            dw += g.t().contiguous() @ x
        del z, g
    out = {"loss": loss, "lse": lse}
    if "x" in case["grad"]:
        out["dx"] = dx
    if "w" in case["grad"]:
        out["dw"] = dw if case["layout"] == "NT" else dw.t().contiguous()
    return out
