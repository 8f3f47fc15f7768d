"""Losses of a projection onto a vocabulary (t0g_linear_cross_entropy, t0g_linear_distill)
against their definitions in 64 bits, at sizes, layouts, masks and values where they can go
wrong; gradients also against differences of the loss.

Tolerances, with u = 2^-24 (f32) and the sums of magnitudes |x||W| and |G||W| taken in 64 bits:
  logits     f32 sums of `hidden` exact products: at most e_z = (hidden + 2) u max |x||W| c
  statistics sums of at most 2^17 terms in f32 by lanes, chunks and joins: 2^10 u relative at the very
             most; exp2, log2 and the products around them: 16 u (1 + |lse| + |z|)
  loss       the sum of the errors of its terms, each weighted as in the loss
  dx, dW     G is rounded to bf16 (2^-8 |G|, half a unit of its 8 bits), its own error is that of the probabilities
             (2 e_z + statistics) |P|, the products are summed in f32 and rounded once to the output type
"""
import sys

import pytest
import torch   # on the host only: the device's buffers and streams are the library's runtime's

import hip_rt
import t0g

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _log(msg):
    print(msg, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def rt():
    r = t0g.GpuRuntime.new(0)
    yield r
    r.close()


@pytest.fixture(autouse=True, params=["rows", "fused"])
def form(request):
    """Every test in both forms (fused falls back to by rows where the operands do not allow it)."""
    t0g.set_loss_form(t0g.LOSS_FORM_FUSED if request.param == "fused" else t0g.LOSS_FORM_ROWS)
    yield request.param
    t0g.set_loss_form(t0g.LOSS_FORM_AUTO)


class Case:
    """One problem: inputs on the host, the call's buffers on the device (each in a filled allocation of its
    own, so that a write outside shows and what lies between rows is not read), and the definition in 64 bits."""

    def __init__(self, rows, vocab, hidden, layout="NT", seed=0, pad=0, offset=0, xpad=None, amp=2.0, c=1.0, scale=0.125,
                 dtype="bf16", int32=False, weights=True, want="xw"):
        self.rows, self.vocab, self.hidden, self.layout = rows, vocab, hidden, layout
        self.c, self.scale, self.int32, self.want = c, scale, int32, want
        self.out_type = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.pad, self.offset, self.xpad = pad, offset, pad if xpad is None else xpad
        g = self.g = torch.Generator().manual_seed(seed)
        self.x = torch.randn(rows, hidden, generator=g).bfloat16()
        self.w = (torch.randn(vocab, hidden, generator=g) * amp * hidden ** -0.5).bfloat16()
        self.labels = torch.randint(0, vocab, (rows,), generator=g)
        self.dloss = (0.25 + torch.rand(rows, generator=g)) if weights else None
        self.teacher = None

    def teach(self, top, tau=1.0, a=0.0, b=1.0, half=False, ldt=0, repeat=False):
        g = self.g
        if repeat or top > self.vocab:
            self.tokens = torch.randint(0, self.vocab, (self.rows, top), generator=g)
        else:
            self.tokens = torch.stack([torch.randperm(self.vocab, generator=g)[:top] for _ in range(max(1, self.rows))])
            self.tokens = self.tokens[:self.rows]
        self.teacher = 2 * torch.randn(self.rows, top, generator=g)
        if half:
            self.teacher = self.teacher.bfloat16()
        self.top, self.tau, self.a, self.b, self.ldt = top, tau, a, b, ldt or top
        if not a:
            self.labels = None
        return self

    # ---- the call
    def place(self, rt, t, ld=None, fill=-7.0):
        """t in a larger device buffer of its own, rows ld apart, `offset` elements from an aligned address:
        the buffer's address and host image, and t's place in the image."""
        rows, cols = (1, t.shape[0]) if t.dim() == 1 else t.shape
        ld = ld or cols
        image = torch.full((self.offset + rows * ld + 64,), fill, dtype=t.dtype)
        view = image[self.offset:self.offset + rows * ld].view(rows, ld)[:, :cols]
        view.copy_(t.view(rows, cols))
        addr = rt.upload(self.raw(image))
        self.held.append(addr)
        return addr, image, (view[0] if t.dim() == 1 else view)

    @staticmethod
    def raw(image):
        return (image.view(torch.int16) if image.dtype == torch.bfloat16 else image).numpy()

    def run(self, rt, max_piece=0, keep=False):
        ints = torch.int32 if self.int32 else torch.int64
        itype = t0g.I32 if self.int32 else t0g.I64
        w = self.w if self.layout == "NT" else self.w.t().contiguous()
        nan = float("nan")
        self.held = []

        def inp(t, ld=None):
            if t is None or t.numel() == 0:
                return 0
            addr, image, _ = self.place(rt, t, ld, nan if t.dtype.is_floating_point else 0)
            return addr + self.offset * image.element_size()

        x, wd = inp(self.x, self.hidden + self.xpad), inp(w, w.shape[1] + self.pad)
        dt = self.out_type
        self.bufs = {"loss": self.place(rt, torch.full((self.rows,), -7.0)), "lse": self.place(rt, torch.full((self.rows,), -7.0))}
        if "x" in self.want:
            self.bufs["dx"] = self.place(rt, torch.full((self.rows, self.hidden), -7.0, dtype=dt), self.hidden + self.pad)
        if "w" in self.want:
            self.bufs["dw"] = self.place(rt, torch.full(w.shape, -7.0, dtype=dt), w.shape[1] + self.pad)

        def out(name):
            if name not in self.bufs or not self.bufs[name][2].numel():
                return 0
            return self.bufs[name][0] + self.offset * self.bufs[name][1].element_size()

        kind = t0g.BF16 if dt == torch.bfloat16 else t0g.F32
        head = dict(transpose=self.layout, lse=out("lse"), dx=out("dx"), dw=out("dw"), dloss=inp(self.dloss),
                    loss_scale=self.scale, logit_scale=self.c, label_type=itype, dx_dtype=kind, dw_dtype=kind,
                    ldx=self.hidden + self.xpad, ldw=w.shape[1] + self.pad, lddx=self.hidden + self.pad,
                    lddw=w.shape[1] + self.pad, max_piece=max_piece)
        labels = inp(self.labels.to(ints)) if self.labels is not None else 0
        if self.teacher is None:
            d = t0g.linear_ce_desc(x, wd, labels, out("loss"), self.rows, self.vocab, self.hidden, **head)
            call = rt.linear_cross_entropy
        else:
            # what lies between the rows must not be read as entries
            d = t0g.linear_distill_desc(x, wd, inp(self.teacher, self.ldt), inp(self.tokens.to(ints), self.ldt), out("loss"),
                                        self.rows, self.vocab, self.hidden, self.top, temperature=self.tau, labels=labels,
                                        label_weight=self.a, distill_weight=self.b, ldt=self.ldt, token_type=itype,
                                        teacher_dtype=t0g.BF16 if self.teacher.dtype == torch.bfloat16 else t0g.F32, **head)
            call = rt.linear_distill
        self.desc, self.call = d, call
        call(d)
        got = self.read(rt)
        if not keep:
            self.free(rt)
        return got

    def read(self, rt):
        """The outputs, after all queued work; the whole buffers go into the images."""
        got = {}
        for k, (addr, image, view) in self.bufs.items():
            raw = self.raw(image)
            raw[:] = rt.read(addr, raw.shape, raw.dtype)
            got[k] = view.clone()
        return got

    def refill(self, rt):
        for addr, image, view in self.bufs.values():
            image.fill_(-7.0)
            rt.write(addr, self.raw(image))

    def free(self, rt):
        for addr in self.held:
            rt.free(addr)
        self.held = []

    def untouched(self):
        for name, (_, b, v) in self.bufs.items():
            mask = torch.ones_like(b, dtype=torch.bool)
            rows, cols = (1, v.shape[0]) if v.dim() == 1 else v.shape
            ld = cols if v.dim() == 1 else v.stride(0)
            mask[self.offset:self.offset + rows * ld].view(rows, ld)[:, :cols] = False
            assert bool((b[mask] == -7.0).all()), f"{name}: written outside"

    # ---- the definition
    def define(self):
        x, w = self.x.double(), self.w.double()
        rows, vocab = self.rows, self.vocab
        usable = torch.zeros(rows, dtype=torch.bool)
        a = 1.0 if self.teacher is None else self.a
        y = self.labels
        labelled = (y >= 0) & (y < vocab) if y is not None else usable.clone()
        q = torch.zeros(rows, vocab, dtype=torch.float64)
        taught = usable.clone()
        if self.teacher is not None:
            for t in range(rows):
                ok = (self.tokens[t] >= 0) & (self.tokens[t] < vocab) & (self.teacher[t] != float("-inf"))
                if ok.any():
                    taught[t] = True
                    q[t].index_add_(0, self.tokens[t][ok], torch.softmax(self.teacher[t][ok].double() / self.tau, 0))
        used = labelled | taught
        x = torch.where(used[:, None], x, torch.zeros_like(x))
        z = self.c * (x @ w.t())
        tau = 1.0 if self.teacher is None else self.tau
        lp, lpt = torch.log_softmax(z, 1), torch.log_softmax(z / tau, 1)
        rate = self.scale * (self.dloss.double() if self.dloss is not None else torch.ones(rows)) * self.c
        loss, grad = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, vocab, dtype=torch.float64)
        size = torch.zeros_like(grad)
        pick = torch.where(labelled, y, torch.zeros_like(y))[:, None] if y is not None else None
        if y is not None:
            loss = loss + torch.where(labelled, -a * lp.gather(1, pick)[:, 0], loss)
            m = (labelled * a * rate)[:, None]
            grad = grad + m * (lp.exp() - torch.zeros_like(grad).scatter_(1, pick, 1.0))
            size = size + m.abs() * lp.exp()
        if self.teacher is not None:
            kl = torch.where(q > 0, q * (torch.log(q.clamp(min=1e-300)) - lpt), torch.zeros_like(q)).sum(1)
            loss = loss + torch.where(taught, self.b * tau * tau * kl, torch.zeros_like(kl))
            m = (taught * self.b * tau * rate)[:, None]
            grad = grad + m * (lpt.exp() - q)
            size = size + m.abs() * (lpt.exp() + 16 * U / 2 ** -8 * q)
        lse = torch.where(used, torch.logsumexp(z / tau, 1), torch.zeros(rows, dtype=torch.float64))
        ez = (self.hidden + 2) * U * self.c * (x.abs() @ w.abs().t()).amax(1) if rows else torch.zeros(0)
        zmax = z.abs().amax(1) if rows else torch.zeros(0)
        stat = 2.0 ** 10 * U + 16 * U * (1 + lse.abs() + zmax / min(tau, 1.0))
        weight = abs(a) + (abs(self.b) * tau * max(1.0, tau) if self.teacher is not None else 0.0)
        dp = 2 * ez / min(1.0, tau) + 2 * stat           # relative error of a probability
        gerr = 2.0 ** -8 * grad.abs() + dp[:, None] * size * 1.01
        acc = (vocab + 8) * U
        out = {"loss": (loss, weight * (2 * ez / min(1.0, tau) + 2 * stat + 16 * U * (1 + loss.abs()))),
               "lse": (lse, ez / tau + stat)}

        def product(left, right, lerr):
            v = left @ right
            mag = left.abs() @ right.abs()
            e = lerr @ right.abs() * 1.01 + (max(self.rows, acc / U) + 8) * U * mag + 1e-30
            return v, e + ((v.abs() + e) * 2.0 ** -8 if self.out_type == torch.bfloat16 else v.abs() * U)

        if "x" in self.want:
            out["dx"] = product(grad, w, gerr)
        if "w" in self.want:
            v, e = product(grad.t(), x, gerr.t())
            out["dw"] = (v, e) if self.layout == "NT" else (v.t(), e.t())
        return out

    def check(self, rt, label="", **kw):
        got, want = self.run(rt, **kw), self.define()
        self.untouched()
        for k, (v, tol) in want.items():
            d = (got[k].double() - v).abs()
            worst = float((d / tol.clamp(min=1e-38)).max()) if d.numel() else 0.0
            _log(f"[loss] {label} {self.rows}x{self.vocab}x{self.hidden} {self.layout} {k}: {worst:.3f} of the bound")
            assert bool((d <= tol).all()), f"{label} {k}: {worst:.3f} times the bound"
        return got


SIZES = [
    (1, 1, 1), (1, 2, 8), (2, 300, 64), (3, 257, 33), (5, 1000, 200), (64, 1000, 256), (130, 4100, 72), (65, 4097, 64),
    (257, 520, 136), (300, 777, 96), (9, 9001, 40),
]


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("rows,vocab,hidden", SIZES)
def test_cross_entropy(rt, rows, vocab, hidden, layout):
    Case(rows, vocab, hidden, layout, seed=rows + vocab).check(rt, "ce")


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("rows,vocab,hidden,pad,offset,xpad", [
    (33, 515, 64, 8, 0, 8), (33, 515, 64, 3, 0, 0), (33, 512, 64, 0, 1, 0), (20, 700, 50, 6, 2, 14), (7, 264, 96, 0, 8, 5)])
def test_strides_and_alignment(rt, rows, vocab, hidden, pad, offset, xpad, layout):
    Case(rows, vocab, hidden, layout, seed=3, pad=pad, offset=offset, xpad=xpad).check(rt, "strides")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("want", ["", "x", "w", "xw"])
def test_outputs_asked_for(rt, want, dtype):
    Case(70, 900, 128, want=want, dtype=dtype, weights=False, scale=1.0, int32=True).check(rt, f"want {want or 'loss'}")


@pytest.mark.parametrize("rows,vocab,max_piece", [(40, 1003, 1), (40, 1003, 8), (40, 1000, 130), (300, 2051, 512), (3, 9000, 4104)])
@pytest.mark.parametrize("layout", ["NT", "NN"])
def test_pieces_of_the_vocabulary(rt, rows, vocab, max_piece, layout):
    """Pieces change neither loss nor gradient beyond the order of f32 sums; labels at a piece's first and last token."""
    c = Case(rows, vocab, 72, layout, seed=5)
    piece = max(8, max_piece & ~7)
    edges = [e for v0 in range(0, vocab, piece) for e in (v0, min(v0 + piece, vocab) - 1)]
    for t in range(rows):
        c.labels[t] = edges[(7 * t) % len(edges)]
    c.check(rt, f"pieces of {max_piece}", max_piece=max_piece)


def test_partial_sums_of_dx_in_groups(rt):
    """More planes of dx than are summed at a time (a plane of 40 MiB, groups of six)."""
    rows, hidden = 10240, 1024
    c = Case(rows, 136, hidden, seed=6, want="x", dtype="f32")
    c.check(rt, "groups", max_piece=8)


def test_missing_labels(rt):
    """Rows without a label: loss, lse and gradient 0, and a NaN or infinity there reaches nothing."""
    c = Case(48, 600, 64, seed=7)
    c.labels[::3] = -100
    c.labels[1::7] = 600
    c.labels[2::11] = 2 ** 40 + 5   # beyond 32 bits: its low word is a valid token
    c.x[0], c.x[3], c.x[2] = float("nan"), float("inf"), float("-inf")
    c.x[1] = 3.0e38
    got = c.check(rt, "missing")
    assert float(got["dx"][0].abs().max()) == 0.0 and float(got["loss"][0]) == 0.0
    c = Case(33, 300, 40, seed=8)
    c.labels[:] = -1
    c.x[:] = float("nan")
    got = c.check(rt, "none left")
    for k in ("loss", "lse", "dx", "dw"):
        assert float(got[k].abs().max()) == 0.0


def test_no_rows(rt):
    c = Case(0, 300, 64, seed=9)
    got = c.run(rt)
    assert got["dw"].shape == (300, 64) and float(got["dw"].abs().max()) == 0.0
    c.untouched()


@pytest.mark.parametrize("amp", [0.0, 60.0, 2000.0])
def test_extreme_logits(rt, amp):
    """Equal logits; a softmax with one token left; logits far beyond what exp takes."""
    c = Case(40, 5000, 64, seed=10, amp=amp)
    c.labels[:20] = (c.x[:20].double() @ c.w.double().t()).argmax(1)
    c.check(rt, f"amplitude {amp}")


def test_a_nan_in_a_row_stays_there(rt):
    c = Case(16, 500, 64, seed=11)
    c.x[5, 3] = float("nan")
    got = c.run(rt)
    rows = [t for t in range(16) if t != 5]
    assert bool(torch.isnan(got["loss"][5])) and bool(torch.isnan(got["dx"][5].float()).all())
    assert bool(torch.isfinite(got["loss"][rows]).all()) and bool(torch.isfinite(got["dx"][rows].float()).all())


@pytest.mark.parametrize("rows,vocab,hidden,top,tau,a,b,layout", [
    (1, 1, 8, 1, 1.0, 0.0, 1.0, "NT"), (1, 300, 64, 7, 2.0, 0.3, 0.7, "NT"), (5, 257, 33, 64, 1.0, 0.0, 2.0, "NN"),
    (64, 1000, 128, 50, 4.0, 0.5, 0.5, "NT"), (130, 4100, 72, 65, 0.5, 0.25, 1.0, "NT"),
    (33, 9000, 64, 256, 2.0, 1.0, 1.0, "NN"), (17, 1500, 64, 1024, 1.0, 0.5, 0.5, "NT"), (300, 520, 96, 3, 3.0, 0.0, 1.0, "NT")])
def test_distill(rt, rows, vocab, hidden, top, tau, a, b, layout):
    Case(rows, vocab, hidden, layout, seed=rows + top).teach(top, tau, a, b).check(rt, f"distill {top} at {tau}")


@pytest.mark.parametrize("half,int32,ldt", [(True, True, 0), (False, True, 12), (True, False, 9)])
def test_teacher_types_and_strides(rt, half, int32, ldt):
    Case(50, 700, 64, seed=12, int32=int32).teach(9, 2.0, 0.5, 0.5, half=half, ldt=ldt).check(rt, "teacher types")


def test_teacher_entries_missing_and_equal(rt):
    c = Case(60, 640, 64, seed=13).teach(40, 2.0, 0.25, 0.75, repeat=True)
    c.tokens[::2, 5:9] = -1
    c.tokens[1::2, 3] = 640
    c.tokens[4, 2] = 2 ** 33 + 1
    c.teacher[::2, 5:9] = float("nan")        # a missing entry's logit is not looked at
    c.teacher[3, 10:20] = float("-inf")       # no probability
    c.teacher[7, :] = float("-inf")           # a row without a teacher
    c.tokens[8, :] = -1
    c.tokens[9, :] = 77                       # one token, forty times
    c.tokens[10, 1:] = -5                     # one entry left
    c.labels[8] = -100                        # neither label nor teacher
    c.x[8] = float("nan")
    c.labels[9], c.labels[11] = 77, c.tokens[11, 0]   # the label is one of the teacher's tokens
    c.check(rt, "entries")
    c = Case(20, 300, 40, seed=14).teach(4)
    c.tokens[:] = -1
    got = c.check(rt, "no teacher left")
    assert float(got["dw"].abs().max()) == 0.0


def test_distill_pieces(rt):
    c = Case(70, 2053, 64, seed=15).teach(90, 2.0, 0.5, 0.5)
    c.check(rt, "distill pieces", max_piece=256)


@pytest.mark.parametrize("teach", [False, True])
def test_gradient_against_differences(rt, teach):
    """Along a direction of +-h the loss's central difference; h and the operands are such that x +- h and
    W +- h are bf16 numbers.  The difference's own error is h^2/6 of the third derivative, at most
    |dz|^3 per row for a log-sum-exp, and the f32 losses' (checked above) over 2h."""
    rows, vocab, hidden, h = 24, 200, 16, 2.0 ** -6
    g = torch.Generator().manual_seed(16)
    c = Case(rows, vocab, hidden, seed=16, dtype="f32", scale=1.0, weights=False)
    c.x = (torch.randint(-31, 32, (rows, hidden), generator=g) / 32.0).bfloat16()
    c.w = (torch.randint(-31, 32, (vocab, hidden), generator=g) / 32.0).bfloat16()
    tau, k = 1.0, 1.0
    if teach:
        tau = 2.0
        c.teach(12, tau, 0.5, 0.5)
        k = 0.5 + 0.5 * tau * tau / tau ** 3
    got = c.run(rt)
    tol_loss = c.define()["loss"][1]
    x, w = c.x.clone(), c.w.clone()
    for name in ("x", "w"):
        base = x if name == "x" else w
        step = torch.where(torch.rand(base.shape, generator=g) < 0.5, -h, h)
        grad = got["d" + name].double()
        losses = []
        for sign in (1, -1):
            moved = (base.double() + sign * step.double()).bfloat16()
            assert bool((moved.double() == base.double() + sign * step.double()).all())
            c.x, c.w = (moved, w) if name == "x" else (x, moved)
            losses.append(c.run(rt)["loss"].double())
        c.x, c.w = x, w
        dz = (step.double() @ w.double().t() if name == "x" else x.double() @ step.double().t()).abs().amax(1)
        third = k * (2 * dz) ** 3 / 6   # dz is the whole step: h is in it
        diff = (losses[0] - losses[1]) / 2
        if name == "x":
            along = (grad * step.double()).sum(1)
            tol = third + tol_loss + 2.0 ** -8 * (grad.abs() * h).sum(1) + 2.0 ** -8 * h * hidden * 2
            assert bool(((along - diff).abs() <= tol).all())
        else:
            along = (grad * step.double()).sum()
            tol = third.sum() + tol_loss.sum() + 2.0 ** -8 * h * 2 * rows * hidden
            assert abs(float(along - diff.sum())) <= float(tol)


def same_again(rt, c, **kw):
    first, again = c.run(rt, **kw), c.run(rt, **kw)
    side = hip_rt.Stream()
    rt.set_stream(side.ptr)
    try:
        other = c.run(rt, **kw)
    finally:
        rt.set_stream(0)
        rt.wait_idle()
        side.destroy()
    for k in first:
        assert torch.equal(first[k], again[k]) and torch.equal(first[k], other[k]), k


def replays(rt, c, other, **kw):
    """Captured after one eager call; replays match it bit for bit, with eager work in between."""
    want = c.run(rt, keep=True, **kw)
    side = hip_rt.Stream()
    rt.set_stream(side.ptr)
    graph = None
    try:
        graph = hip_rt.Graph(side, lambda: c.call(c.desc))
        for _ in range(3):
            c.refill(rt)
            graph.launch(side)
            got = c.read(rt)
            for k in want:
                assert torch.equal(got[k], want[k]), k
            other.check(rt, "between replays")
    finally:
        rt.set_stream(0)
        rt.wait_idle()
        if graph:
            graph.destroy()
        side.destroy()
        c.free(rt)


def test_same_bits_again_and_on_another_stream(rt):
    same_again(rt, Case(200, 3000, 128, seed=17).teach(30, 2.0, 0.5, 0.5), max_piece=1024)


def test_graph_replays(rt):
    replays(rt, Case(96, 2000, 64, seed=18).teach(20, 2.0, 0.5, 0.5), Case(30, 500, 64, seed=19), max_piece=800)


def test_capture_without_scratch_is_refused():
    with t0g.GpuRuntime.new(0) as fresh:
        c = Case(40, 400, 64, seed=20)
        with t0g.GpuRuntime.new(0) as warm:
            want = c.run(warm)
        c.run(warm_up := t0g.GpuRuntime.new(0), keep=True)   # buffers and descriptor; `fresh` has no scratch yet
        side = hip_rt.Stream()
        fresh.set_stream(side.ptr)
        code = []

        def call():
            with pytest.raises(t0g.T0gError) as e:
                fresh.linear_cross_entropy(c.desc)
            code.append((e.value.code, str(e.value)))

        graph = hip_rt.Graph(side, call)
        assert code[0][0] == t0g.ERR_INVALID_ARG and "capture" in code[0][1]
        c.refill(warm_up)
        fresh.linear_cross_entropy(c.desc)   # the handle is as usable as before
        fresh.wait_idle()
        got = c.read(warm_up)
        for k in want:
            assert torch.equal(got[k], want[k]), k
        graph.destroy()
        fresh.set_stream(0)
        side.destroy()
        c.free(warm_up)
        warm_up.close()


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("rows,vocab,hidden,pad,offset,xpad,max_piece", [
    (96, 515, 33, 0, 0, 0, 0), (100, 1003, 65, 3, 1, 2, 0), (130, 777, 127, 1, 0, 0, 256), (100, 515, 1023, 1, 0, 1, 104),
    (256, 515, 33, 0, 0, 0, 0), (300, 1003, 65, 3, 1, 2, 0), (260, 1285, 127, 1, 0, 0, 256), (257, 2051, 200, 5, 0, 0, 768),
    (300, 130, 71, 0, 3, 7, 0), (512, 515, 33, 0, 0, 0, 0), (600, 1003, 65, 3, 1, 2, 0), (513, 1285, 127, 1, 0, 0, 256),
    (520, 2051, 200, 5, 0, 0, 768), (512, 130, 71, 0, 3, 7, 0), (530, 515, 1023, 1, 0, 1, 104)])
def test_copied_weight(rt, rows, vocab, hidden, pad, offset, xpad, max_piece, layout):
    """Rows that are not whole 16-byte pieces; from 512 on the weight is copied (in both forms of the call)."""
    Case(rows, vocab, hidden, layout, seed=rows + vocab, pad=pad, offset=offset, xpad=xpad).check(
        rt, "copied", max_piece=max_piece)


@pytest.mark.parametrize("rows,vocab,hidden,layout,pad,offset,xpad", [
    (5, 600, 64, "NT", 8, 0, 3), (120, 600, 64, "NT", 0, 0, 3), (300, 600, 64, "NT", 0, 1, 0), (300, 601, 63, "NN", 0, 0, 0),
    (300, 600, 63, "NN", 0, 0, 0), (20, 600, 63, "NN", 8, 0, 1),
    (600, 600, 64, "NT", 0, 1, 0), (600, 601, 63, "NN", 0, 0, 0), (600, 601, 63, "NT", 1, 0, 0)])
def test_loss_alone_of_unaligned_operands(rt, rows, vocab, hidden, layout, pad, offset, xpad):
    c = Case(rows, vocab, hidden, layout, seed=27, pad=pad, offset=offset, xpad=xpad, want="")
    c.labels[::3] = -1
    c.x[3] = float("nan")
    c.check(rt, "loss alone")


# ---- sizes around the fused form's tile -------------------------------------------------

FUSED = [(256, 256, 64), (257, 1000, 72), (300, 2049, 136), (256, 131, 64), (513, 1283, 320), (260, 8, 8), (1000, 640, 40)]


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("rows,vocab,hidden", FUSED)
def test_fused_cross_entropy(rt, rows, vocab, hidden, layout):
    Case(rows, vocab, hidden, layout, seed=rows + vocab).check(rt, "fused ce")


@pytest.mark.parametrize("layout,vocab", [("NT", 2307), ("NT", 2304), ("NN", 2304)])
@pytest.mark.parametrize("max_piece", [0, 256, 1000])
def test_fused_pieces(rt, max_piece, layout, vocab):
    """Pieces computed twice and the last, kept one; labels at tiles' and pieces' edges, rows without one."""
    c = Case(300, vocab, 200, layout, seed=21, pad=8)
    edges = [e for v0 in range(0, vocab, 128) for e in (v0, min(v0 + 128, vocab) - 1)]
    for t in range(300):
        c.labels[t] = edges[(5 * t) % len(edges)] if t % 4 else -100
    c.x[4], c.x[8] = float("nan"), float("inf")
    c.check(rt, f"fused pieces of {max_piece}", max_piece=max_piece)


@pytest.mark.parametrize("rows,vocab,hidden,top,tau,a,b,max_piece", [
    (256, 300, 64, 3, 1.0, 0.0, 1.0, 0), (300, 2051, 128, 100, 2.0, 0.5, 0.5, 0), (300, 2051, 128, 100, 2.0, 0.5, 0.5, 512),
    (270, 1100, 64, 1024, 0.5, 0.25, 1.0, 256), (512, 900, 72, 40, 4.0, 1.0, 1.0, 0), (300, 1536, 64, 64, 1.0, 0.5, 0.5, 768)])
def test_fused_distill(rt, rows, vocab, hidden, top, tau, a, b, max_piece):
    """Many entries of a row in one tile among them, equal tokens, missing ones, rows without any."""
    c = Case(rows, vocab, hidden, seed=rows + top).teach(top, tau, a, b, repeat=top > 500)
    c.tokens[::5, top // 2:] = -1
    c.tokens[7] = -1
    c.tokens[9] = torch.randint(0, 100, (top,), generator=c.g)
    if a:
        c.labels[::3] = -100
        c.labels[1] = c.tokens[1, 0]
    c.check(rt, f"fused distill {top} at {tau}", max_piece=max_piece)


@pytest.mark.parametrize("amp", [0.0, 60.0, 2000.0])
@pytest.mark.parametrize("max_piece", [0, 512])
def test_fused_extreme_logits(rt, amp, max_piece):
    c = Case(256, 1500, 64, seed=22, amp=amp)
    c.labels[:128] = (c.x[:128].double() @ c.w.double().t()).argmax(1)
    c.check(rt, f"fused amplitude {amp}", max_piece=max_piece)


def test_fused_nan_in_a_row_stays_there(rt):
    c = Case(300, 1500, 64, seed=23)
    c.x[5, 3] = float("nan")
    got = c.run(rt)
    rows = [t for t in range(300) if t != 5]
    assert bool(torch.isnan(got["loss"][5])) and bool(torch.isnan(got["dx"][5].float()).all())
    assert bool(torch.isfinite(got["loss"][rows]).all()) and bool(torch.isfinite(got["dx"][rows].float()).all())


@pytest.mark.parametrize("want,dtype", [("", "f32"), ("x", "f32"), ("w", "f32"), ("xw", "bf16")])
def test_fused_outputs_asked_for(rt, want, dtype):
    Case(320, 2100, 128, want=want, dtype=dtype, weights=False, scale=1.0, int32=True, c=0.5).check(rt, "fused outputs")


def test_fused_same_bits_again_and_on_another_stream(rt):
    same_again(rt, Case(400, 3000, 128, seed=24).teach(30, 2.0, 0.5, 0.5), max_piece=1024)


def test_fused_graph_replays(rt):
    replays(rt, Case(300, 2000, 64, seed=25).teach(20, 2.0, 0.5, 0.5), Case(260, 500, 64, seed=26), max_piece=768)


@pytest.mark.parametrize("rows,vocab,hidden,want,top", [(160, 54000, 64, "xw", 0), (129, 66001, 40, "x", 0),
                                                          (140, 40000, 64, "", 0), (135, 63000, 64, "xw", 60),
                                                          (2100, 4100, 64, "xw", 300)])
def test_chosen_by_size(rt, form, rows, vocab, hidden, want, top):
    """Sizes at which the choice between the forms lies; a teacher with more tokens than the fused form takes."""
    if form == "rows":
        t0g.set_loss_form(t0g.LOSS_FORM_AUTO)
    c = Case(rows, vocab, hidden, seed=28, want=want, amp=4.0)
    if top:
        c.teach(top, 2.0, 0.5, 0.5)
    c.check(rt, "by size")


@pytest.mark.parametrize("rows,vocab,hidden,layout,dtype,pad,max_piece", [
    (1, 65600, 64, "NT", "bf16", 0, 0), (16, 9100, 470, "NT", "bf16", 2, 0), (17, 9100, 470, "NT", "f32", 0, 0),
    (32, 8200, 520, "NN", "bf16", 0, 0), (31, 65537, 65, "NN", "bf16", 0, 0), (33, 40000, 112, "NT", "f32", 0, 0),
    (64, 66001, 64, "NT", "bf16", 0, 30000), (20, 33000, 136, "NN", "f32", 8, 16000), (64, 8200, 520, "NN", "bf16", 0, 0)])
def test_dw_of_few_rows(rt, rows, vocab, hidden, layout, dtype, pad, max_piece):
    """Weights of at least 2^22 values with few rows, whose dW has a kernel of its own: its row counts, ragged tiles,
    both outputs and stores, and a NaN in an ignored row."""
    c = Case(rows, vocab, hidden, layout, seed=60 + rows, pad=pad, dtype=dtype)
    if rows > 1:
        c.labels[rows // 2] = -100
        c.x[rows // 2, 5] = float("nan")
    c.labels[0] = vocab - 1
    c.check(rt, f"{rows} rows", max_piece=max_piece)


@pytest.mark.parametrize("vocab,top", [(150, 1024), (150, 64), (65, 63), (2, 300), (5000, 257), (40, 62)])
def test_teacher_entries_repeated(rt, vocab, top):
    """Many equal tokens in a row, over all of the sorting's parts; some missing, and the label among them."""
    c = Case(9, vocab, 64, seed=80 + top).teach(top, 2.0, 0.5, 0.5, repeat=True)
    c.tokens[:, ::5] = -1
    c.tokens[1, 1:] = c.tokens[1, 1].clamp(min=0)
    c.tokens[2] = -1
    c.labels[3] = c.tokens[3, 1].clamp(min=0)
    c.check(rt, f"{top} entries of {vocab} tokens")


@pytest.mark.parametrize("rows", [5, 300])
def test_weight_past_32_bits(rt, rows):
    """A weight of 2^31 + 146 M values (4.6 GB), zero but for its last 300 tokens: the logits elsewhere are 0, so the
    definition needs those alone.  G's error is 2^-8 (its bf16) + 0.7 2^-9 (kept exponentials) + 2 e_z and the
    statistics' 2^-14; dW's sums add (rows + 2) u of their magnitudes, dx's (vocab + 2) u, and the outputs are f32."""
    vocab, hidden, live = 140000, 16384, 300
    g = torch.Generator().manual_seed(91)
    x = torch.randn(rows, hidden, generator=g).bfloat16()
    w = (2.0 * hidden ** -0.5 * torch.randn(live, hidden, generator=g)).bfloat16()
    labels = torch.randint(0, vocab, (rows,), generator=g)
    labels[1::2] = torch.randint(vocab - live, vocab, (rows // 2,), generator=g)
    held = []

    def up(t):
        held.append(rt.upload(t.contiguous().view(torch.int16).numpy() if t.dtype == torch.bfloat16 else t.numpy()))
        return held[-1]

    try:
        tail = 2 * hidden * (vocab - live)
        wa = rt.alloc_zero(2 * hidden * vocab)
        held.append(wa)
        rt.write(wa + tail, w.view(torch.int16).numpy())
        sizes = {"loss": 4 * rows, "dx": 4 * rows * hidden, "dw": 4 * vocab * hidden}
        out = {k: rt.alloc(n) for k, n in sizes.items()}
        held += out.values()
        _log(f"{rows} rows")
        rt.linear_cross_entropy(t0g.linear_ce_desc(up(x), wa, up(labels), out["loss"], rows, vocab, hidden, dx=out["dx"],
                                                   dw=out["dw"], dx_dtype=t0g.F32, dw_dtype=t0g.F32))
        rt.wait_idle()
        first = vocab - live
        xd, wd = x.double(), w.double()
        z = xd @ wd.t()
        lse = torch.log(torch.exp(z).sum(1) + first)
        mag = xd.abs() @ wd.abs().t()
        ez = float((hidden + 2) * U * mag.max())
        rel = 2.0 ** -8 + 0.7 * 2.0 ** -9 + 2 * ez + 2.0 ** -14
        in_tail = labels >= first
        zy = torch.where(in_tail, z[torch.arange(rows), (labels - first).clamp(min=0)], torch.zeros(rows, dtype=torch.float64))
        loss = torch.from_numpy(rt.read(out["loss"], (rows,), "float32").copy()).double()
        assert float((loss - (lse - zy)).abs().max()) <= 2 * ez + 2.0 ** -14 + 16 * U * 20
        p = torch.exp(z - lse[:, None])
        tail_labels = torch.zeros_like(p)
        tail_labels[in_tail, (labels - first)[in_tail]] = 1.0
        grad, size = p - tail_labels, p + tail_labels
        dx = torch.from_numpy(rt.read(out["dx"], (rows, hidden), "float32").copy()).double()
        bound = (rel + (vocab + 2) * U) * (size @ wd.abs())
        assert bool(((dx - grad @ wd).abs() <= bound).all())
        dw = torch.from_numpy(rt.read(out["dw"] + 4 * hidden * first, (live, hidden), "float32").copy()).double()
        bound = (rel + (rows + 2) * U) * (size.t() @ xd.abs())
        assert bool(((dw - grad.t() @ xd).abs() <= bound).all())
        for v in (0, 65537, 131071, 131072, first - 1, int(labels[0])):
            hit = (labels == v).double()
            gv = torch.exp(-lse) - hit
            got = torch.from_numpy(rt.read(out["dw"] + 4 * hidden * v, (hidden,), "float32").copy()).double()
            if v < first:
                assert bool(((got - gv @ xd).abs() <= (rel + (rows + 2) * U) * ((torch.exp(-lse) + hit) @ xd.abs())).all()), v
    finally:
        rt.wait_idle()
        for a in held:
            rt.free(a)


# ---- weights, temperatures and masks beyond the usual ones ------------------------------

@pytest.mark.parametrize("rows,vocab,hidden,top,tau,a,b,max_piece", [
    (1, 40, 16, 1, 1.0, 1.0, -1.0, 0), (5, 300, 64, 7, 1.0, 1.0, -1.0, 0), (140, 17000, 64, 9, 1.0, -0.5, 0.5, 0),
    (40, 1003, 64, 70, 1.0, 2.0, -2.0, 256), (300, 2051, 72, 20, 1.0, 1.0, -1.0, 0), (300, 2051, 72, 90, 1.0, -1.0, 1.0, 512),
    (300, 700, 64, 12, 2.0, 1.0, -0.5, 0)])
def test_weights_that_cancel(rt, rows, vocab, hidden, top, tau, a, b, max_piece):
    """Of labels and teacher with one softmax: the dense parts of the gradient cancel, G = rate a (Q - onehot) remains."""
    c = Case(rows, vocab, hidden, seed=100 + rows + top).teach(top, tau, a, b)
    if rows > 3:
        c.labels[2] = -100
        c.tokens[3] = -1
    c.check(rt, f"weights {a} and {b}", max_piece=max_piece)


@pytest.mark.parametrize("max_piece", [0, 512])
@pytest.mark.parametrize("amp,tau", [(30.0, 20.0), (60.0, 50.0), (60.0, 4.5), (60.0, 4.0), (4.0, 0.1), (4.0, 0.4)])
def test_temperatures_on_wide_logits(rt, amp, tau, max_piece):
    """Tokens far below the others, which the labels' softmax has lost and the teacher's at its temperature has not, and
    a temperature that sharpens.  (1500 tokens: a dW column is the sum of few rows' gradients.)"""
    c = Case(300, 1500, 64, seed=int(10 * tau), amp=amp).teach(20, tau, 0.5, 0.5)
    c.labels[:100] = (c.x[:100].double() @ c.w.double().t()).argmax(1)
    c.check(rt, f"amplitude {amp} at {tau}", max_piece=max_piece)


@pytest.mark.parametrize("value", [-float("inf"), -3.3895313892515355e38])
@pytest.mark.parametrize("rows,vocab,taught,max_piece", [
    (4, 2051, False, 0), (4, 2051, True, 256), (40, 20000, False, 0), (40, 20000, True, 0),
    (300, 2051, False, 0), (300, 2051, True, 0), (300, 2051, False, 256), (300, 2051, True, 512)])
def test_tokens_masked_by_a_bias(rt, rows, vocab, taught, max_piece, value):
    """The first hidden value is 1 and the weight's first column a bias that is -infinity or the type's lowest
    value for most of the vocabulary, whole blocks, chunks and pieces of it: as if those tokens were not there.  An
    infinite weight has no dx (0 times infinity)."""
    hidden = 64
    c = Case(rows, vocab, hidden, seed=120 + rows, want="w" if value == -float("inf") else "xw")
    seen = torch.cat([torch.arange(300, 500), torch.arange(1100, 1160), torch.tensor([vocab - 1])])
    few = Case(rows, len(seen), hidden, seed=121 + rows, want=c.want)
    c.x[:, 0], c.w[:, 0] = 1.0, 0.0
    few.x, few.w, few.dloss = c.x, c.w[seen].clone(), c.dloss
    if taught:
        few.teach(12, 2.0, 0.5, 0.5)
        c.teach(12, 2.0, 0.5, 0.5)
        c.tokens, c.teacher = seen[few.tokens], few.teacher
    c.labels = seen[few.labels]
    hidden_tokens = torch.ones(vocab, dtype=torch.bool)
    hidden_tokens[seen] = False
    c.w[hidden_tokens, 0] = value
    got = c.run(rt, max_piece=max_piece)
    c.untouched()
    assert not bool(got["dw"][hidden_tokens].double().abs().any())
    got["dw"] = got["dw"][seen]
    for k, (v, tol) in few.define().items():
        worst = float(((got[k].double() - v).abs() / tol).max())
        _log(f"[loss] masked {rows}x{vocab} {k}: {worst:.3f} of the bound")
        assert bool(((got[k].double() - v).abs() <= tol).all()), k


def test_a_graph_outlives_a_larger_scratch(form):
    """A captured call's scratch stays when a larger call takes a larger one, twice: replays give the eager
    bits, with buffers of every size taken and filled in between."""
    size = t0g.linear_loss_scratch_size
    with t0g.GpuRuntime.new(0) as fresh:
        c = Case(300, 2000, 64, seed=140).teach(20, 2.0, 0.5, 0.5)
        want = c.run(fresh, keep=True)
        side = hip_rt.Stream()
        fresh.set_stream(side.ptr)
        graph, last = None, size(c.desc)
        try:
            graph = hip_rt.Graph(side, lambda: c.call(c.desc))
            for rows, vocab in ((400, 6000), (500, 20000)):
                larger = Case(rows, vocab, 72, seed=rows)
                larger.check(fresh, "larger call after a capture")
                assert size(larger.desc) > last + (1 << 20)
                filled = [fresh.alloc(n) for n in (last, last, last // 2, last // 4)]
                for addr, n in zip(filled, (last, last, last // 2, last // 4)):
                    fresh.memset(addr, 0xFF, n)
                last = size(larger.desc)
                for _ in range(2):
                    c.refill(fresh)
                    graph.launch(side)
                    got = c.read(fresh)
                    for k in want:
                        assert torch.equal(got[k], want[k]), k
                    larger.check(fresh, "between replays")
                for addr in filled:
                    fresh.free(addr)
        finally:
            fresh.set_stream(0)
            fresh.wait_idle()
            if graph:
                graph.destroy()
            side.destroy()
            c.free(fresh)


@pytest.mark.parametrize("rows,vocab,hidden,layout,want", [
    (5, 140000, 16385, "NT", "xw"), (5, 140001, 16384, "NT", "x"), (130, 140001, 16384, "NT", ""),
    (5, 140001, 16384, "NN", "xw"), (140, 131080, 16385, "NN", "xw"), (2, 131080, 16385, "NN", "")])
def test_weight_past_31_bits_of_unaligned_operands(rt, rows, vocab, hidden, layout, want):
    """Weights of 2^31 values and more of which some product's operands are not whole 16-byte pieces.  Zero but for the
    last 200 tokens, the definition and the bounds as in test_weight_past_32_bits."""
    live = 200
    first = vocab - live
    nt = layout == "NT"
    g = torch.Generator().manual_seed(rows + vocab)
    x = torch.randn(rows, hidden, generator=g).bfloat16()
    w = (2.0 * hidden ** -0.5 * torch.randn(live, hidden, generator=g)).bfloat16()
    labels = torch.randint(0, vocab, (rows,), generator=g)
    labels[1::2] = torch.randint(first, vocab, (rows // 2,), generator=g)
    held = []

    def up(t):
        held.append(rt.upload(t.contiguous().view(torch.int16).numpy() if t.dtype == torch.bfloat16 else t.numpy()))
        return held[-1]

    try:
        wa = rt.alloc_zero(2 * hidden * vocab)
        held.append(wa)
        if nt:
            rt.write(wa + 2 * hidden * first, w.view(torch.int16).numpy())
        else:
            columns = w.t().contiguous().view(torch.int16).numpy()
            for h in range(hidden):
                rt.write(wa + 2 * (h * vocab + first), columns[h])
        out = {"loss": rt.alloc(4 * rows), "dx": rt.alloc(4 * rows * hidden) if "x" in want else 0,
               "dw": rt.alloc(4 * vocab * hidden) if "w" in want else 0}
        held += [a for a in out.values() if a]
        _log(f"{rows}x{vocab}x{hidden} {layout} {want}")
        rt.linear_cross_entropy(t0g.linear_ce_desc(up(x), wa, up(labels), out["loss"], rows, vocab, hidden, transpose=layout,
                                                   dx=out["dx"], dw=out["dw"], dx_dtype=t0g.F32, dw_dtype=t0g.F32))
        rt.wait_idle()
        xd, wd = x.double(), w.double()
        z = xd @ wd.t()
        lse = torch.log(torch.exp(z).sum(1) + first)
        ez = float((hidden + 2) * U * (xd.abs() @ wd.abs().t()).max())
        rel = 2.0 ** -8 + 0.7 * 2.0 ** -9 + 2 * ez + 2.0 ** -14
        in_tail = labels >= first
        zy = torch.where(in_tail, z[torch.arange(rows), (labels - first).clamp(min=0)], torch.zeros(rows, dtype=torch.float64))
        loss = torch.from_numpy(rt.read(out["loss"], (rows,), "float32").copy()).double()
        assert float((loss - (lse - zy)).abs().max()) <= 2 * ez + 2.0 ** -14 + 16 * U * 20
        p = torch.exp(z - lse[:, None])
        tail_labels = torch.zeros_like(p)
        tail_labels[in_tail, (labels - first)[in_tail]] = 1.0
        grad, size = p - tail_labels, p + tail_labels
        if "x" in want:
            dx = torch.from_numpy(rt.read(out["dx"], (rows, hidden), "float32").copy()).double()
            assert bool(((dx - grad @ wd).abs() <= (rel + (vocab + 2) * U) * (size @ wd.abs())).all())
        if "w" not in want:
            return
        # tokens, or hidden columns, of dW at its ends, inside and where a piece or a tile may end
        for i in (0, 1, 255, 256, 8191, 16383) + ((131071, first - 1, int(labels[0]), vocab - 2, vocab - 1) if nt else (hidden - 1,)):
            n = hidden if nt else vocab
            got = torch.from_numpy(rt.read(out["dw"] + 4 * n * i, (n,), "float32").copy()).double()
            if nt:
                hit = (labels == i).double()
                pi = p[:, i - first] if i >= first else torch.exp(-lse)
                want_row, mag = (pi - hit) @ xd, (pi + hit) @ xd.abs()
            else:
                dense = (torch.exp(-lse) * xd[:, i]).sum()
                want_row, mag = torch.full((vocab,), float(dense), dtype=torch.float64), torch.exp(-lse) @ xd.abs()[:, i]
                mag = torch.full((vocab,), float(mag), dtype=torch.float64)
                want_row[first:], mag[first:] = p.t() @ xd[:, i], p.t() @ xd.abs()[:, i]
                want_row.index_add_(0, labels, -xd[:, i])
                mag.index_add_(0, labels, xd.abs()[:, i])
            assert bool(((got - want_row).abs() <= (rel + (rows + 2) * U) * mag).all()), i
    finally:
        rt.wait_idle()
        for a in held:
            rt.free(a)


def test_hidden_states_past_31_bits(rt):
    """300000 rows of 8192 (4.9 GB), zero but for ten of them around where byte and element offsets pass 31 and 32 bits,
    over a vocabulary narrower than a tile.  Of a zero row the logits are 0 and G = rate (1/V - onehot); bounds as in
    test_weight_past_32_bits, and dx is rounded to bf16."""
    rows, vocab, hidden = 300000, 232, 8192
    g = torch.Generator().manual_seed(150)
    live = torch.tensor([0, 1, 5, 131071, 131072, 262143, 262144, 262145, 299998, 299999])
    x = torch.randn(len(live), hidden, generator=g).bfloat16()
    w = (2.0 * hidden ** -0.5 * torch.randn(vocab, hidden, generator=g)).bfloat16()
    labels = torch.randint(0, vocab, (rows,), generator=g)
    held = []

    def up(t):
        held.append(rt.upload(t.contiguous().view(torch.int16).numpy() if t.dtype == torch.bfloat16 else t.numpy()))
        return held[-1]

    try:
        xa = rt.alloc_zero(2 * rows * hidden)
        held.append(xa)
        for i, row in zip(live.tolist(), x):
            rt.write(xa + 2 * hidden * i, row.view(torch.int16).numpy())
        loss, dx, dw = rt.alloc(4 * rows), rt.alloc(2 * rows * hidden), rt.alloc(4 * vocab * hidden)
        held += [loss, dx, dw]
        _log("300000x232x8192")
        rt.linear_cross_entropy(t0g.linear_ce_desc(xa, up(w), up(labels), loss, rows, vocab, hidden, dx=dx, dw=dw,
                                                   dw_dtype=t0g.F32))
        rt.wait_idle()
        xd, wd = x.double(), w.double()
        z = xd @ wd.t()
        ez = float((hidden + 2) * U * (xd.abs() @ wd.abs().t()).max())
        rel = 2.0 ** -8 + 0.7 * 2.0 ** -9 + 2 * ez + 2.0 ** -14
        want = torch.full((rows,), float(torch.log(torch.tensor(float(vocab), dtype=torch.float64))), dtype=torch.float64)
        want[live] = torch.logsumexp(z, 1) - z.gather(1, labels[live][:, None])[:, 0]
        got = torch.from_numpy(rt.read(loss, (rows,), "float32").copy()).double()
        assert float((got - want).abs().max()) <= 2 * ez + 2.0 ** -14 + 16 * U * 20
        onehot = torch.nn.functional.one_hot(labels[live], vocab).double()
        p = torch.softmax(z, 1)
        grad, size = p - onehot, p + onehot
        dwd = torch.from_numpy(rt.read(dw, (vocab, hidden), "float32").copy()).double()
        assert bool(((dwd - grad.t() @ xd).abs() <= (rel + (rows + 2) * U) * (size.t() @ xd.abs())).all())
        for i in live.tolist() + [2, 131073, 262146, 270000, 299997]:
            at = (live == i).nonzero()
            dense = p[at[0, 0]] if len(at) else torch.full((vocab,), 1.0 / vocab, dtype=torch.float64)
            hit = torch.nn.functional.one_hot(labels[i], vocab).double()
            v, mag = (dense - hit) @ wd, (dense + hit) @ wd.abs()
            e = (rel + (vocab + 2) * U) * mag
            got = torch.from_numpy(rt.read(dx + 2 * hidden * i, (hidden,), "int16").copy()).view(torch.bfloat16).double()
            assert bool(((got - v).abs() <= e + 2.0 ** -8 * (v.abs() + e)).all()), i
    finally:
        rt.wait_idle()
        for a in held:
            rt.free(a)
