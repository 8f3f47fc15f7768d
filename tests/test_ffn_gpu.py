"""The feed-forward layer's operators (t0g_rms_norm, t0g_fp8_quantize, t0g_fp8_gemm, t0g_gated_linear and their
gradients) against their definitions in 64 bits, at sizes, strides, types and values where they can go wrong;
gradients also against differences.

Tolerances, with u = 2^-24 (f32), half a unit of bf16 2^-8 and of e4m3 / e5m2 2^-4 / 2^-3, relative:
  norm      the sum of squares goes through at most 64 f32 roundings (a thread's values, its row of 16 lanes, the
            wave's four, the workgroup's waves); quotient, root, reciprocal and the products around them 8 more
  8 bits    a value is off by half a unit of its type, and by what moves it over a border: 2^-20 of itself
  products  exact in f32, summed in f32; a matrix unit may cut instead of round, 2 u a term and a join
            8-bit ones for a bf16 result: 7 of each 8 neighbouring products lose at most 2^-13 of the eighth's
            power of two, which is at most the product of the largest of the 8 values of A and of B
  act       exponential and reciprocal within 2^-22 each: 2^-20 of the activation with the products around them
"""
import pytest
import torch   # on the host only: the device's buffers and streams are the library's runtime's

import hip_rt
import t0g

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
TYPES = {torch.float32: t0g.F32, torch.bfloat16: t0g.BF16, torch.float8_e4m3fn: t0g.E4M3, torch.float8_e5m2: t0g.E5M2}
MOST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
BF16, F32, E4, E5 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e5m2


@pytest.fixture(scope="module")
def rt():
    r = t0g.GpuRuntime.new(0)
    yield r
    r.close()


def raw(t):
    size = t.element_size()
    return (t.view(torch.uint8) if size == 1 else t.view(torch.int16) if size == 2 else t).numpy()


class Bufs:
    """Device copies of host arrays, each in a filled allocation of its own, `offset` elements from an aligned address and
    rows `pad` elements further apart than packed: a write outside shows, and what lies between rows is not a number."""

    def __init__(self, rt, pad=0, offset=0):
        self.rt, self.pad, self.offset, self.held, self.outs = rt, pad, offset, [], {}

    def _place(self, t, ld, fill):
        rows, cols = t.shape
        image = torch.full((self.offset + rows * ld + 64,), fill, dtype=torch.float32).to(t.dtype)
        view = image[self.offset:self.offset + rows * ld].view(rows, ld)[:, :cols]
        view.copy_(t)
        addr = self.rt.upload(raw(image))
        self.held.append(addr)
        return addr, image, view

    def inp(self, t, packed=False):
        """(address, leading dimension)"""
        if t is None:
            return 0, 0
        if t.dim() == 1:
            t = t[None, :]
        ld = t.shape[1] + (0 if packed else self.pad)
        addr, image, _ = self._place(t, ld, float("nan"))
        return addr + self.offset * image.element_size(), ld

    def out(self, name, shape, dtype, packed=False):
        rows, cols = shape
        ld = cols + (0 if packed else self.pad)
        self.outs[name] = self._place(torch.full((rows, cols), -7.0, dtype=torch.float32).to(dtype), ld, -7.0)
        return self.outs[name][0] + self.offset * self.outs[name][1].element_size(), ld

    def read(self, free=True):
        """The outputs; what surrounds them must be as it was."""
        got = {}
        for name, (addr, image, view) in self.outs.items():
            r = raw(image)
            r[:] = self.rt.read(addr, r.shape, r.dtype)
            got[name] = view.clone()
            copy = image.clone()
            rows, cols = view.shape
            ld = view.stride(0)
            copy[self.offset:self.offset + rows * ld].view(rows, ld)[:, :cols] = torch.full((1,), -7.0).to(image.dtype)
            assert bool((copy.float() == -7.0).all()), f"{name}: written outside"
        if free:
            for a in self.held:
                self.rt.free(a)
        return got


def near(got, want, bound, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    off = torch.where(torch.isnan(want), torch.zeros_like(want), (got - want).abs() - bound)
    at = int(off.argmax())
    assert float(off.max()) <= 0, (f"{what}: off by {float((got - want).abs().flatten()[at]):.3g} at {at}, "
                                   f"{float(got.flatten()[at]):.6g} for {float(want.flatten()[at]):.6g}")


def blocks(n):
    return (n + 127) // 128


def scales_of(v, dtype, tile=False):
    """[blocks of columns][rows, or blocks of rows] of v in 64 bits."""
    rows, cols = v.shape
    high = 128 if tile else 1
    p = torch.zeros((-(-rows // high) * high, blocks(cols) * 128), dtype=torch.float64)
    p[:rows, :cols] = v
    return (p.reshape(-1, high, blocks(cols), 128).abs().amax(dim=(1, 3)).clamp(min=2.0 ** -100) / MOST[dtype]).t()


def spread(s, shape, tile=False):
    """Each value's scale."""
    s = s.t().repeat_interleave(128, dim=1)[:, :shape[1]]
    return s.repeat_interleave(128, dim=0)[:shape[0]] if tile else s


def check_f8(q, scales, v, dtype, tile=False, slack=0.0, what=""):
    """q and its scales against v in 64 bits, itself off by at most `slack` of itself."""
    want = scales_of(v, dtype, tile)
    near(scales, want, (slack + 4 * U) * want, f"{what}: scales")
    units = v / spread(want, v.shape, tile)
    d = slack + 2.0 ** -20
    # the type's rounding does not fall: it lies between those of the ends of what the value may be
    lo, hi = ((units * (1 + s * d * units.sign())).float().clamp(-MOST[dtype], MOST[dtype]).to(dtype).double() for s in (-1, 1))
    got = q.double()
    assert bool(((got >= lo) & (got <= hi)).all()), f"{what}: a value is rounded to another neighbour"


def data(g, rows, cols, dtype=BF16, scale=1.0):
    return (torch.randn(rows, cols, generator=g) * scale).to(dtype)


# ---- the norm ---------------------------------------------------------------------------
NORM_REL = 72 * U


def norm_of(x, r, w, offset, eps):
    s = x.double() + (r.double() if r is not None else 0.0)
    rho = (s.square().mean(1, keepdim=True) + eps) ** -0.5
    return s, rho, s * rho * ((w.double() + offset) if w is not None else 1.0)


@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (2, 64), (5, 127), (4, 128), (3, 129), (2, 512), (3, 513), (2, 1000),
                                         (3, 2048), (2, 2049), (2, 3001), (2, 3000), (2, 12001), (2, 12000), (300, 1023), (2, 4096), (3, 4097), (2, 8192), (2, 8193), (2, 16383),
                                         (1, 16384)])
@pytest.mark.parametrize("xt,rt_,wt,yt", [(BF16, BF16, BF16, BF16), (F32, F32, F32, F32), (BF16, F32, F32, BF16), (F32, None, None, F32)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1)])
def test_norm(rt, rows, hidden, xt, rt_, wt, yt, pad, offset):
    g = torch.Generator().manual_seed(rows + hidden)
    x = data(g, rows, hidden, xt, 2.0)
    r = data(g, rows, hidden, rt_, 2.0) if rt_ else None
    w = data(g, 1, hidden, wt)[0] if wt else None
    woff, eps, st, qt = (1.0 if wt == F32 else 0.0), 1e-5, rt_ or xt, E4 if xt == BF16 else E5
    b = Bufs(rt, pad, offset)
    (xa, ldx), (ra, ldr), (wa, _) = b.inp(x), b.inp(r), b.inp(w, True)
    (sa, lds), (ya, ldy) = b.out("sum", x.shape, st), b.out("y", x.shape, yt)
    (qa, ldq), (ca, ldsc) = b.out("q", x.shape, qt), b.out("scales", (blocks(hidden), rows), F32)
    rt.rms_norm(t0g.rms_norm_desc(
        xa, wa, rows, hidden, eps=eps, residual=ra, sum=sa, y=ya, q=qa, scales=ca, weight_offset=woff, ldx=ldx, ldr=ldr, ldsum=lds,
        ldy=ldy, ldq=ldq, ldsc=ldsc, x_dtype=TYPES[xt], residual_dtype=TYPES[rt_ or BF16], weight_dtype=TYPES[wt or BF16],
        sum_dtype=TYPES[st], y_dtype=TYPES[yt], q_dtype=TYPES[qt]))
    got = b.read()
    s, _, y = norm_of(x, r, w, woff, eps)
    near(got["sum"], s, (HALF[st] + U) * s.abs() + U * x.double().abs(), "sum")
    # where x and residual cancel in f32 the sum is off by a unit of the larger; the bound on y follows it
    lost = U * (x.double().abs() / s.abs().clamp(min=1e-300)).clamp(max=1e6) if rt_ == F32 else torch.zeros_like(s)
    near(got["y"], y, (HALF[yt] + NORM_REL + lost) * y.abs(), "y")
    if rt_ != F32:
        check_f8(got["q"], got["scales"], y, qt, slack=NORM_REL, what="q")


@pytest.mark.parametrize("how", ["sum is x", "sum is residual", "y is x"])
@pytest.mark.parametrize("hidden", [100, 4096, 16000])
def test_norm_in_place(rt, how, hidden):
    g = torch.Generator().manual_seed(hidden)
    x, r, w = data(g, 7, hidden), data(g, 7, hidden), data(g, 1, hidden)[0]
    b = Bufs(rt)
    (xa, _), (ra, _), (wa, _) = b.inp(x), b.inp(r), b.inp(w, True)
    ya, _ = b.out("y", x.shape, BF16)
    y, s = (xa, 0) if how == "y is x" else (ya, xa if how == "sum is x" else ra)
    rt.rms_norm(t0g.rms_norm_desc(xa, wa, 7, hidden, residual=ra, y=y, sum=s))
    sums, _, want = norm_of(x, r, w, 0.0, 1e-6)
    got_y = torch.from_numpy(rt.read(y, (7, hidden), "int16")).view(BF16)
    near(got_y, want, (2.0 ** -8 + NORM_REL) * want.abs(), how)
    if s:
        near(torch.from_numpy(rt.read(s, (7, hidden), "int16")).view(BF16), sums, 2.0 ** -8 * sums.abs(), how)
    for a in b.held:
        rt.free(a)


def test_norm_of_zeros_infinities_and_nan(rt):
    """Rows of zeros give zeros (and their blocks the least scale); an infinity or a NaN spoils its own row only."""
    x = torch.ones(4, 300)
    x[0], x[1, 5], x[2, 290] = 0.0, float("inf"), float("nan")
    b = Bufs(rt)
    (xa, _), (ya, _), (qa, _) = b.inp(x.bfloat16()), b.out("y", x.shape, F32), b.out("q", x.shape, E4)
    ca, _ = b.out("scales", (3, 4), F32)
    rt.rms_norm(t0g.rms_norm_desc(xa, 0, 4, 300, y=ya, q=qa, scales=ca, y_dtype=t0g.F32))
    got = b.read()
    assert bool((got["y"][0] == 0).all() and (got["q"][0].float() == 0).all())
    assert bool((got["scales"][:, 0] == torch.tensor(2.0 ** -100) / 448.0).all())
    assert bool(torch.isnan(got["y"][1, 5]) and torch.isnan(got["y"][2]).all())
    assert bool(((got["y"][3] - 1).abs() < 1e-5).all() and torch.isfinite(got["q"][3].float()).all())
    stands = got["q"].float() * got["scales"].t().repeat_interleave(128, dim=1)[:, :300]
    assert bool(torch.isnan(stands[1, :128]).all() and torch.isnan(stands[2]).all())


@pytest.mark.parametrize("rows,hidden", [(1, 1), (2, 5), (3, 64), (1, 129), (4, 512), (700, 300), (1500, 2047), (3, 3001), (3, 3000), (3, 4096), (3, 4100),
                                         (2, 12001), (2, 12000), (5, 8192), (2, 8195), (515, 16384)])
@pytest.mark.parametrize("xt,yt,wt,st", [(BF16, BF16, BF16, BF16), (F32, F32, F32, F32), (F32, BF16, None, None), (BF16, F32, F32, F32)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (5, 1)])
def test_norm_backward(rt, rows, hidden, xt, yt, wt, st, pad, offset):
    if rows * hidden > 1 << 22 and (pad, yt) != (0, BF16):
        pytest.skip("the large size in two forms")
    g = torch.Generator().manual_seed(rows * 3 + hidden)
    x, dy = data(g, rows, hidden, xt, 2.0), data(g, rows, hidden, yt)
    w = data(g, 1, hidden, wt)[0] if wt else None
    ds = data(g, rows, hidden, st) if st else None
    woff, eps = (1.0 if wt == F32 else 0.0), 1e-5
    dwt = F32 if yt == BF16 else BF16
    b = Bufs(rt, pad, offset)
    (ya, ldy), (xa, ldx), (wa, _), (sa, lds) = b.inp(dy), b.inp(x), b.inp(w, True), b.inp(ds)
    (dxa, lddx), (dwa, _) = b.out("dx", x.shape, xt), b.out("dw", (1, hidden), dwt, True)
    d = t0g.rms_norm_backward_desc(
        ya, xa, wa, rows, hidden, eps=eps, dsum=sa, dx=dxa, dw=dwa, weight_offset=woff, lddy=ldy, ldx=ldx, ldds=lds, lddx=lddx,
        dy_dtype=TYPES[yt], x_dtype=TYPES[xt], weight_dtype=TYPES[wt or BF16], dsum_dtype=TYPES[st or BF16], dx_dtype=TYPES[xt],
        dw_dtype=TYPES[dwt])
    rt.rms_norm_backward(d)
    got = b.read()
    s, rho, _ = norm_of(x, None, None, 0.0, eps)
    n, gr = s * rho, dy.double() * ((w.double() + woff) if w is not None else 1.0)
    add = ds.double() if ds is not None else torch.zeros_like(s)
    want = rho * (gr - n * (gr * n).mean(1, keepdim=True)) + add
    size = rho * (gr.abs() + n.abs() * (gr * n).abs().mean(1, keepdim=True)) + add.abs()
    near(got["dx"], want, HALF[xt] * want.abs() + 2 * NORM_REL * size, "dx")
    each = dy.double() * n
    dw, size = each.sum(0, keepdim=True), each.abs().sum(0, keepdim=True)
    near(got["dw"], dw, HALF[dwt] * dw.abs() + (NORM_REL + (rows + 34) * U) * size, "dw")


def test_norm_backward_against_differences(rt):
    """(L(x + h e) - L(x - h e)) / 2 h of L = sum dy y(x), in 64 bits; curvature and the call's own rounding within 1e-4."""
    g = torch.Generator().manual_seed(3)
    x, dy, w = data(g, 2, 40, F32), data(g, 2, 40, F32), data(g, 1, 40, F32)[0]
    b = Bufs(rt)
    (ya, _), (xa, _), (wa, _) = b.inp(dy), b.inp(x), b.inp(w, True)
    (dxa, _), (dwa, _) = b.out("dx", x.shape, F32), b.out("dw", (1, 40), F32)
    f = t0g.F32
    rt.rms_norm_backward(t0g.rms_norm_backward_desc(ya, xa, wa, 2, 40, dx=dxa, dw=dwa, dy_dtype=f, x_dtype=f, weight_dtype=f, dx_dtype=f))
    got = b.read()
    loss = lambda x, w: (dy.double() * norm_of(x, None, w, 0.0, 1e-6)[2]).sum()   # noqa: E731
    for i in range(0, 40, 7):
        h = torch.zeros(2, 40, dtype=torch.float64)
        h[1, i] = 1e-5
        assert abs((loss(x.double() + h, w) - loss(x.double() - h, w)) / 2e-5 - got["dx"][1, i]) < 1e-4
        assert abs((loss(x, w.double() + h[1]) - loss(x, w.double() - h[1])) / 2e-5 - got["dw"][0, i]) < 1e-4


@pytest.mark.parametrize("alias", ["dy", "x", "dsum"])
def test_norm_backward_in_place(rt, alias):
    g = torch.Generator().manual_seed(9)
    x, dy, ds, w = data(g, 600, 1000), data(g, 600, 1000), data(g, 600, 1000), data(g, 1, 1000)[0]
    got = []
    for own in (True, False):
        b = Bufs(rt)
        (ya, _), (xa, _), (sa, _), (wa, _) = b.inp(dy), b.inp(x), b.inp(ds), b.inp(w, True)
        (dxa, _), (dwa, _) = b.out("dx", x.shape, BF16), b.out("dw", (1, 1000), F32)
        to = dxa if own else {"dy": ya, "x": xa, "dsum": sa}[alias]
        rt.rms_norm_backward(t0g.rms_norm_backward_desc(ya, xa, wa, 600, 1000, dsum=sa, dx=to, dw=dwa))
        got.append((rt.read(to, (600, 1000), "int16"), rt.read(dwa, (1000,), "int32")))
        for a in b.held:
            rt.free(a)
    assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all()


# ---- 8 bits -----------------------------------------------------------------------------
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 64), (3, 127), (16, 128), (5, 129), (127, 200), (128, 256), (129, 255), (130, 4097),
                                       (7, 11008), (1000, 72)])
@pytest.mark.parametrize("xt,qt", [(BF16, E4), (F32, E5), (F32, E4)])
@pytest.mark.parametrize("block,want", [("row", "q"), ("row", "q qt"), ("row", "qt"), ("tile", "q"), ("tile", "q qt"), ("tile", "qt")])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1)])
def test_quantize(rt, rows, cols, xt, qt, block, want, pad, offset):
    g = torch.Generator().manual_seed(rows * 7 + cols)
    tile = block == "tile"
    x = data(g, rows, cols, F32, 3.0) * torch.exp(2.0 * torch.randn(rows, 1, generator=g))
    if rows > 2:
        x[rows // 2] = 0.0
    x = x.to(xt)
    b = Bufs(rt, pad, offset)
    xa, ldx = b.inp(x)
    kw = {"q": 0, "scales": 0}
    if "q" in want.split():
        kw["q"], kw["ldq"] = b.out("q", (rows, cols), qt)
        kw["scales"], kw["ldsc"] = b.out("scales", (blocks(cols), blocks(rows) if tile else rows), F32)
    if "qt" in want.split():
        kw["qt"], kw["ldqt"] = b.out("qt", (cols, rows), qt)
        kw["scales_t"], kw["ldsct"] = b.out("scales_t", (blocks(rows), blocks(cols) if tile else cols), F32)
    q, scales = kw.pop("q"), kw.pop("scales")
    rt.fp8_quantize(t0g.fp8_quantize_desc(xa, q, scales, rows, cols, ldx=ldx, x_dtype=TYPES[xt], q_dtype=TYPES[qt],
                                          block=t0g.BLOCK_TILE if tile else t0g.BLOCK_ROW, **kw))
    got = b.read()
    if "q" in got:
        check_f8(got["q"], got["scales"], x.double(), qt, tile, what="q")
    if "qt" in got:
        check_f8(got["qt"], got["scales_t"], x.double().t(), qt, tile, what="qt")


def test_quantize_of_extremes(rt):
    """The type's largest magnitudes, subnormal inputs, and blocks with an infinity or a NaN."""
    x = torch.zeros(5, 256)
    x[0, 0], x[0, 1] = 3.3895313892515355e38, -3.3895313892515355e38
    x[1, :4] = torch.tensor([1e-38, -1e-39, 2.0 ** -133, 0.0])
    x[2, 130], x[3, 3], x[4, 200] = float("inf"), float("nan"), -1.0
    for qt in (E4, E5):
        b = Bufs(rt)
        (xa, _), (qa, _), (ca, _) = b.inp(x.bfloat16()), b.out("q", x.shape, qt), b.out("scales", (2, 5), F32)
        rt.fp8_quantize(t0g.fp8_quantize_desc(xa, qa, ca, 5, 256, q_dtype=TYPES[qt]))
        got = b.read()
        stands = got["q"].float() * got["scales"].t().repeat_interleave(128, dim=1)
        assert float(got["q"][0, 0]) == MOST[qt] and float(got["q"][0, 1]) == -MOST[qt]
        # 1e-38 over the least scale, 2^-100 / 57344 = 1.4e-35, is 47 units of e5m2's 2^-16; over e4m3's 1.8e-33 it is below half
        # a unit of 2^-9
        fine = [0, 1, 4]
        check_f8(got["q"][fine], got["scales"][:, fine], x.bfloat16().double()[fine], qt, what="extremes")
        assert bool((got["q"][1].float() == 0).all()) == (qt == E4)
        assert bool(torch.isnan(stands[2, 128:]).all() and (stands[2, :128] == 0).all())
        assert bool(torch.isnan(stands[3, :128]).all() and (stands[3, 128:] == 0).all())
        assert float(got["q"][4, 200]) == -MOST[qt]


# ---- the 8-bit product ------------------------------------------------------------------
def f8_operand(g, rows, cols, dtype, tile):
    v = torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    s = scales_of(v.double(), dtype, tile).float()
    return (v.double() / spread(s.double(), v.shape, tile)).float().clamp(-MOST[dtype], MOST[dtype]).to(dtype), s.contiguous()


def f8_gemm(rt, m, n, k, at, bt, block, out, pad=0, offset=0, seed=0):
    g = torch.Generator().manual_seed(seed + m + 3 * n + 5 * k)
    tile = block == "tile"
    (a, sa), (b, sb) = f8_operand(g, m, k, at, False), f8_operand(g, n, k, bt, tile)
    bufs = Bufs(rt, pad, offset)
    (aa, lda), (ba, ldb), (sa_, ldas), (sb_, ldbs) = bufs.inp(a), bufs.inp(b), bufs.inp(sa), bufs.inp(sb)
    ca, ldc = bufs.out("c", (m, n), out)
    rt.fp8_gemm(t0g.fp8_gemm_desc(aa, sa_, ba, sb_, ca, m, n, k, lda=lda, ldb=ldb, ldc=ldc, ldas=ldas, ldbs=ldbs, a_dtype=TYPES[at],
                                  b_dtype=TYPES[bt], b_block=t0g.BLOCK_TILE if tile else t0g.BLOCK_ROW, out_dtype=TYPES[out]))
    got = bufs.read()["c"]
    av, bv = a.double() * spread(sa.double(), a.shape), b.double() * spread(sb.double(), b.shape, tile)
    want, size = av @ bv.t(), av.abs() @ bv.abs().t()
    bound = 2 * (min(k, 128) + blocks(k) + 70) * U * size
    if out == BF16:
        bound += 7 * 2.0 ** -13 * (largest8(av) @ largest8(bv).t())
    near(got, want, HALF[out] * (want.abs() + bound) + bound, f"{m}x{n}x{k}")


def largest8(v):
    """The largest magnitude of each 8 neighbouring columns."""
    p = torch.zeros((v.shape[0], -(-v.shape[1] // 8) * 8), dtype=torch.float64)
    p[:, :v.shape[1]] = v.abs()
    return p.reshape(v.shape[0], -1, 8).amax(dim=2)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (1, 300, 1000), (2, 17, 130), (7, 100, 64), (15, 250, 1024), (16, 257, 200),
                                   (17, 64, 129), (31, 128, 2049), (32, 1000, 512), (33, 129, 384), (63, 513, 640), (64, 256, 1025),
                                   (65, 200, 256), (100, 300, 4100), (127, 127, 127), (128, 128, 256), (129, 129, 129), (200, 1500, 272),
                                   (256, 256, 512), (257, 511, 1040), (700, 600, 330), (1, 5000, 96), (513, 300, 6000)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("at,bt,out", [(E4, E4, BF16), (E5, E4, F32), (E4, E5, F32), (E5, E5, BF16)])
def test_f8_gemm(rt, m, n, k, block, at, bt, out):
    f8_gemm(rt, m, n, k, at, bt, block, out)


@pytest.mark.parametrize("m,n,k", [(4096, 4096, 128), (3900, 4200, 1200), (4100, 8000, 400), (8200, 2500, 1040)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("at,bt,out", [(E4, E4, BF16), (E5, E4, BF16), (E4, E5, F32)])
def test_f8_gemm_many_tiles(rt, m, n, k, block, at, bt, out):
    f8_gemm(rt, m, n, k, at, bt, block, out)


@pytest.mark.parametrize("m,n,k", [(1, 77, 300), (3, 640, 512), (16, 129, 1000), (40, 130, 256), (70, 400, 784), (300, 290, 640)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("pad,offset", [(3, 1), (16, 16), (1, 0), (128, 4)])
def test_f8_gemm_strides(rt, m, n, k, block, pad, offset):
    f8_gemm(rt, m, n, k, E4, E4, block, F32, pad, offset)


@pytest.mark.parametrize("m,n,k", [(2, 40, 300), (200, 300, 512)])
def test_f8_gemm_keeps_nan_in_its_row(rt, m, n, k):
    """A NaN among A's values, or in a scale, is the result's in its row; a NaN of B in its column."""
    g = torch.Generator().manual_seed(5)
    (a, sa), (b, sb) = f8_operand(g, m, k, E4, False), f8_operand(g, n, k, E4, True)
    a.view(torch.uint8)[1, k - 1] = 0x7F
    b.view(torch.uint8)[3, 7] = 0xFF
    bufs = Bufs(rt)
    (aa, _), (ba, _), (sa_, _), (sb_, _) = bufs.inp(a), bufs.inp(b), bufs.inp(sa), bufs.inp(sb)
    ca, _ = bufs.out("c", (m, n), F32)
    rt.fp8_gemm(t0g.fp8_gemm_desc(aa, sa_, ba, sb_, ca, m, n, k, out_dtype=t0g.F32))
    nan = torch.isnan(bufs.read()["c"])
    want = torch.zeros_like(nan)
    want[1], want[:, 3] = True, True
    assert torch.equal(nan, want)


# ---- gated projections ------------------------------------------------------------------
ACT = {"silu": (1.0, 1.1, 0.5), "gelu": (1.702, 1.13, 0.86), "relu": (None, 1.0, 0.0)}   # k, largest slope and curvature


def act_of(name, g):
    k = ACT[name][0]
    if k is None:
        return g.clamp(min=0.0), (g > 0).double()
    s = torch.sigmoid(k * g)
    return g * s, s + k * g * s * (1 - s)


class Gated:
    def __init__(self, rt, rows, f, hidden, layout="NT", act="silu", pad=0, offset=0, apart=False, seed=0, amp=1.0):
        self.rt, self.rows, self.f, self.hidden, self.layout, self.act = rt, rows, f, hidden, layout, act
        g = torch.Generator().manual_seed(seed + rows + 3 * f + 5 * hidden)
        self.x = data(g, rows, hidden)
        self.wg, self.wu = data(g, f, hidden, scale=amp * hidden ** -0.5), data(g, f, hidden, scale=amp * hidden ** -0.5)
        self.dh = data(g, rows, f)
        self.b = b = Bufs(rt, pad, offset)
        self.xa, self.ldx = b.inp(self.x)
        lay = (lambda w: w) if layout == "NT" else (lambda w: w.t().contiguous())
        if apart:
            (self.ga, self.ldw), (self.ua, _) = b.inp(lay(self.wg)), b.inp(lay(self.wu))
        else:   # one tensor of both
            both = torch.cat([lay(self.wg), lay(self.wu)], dim=0 if layout == "NT" else 1)
            self.ga, self.ldw = b.inp(both)
            self.ua = self.ga + 2 * (f * self.ldw if layout == "NT" else f)
        x, wg, wu = self.x.double(), self.wg.double(), self.wu.double()
        self.g, self.u = x @ wg.t(), x @ wu.t()
        self.eg, self.eu = (2 * (hidden + 70) * U * (x.abs() @ w.abs().t()) for w in (wg, wu))

    def forward(self, keep=False, out=BF16):
        b, shape = self.b, (self.rows, self.f)
        ha, ldh = b.out("h", shape, out)
        kw = {}
        if keep:
            (kw["gate"], kw["ldg"]), (kw["up"], _) = b.out("gate", shape, BF16), b.out("up", shape, BF16)
        self.rt.gated_linear(t0g.gated_linear_desc(self.xa, self.ga, self.ua, ha, self.rows, self.f, self.hidden, transpose=self.layout,
                                                   activation=self.act, ldx=self.ldx, ldw=self.ldw, ldh=ldh, h_dtype=TYPES[out], **kw))
        got = b.read(free=False)
        a, _ = act_of(self.act, self.g)
        h = a * self.u
        bound = HALF[out] * h.abs() + 2.0 ** -20 * h.abs() + ACT[self.act][1] * self.eg * (self.u.abs() + self.eu) + a.abs() * self.eu
        near(got["h"], h, bound, "h")
        if keep:
            near(got["gate"], self.g, 2.0 ** -8 * self.g.abs() + 1.01 * self.eg, "gate")
            near(got["up"], self.u, 2.0 ** -8 * self.u.abs() + 1.01 * self.eu, "up")

    def backward(self, kept, want="xgu", dht=BF16, dxt=BF16, dwt=BF16, stacked=False):
        """kept: from bf16 products of the host's (the call's inputs), else computed again inside."""
        b, kw = self.b, {}
        g, u = self.g, self.u
        if kept:
            gb, ub = g.to(BF16), u.to(BF16)
            (kw["gate"], kw["ldg"]), (kw["up"], _) = b.inp(gb), b.inp(ub)
            g, u = gb.double(), ub.double()
        dh = self.dh.to(dht)
        da, lddh = b.inp(dh)
        wshape = (self.f, self.hidden) if self.layout == "NT" else (self.hidden, self.f)
        outs = dict(dx=0, dwg=0, dwu=0)
        if "x" in want:
            outs["dx"], kw["lddx"] = b.out("dx", self.x.shape, dxt)
        if stacked:
            axis = 0 if self.layout == "NT" else 1
            both = list(wshape)
            both[axis] *= 2
            outs["dwg"], kw["lddw"] = b.out("dw", both, dwt)
            outs["dwu"] = outs["dwg"] + (2 if dwt == BF16 else 4) * (self.f * kw["lddw"] if axis == 0 else self.f)
        else:
            if "g" in want:
                outs["dwg"], kw["lddw"] = b.out("dwg", wshape, dwt)
            if "u" in want:
                outs["dwu"], kw["lddw"] = b.out("dwu", wshape, dwt)
        self.rt.gated_linear_backward(t0g.gated_linear_backward_desc(
            da, self.xa, self.ga, self.ua, self.rows, self.f, self.hidden, transpose=self.layout, activation=self.act, lddh=lddh,
            ldx=self.ldx, ldw=self.ldw, dh_dtype=TYPES[dht], dx_dtype=TYPES[dxt], dw_dtype=TYPES[dwt], **outs, **kw))
        got = b.read()
        if stacked:
            got["dwg"], got["dwu"] = got["dw"].chunk(2, dim=0 if self.layout == "NT" else 1)
        dh = dh.double()
        a, slope = act_of(self.act, g)
        dg, du = dh * u * slope, dh * a
        # their rounding to bf16, the activation's own error, and that of products computed again
        eg, eu = (2.0 ** -8 + 2.0 ** -18) * dg.abs() + 2.0 ** -20 * (dh * u).abs(), (2.0 ** -8 + 2.0 ** -18) * du.abs()
        if not kept:
            eg = eg + 1.01 * dh.abs() * (self.eu * ACT[self.act][1] + (u.abs() + self.eu) * ACT[self.act][2] * self.eg)
            eu = eu + 1.01 * dh.abs() * ACT[self.act][1] * self.eg
            if self.act == "relu":   # the slope's step, where the gate's sign is within its error
                unsure = self.g.abs() <= self.eg
                eg, eu = eg + (dh * u).abs() * unsure, eu
        x, wg, wu = self.x.double(), self.wg.double(), self.wu.double()
        near_ = lambda name, v, e, size, terms, t: near(got[name], v, HALF[t] * v.abs() + 1.01 * e + 2 * (terms + 70) * U * size, name)   # noqa: E731
        if "x" in want:
            near_("dx", dg @ wg + du @ wu, eg @ wg.abs() + eu @ wu.abs(), dg.abs() @ wg.abs() + du.abs() @ wu.abs(), 2 * self.f, dxt)
        for name, d, e in (("dwg", dg, eg), ("dwu", du, eu)):
            if name in got:
                v, e, size = d.t() @ x, e.t() @ x.abs(), d.abs().t() @ x.abs()
                if self.layout == "NN":
                    v, e, size = v.t(), e.t(), size.t()
                near_(name, v, e, size, self.rows, dwt)
        return got

    def free(self):
        for a in self.b.held:
            self.rt.free(a)


@pytest.mark.parametrize("rows,f,hidden", [(1, 1, 1), (1, 64, 64), (1, 300, 1000), (3, 65, 72), (8, 128, 520), (15, 200, 128), (16, 63, 200),
                                           (17, 129, 77), (32, 256, 1024), (33, 100, 2049), (64, 72, 4096), (65, 64, 65), (100, 1000, 136),
                                           (128, 64, 64), (129, 66, 130), (300, 520, 264), (520, 300, 1025), (1, 2000, 4096)])
@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act,out,pad,offset,apart", [("silu", BF16, 0, 0, False), ("gelu", F32, 3, 1, False), ("relu", BF16, 8, 8, True)])
def test_gated(rt, rows, f, hidden, layout, act, out, pad, offset, apart):
    c = Gated(rt, rows, f, hidden, layout, act, pad, offset, apart)
    c.forward(keep=act != "silu", out=out)
    c.free()


@pytest.mark.parametrize("rows,f,hidden", [(2048, 4096, 64), (2000, 4200, 200), (4100, 2050, 330), (300, 16400, 77)])
@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act,out,keep,pad,offset,apart", [("silu", BF16, True, 0, 0, False), ("gelu", F32, False, 8, 8, True),
                                                           ("silu", BF16, False, 3, 1, False)])
def test_gated_many_tiles(rt, rows, f, hidden, layout, act, out, keep, pad, offset, apart):
    c = Gated(rt, rows, f, hidden, layout, act, pad, offset, apart)
    c.forward(keep, out)
    c.free()


@pytest.mark.parametrize("rows,f,hidden", [(1, 1, 1), (1, 64, 64), (3, 65, 72), (16, 63, 200), (17, 128, 77), (64, 72, 512), (130, 264, 136),
                                           (300, 520, 264), (520, 301, 129)])
@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act,kept,pad,offset,apart,stacked,types", [
    ("silu", True, 0, 0, False, False, (BF16, BF16, BF16)), ("gelu", False, 0, 0, False, True, (F32, F32, F32)),
    ("silu", False, 3, 1, True, False, (BF16, F32, BF16)), ("relu", True, 8, 8, True, True, (F32, BF16, F32))])
def test_gated_backward(rt, rows, f, hidden, layout, act, kept, pad, offset, apart, stacked, types):
    c = Gated(rt, rows, f, hidden, layout, act, pad, offset, apart, seed=7)
    c.backward(kept, dht=types[0], dxt=types[1], dwt=types[2], stacked=stacked)


@pytest.mark.parametrize("want", ["x", "g", "u", "gu", "xu"])
@pytest.mark.parametrize("kept", [True, False])
def test_gated_backward_of_some(rt, want, kept):
    Gated(rt, 70, 136, 96).backward(kept, want)


@pytest.mark.parametrize("layout", ["NT", "NN"])
def test_gated_backward_of_no_rows(rt, layout):
    """No rows: dx has none, the weights' gradients are zeros."""
    c = Gated(rt, 1, 40, 72, layout)
    shape = (40, 72) if layout == "NT" else (72, 40)
    (ga, _), (ua, _) = c.b.out("dwg", shape, BF16), c.b.out("dwu", shape, F32)
    da, _ = c.b.inp(c.dh)
    rt.gated_linear(t0g.gated_linear_desc(0, 0, 0, 0, 0, 40, 72, transpose=layout))
    rt.gated_linear_backward(t0g.gated_linear_backward_desc(0, 0, c.ga, c.ua, 0, 40, 72, transpose=layout, dwg=ga))
    rt.gated_linear_backward(t0g.gated_linear_backward_desc(0, 0, c.ga, c.ua, 0, 40, 72, transpose=layout, dwu=ua, dw_dtype=t0g.F32))
    got = c.b.read()
    assert bool((got["dwg"] == 0).all() and (got["dwu"] == 0).all())


def test_gated_backward_against_differences(rt):
    """Of L = sum dh h, in 64 bits, by one weight and one input value at a time; the call's own rounding (bf16 operands,
    2^-8 of the terms) and the curvature over a step of 1e-4 within 2 %  of the gradient's largest value."""
    c = Gated(rt, 3, 24, 32)
    x, wg, wu, dh = (t.double() for t in (c.x, c.wg, c.wu, c.dh))
    got = c.backward(False, dxt=F32, dwt=F32)
    loss = lambda x, wg, wu: (dh * act_of("silu", x @ wg.t())[0] * (x @ wu.t())).sum()   # noqa: E731
    for name, t, args in (("dx", x, 0), ("dwg", wg, 1), ("dwu", wu, 2)):
        for i in range(0, t.numel(), 37):
            h = torch.zeros_like(t)
            h.view(-1)[i] = 1e-4
            ends = [[x, wg, wu], [x, wg, wu]]
            ends[0][args], ends[1][args] = t + h, t - h
            slope = (loss(*ends[0]) - loss(*ends[1])) / 2e-4
            assert abs(slope - got[name].reshape(-1)[i]) <= 0.02 * got[name].abs().max(), (name, i)


def test_rows_far_apart(rt):
    """Rows 2.4 GB apart, the third beyond 2^32 bytes: norms, 8-bit values, and products of few and of more rows."""
    ld, rows, k = 1_200_000_003, 3, 300
    big = rt.alloc((2 * ld + 64 * 512) * 2)
    try:
        g = torch.Generator().manual_seed(1)
        x, w = data(g, rows, k), data(g, 1, k)[0]
        for r in range(rows):
            rt.write(big + 2 * r * ld, raw(x[r].clone()))
        b = Bufs(rt)
        (wa, _), (ya, _), (dya, _) = b.inp(w, True), b.out("y", x.shape, F32), b.inp(data(g, rows, k))
        (qa, _), (ca, _), (ta, _), (tc, _) = (b.out("q", x.shape, E4), b.out("scales", (3, rows), F32), b.out("qt", (k, rows), E4),
                                              b.out("scales_t", (1, k), F32))
        rt.rms_norm(t0g.rms_norm_desc(big, wa, rows, k, y=ya, y_dtype=t0g.F32, ldx=ld))
        rt.fp8_quantize(t0g.fp8_quantize_desc(big, qa, ca, rows, k, qt=ta, scales_t=tc, ldx=ld))
        got = b.read()
        y = norm_of(x, None, w, 0.0, 1e-6)[2]
        near(got["y"], y, (U + NORM_REL) * y.abs(), "y")
        check_f8(got["q"], got["scales"], x.double(), E4, what="q")
        check_f8(got["qt"], got["scales_t"], x.double().t(), E4, what="qt")
        # the same memory as B's rows, bytes apart the same
        for m in (2, 40):
            (a, sa), (q, sq) = f8_operand(g, m, k, E4, False), f8_operand(g, rows, k, E4, False)
            for r in range(rows):
                rt.write(big + 2 * r * ld, raw(q[r].clone()))
            b = Bufs(rt)
            (aa, _), (sa_, _), (sq_, _), (ca, _) = b.inp(a), b.inp(sa), b.inp(sq), b.out("c", (m, rows), F32)
            rt.fp8_gemm(t0g.fp8_gemm_desc(aa, sa_, big, sq_, ca, m, rows, k, ldb=2 * ld, b_block=t0g.BLOCK_ROW, out_dtype=t0g.F32))
            av, bv = a.double() * spread(sa.double(), a.shape), q.double() * spread(sq.double(), q.shape)
            near(b.read()["c"], av @ bv.t(), 2 * (128 + 3 + 70) * U * (av.abs() @ bv.abs().t()) + U * (av @ bv.t()).abs(), f"{m} rows")
    finally:
        rt.wait_idle()
        rt.free(big)


def test_empty_calls(rt):
    """No rows, or no columns of the product: nothing is written, and NULL arrays are no error."""
    rt.rms_norm(t0g.rms_norm_desc(0, 0, 0, 64, y=4096))
    rt.fp8_quantize(t0g.fp8_quantize_desc(0, 4096, 8192, 0, 64))
    rt.fp8_gemm(t0g.fp8_gemm_desc(0, 0, 0, 0, 0, 0, 64, 64))
    rt.fp8_gemm(t0g.fp8_gemm_desc(0, 0, 0, 0, 0, 64, 0, 64))
    b = Bufs(rt)
    dwa, _ = b.out("dw", (1, 64), F32)
    rt.rms_norm_backward(t0g.rms_norm_backward_desc(0, 0, 0, 0, 64, dw=dwa))
    assert bool((b.read()["dw"] == 0).all())


# ---- together ---------------------------------------------------------------------------
class Layer:
    """A feed-forward layer as a program runs it, in 8 bits (serving) or bf16 with its backward pass (training)."""

    def __init__(self, rt, rows, hidden, f, seed=0):
        self.rt, self.rows, self.hidden, self.f = rt, rows, hidden, f
        g = torch.Generator().manual_seed(seed)
        self.x, self.r = data(g, rows, hidden), data(g, rows, hidden)
        self.w = (1 + 0.1 * torch.randn(1, hidden, generator=g)).bfloat16()
        self.wgu, self.wd = data(g, 2 * f, hidden, scale=hidden ** -0.5), data(g, hidden, f, scale=f ** -0.5)
        self.dy = data(g, rows, hidden)
        self.b = b = Bufs(rt)
        self.a = {n: b.inp(getattr(self, n), True)[0] for n in ("x", "r", "w", "wgu", "wd", "dy")}
        self.n = 0

    def out(self, name, rows, cols, dtype):
        return self.b.out(name, (rows, cols), dtype)[0]

    def serve(self):
        """norm in 8 bits -> gate and up in 8 bits; norm in bf16 -> gated -> 8 bits -> down in 8 bits."""
        rt, a, t, h, f = self.rt, self.a, self.rows, self.hidden, self.f
        o = {n: self.out(n, *s) for n, s in dict(
            sum=(t, h, BF16), n=(t, h, BF16), q=(t, h, E4), qs=(blocks(h), t, F32), w8=(2 * f, h, E4), w8s=(blocks(h), blocks(2 * f), F32),
            d8=(h, f, E4), d8s=(blocks(f), blocks(h), F32), gu=(t, 2 * f, F32), h=(t, f, BF16), h8=(t, f, E4), h8s=(blocks(f), t, F32),
            y=(t, h, F32)).items()}
        rt.fp8_quantize(t0g.fp8_quantize_desc(a["wgu"], o["w8"], o["w8s"], 2 * f, h, block=t0g.BLOCK_TILE))
        rt.fp8_quantize(t0g.fp8_quantize_desc(a["wd"], o["d8"], o["d8s"], h, f, block=t0g.BLOCK_TILE))

        def go():
            rt.rms_norm(t0g.rms_norm_desc(a["x"], a["w"], t, h, residual=a["r"], sum=o["sum"], y=o["n"], q=o["q"], scales=o["qs"]))
            rt.fp8_gemm(t0g.fp8_gemm_desc(o["q"], o["qs"], o["w8"], o["w8s"], o["gu"], t, 2 * f, h, out_dtype=t0g.F32))
            rt.gated_linear(t0g.gated_linear_desc(o["n"], a["wgu"], a["wgu"] + 2 * f * h, o["h"], t, f, h))
            rt.fp8_quantize(t0g.fp8_quantize_desc(o["h"], o["h8"], o["h8s"], t, f))
            rt.fp8_gemm(t0g.fp8_gemm_desc(o["h8"], o["h8s"], o["d8"], o["d8s"], o["y"], t, h, f, out_dtype=t0g.F32))
        return go

    def train(self):
        """norm -> gated -> down (a GEMM) and back: dh = dy Wd, the gated pair's gradients, the norm's."""
        rt, a, t, h, f = self.rt, self.a, self.rows, self.hidden, self.f
        o = {n: self.out(n, *s) for n, s in dict(
            sum=(t, h, BF16), n=(t, h, BF16), h=(t, f, BF16), gate=(t, f, BF16), up=(t, f, BF16), y=(t, h, BF16), dh=(t, f, BF16),
            dn=(t, h, BF16), dw=(2 * f, h, F32), dx=(t, h, BF16), dnw=(1, h, F32)).items()}

        def go():
            rt.rms_norm(t0g.rms_norm_desc(a["x"], a["w"], t, h, residual=a["r"], sum=o["sum"], y=o["n"]))
            rt.gated_linear(t0g.gated_linear_desc(o["n"], a["wgu"], a["wgu"] + 2 * f * h, o["h"], t, f, h, gate=o["gate"], up=o["up"]))
            rt.gemm_desc(t0g.gemm_desc(o["h"], a["wd"], o["y"], t, h, f, out_dtype=t0g.BF16))
            rt.gemm_desc(t0g.gemm_desc(a["dy"], a["wd"], o["dh"], t, f, h, transpose="NN", out_dtype=t0g.BF16))
            rt.gated_linear_backward(t0g.gated_linear_backward_desc(
                o["dh"], o["n"], a["wgu"], a["wgu"] + 2 * f * h, t, f, h, gate=o["gate"], up=o["up"], dx=o["dn"], dwg=o["dw"],
                dwu=o["dw"] + 4 * f * h, dw_dtype=t0g.F32))
            rt.rms_norm_backward(t0g.rms_norm_backward_desc(o["dn"], o["sum"], a["w"], t, h, dsum=a["dy"], dx=o["dx"], dw=o["dnw"]))
        return go


@pytest.mark.parametrize("rows", [1, 37, 300])
def test_layer_in_8_bits(rt, rows):
    """Every step against the definition on the step's own inputs, as the device holds them."""
    c = Layer(rt, rows, 384, 712, seed=rows)
    c.serve()()
    got = c.b.read()
    s, _, y = norm_of(c.x, c.r, c.w[0], 0.0, 1e-6)
    near(got["n"], y, (2.0 ** -8 + NORM_REL) * y.abs(), "norm")
    check_f8(got["q"], got["qs"], y, E4, slack=NORM_REL, what="norm")
    check_f8(got["w8"], got["w8s"], c.wgu.double(), E4, True, what="weights")

    def product(q, qs, w, ws, name):
        a, b = q.double() * spread(qs.double(), q.shape), w.double() * spread(ws.double(), w.shape, True)
        near(got[name], a @ b.t(), 2 * (128 + blocks(q.shape[1]) + 70) * U * (a.abs() @ b.abs().t()), name)

    product(got["q"], got["qs"], got["w8"], got["w8s"], "gu")
    check_f8(got["h8"], got["h8s"], got["h"].double(), E4, what="h")
    product(got["h8"], got["h8s"], got["d8"], got["d8s"], "y")


@pytest.mark.parametrize("what", ["serve", "train"])
def test_layer_captured(rt, what):
    """A layer's calls in a graph: replays between eager work give what the eager calls gave, and so does a second graph of
    another size of the same handle, whose scratch is larger."""
    stream = hip_rt.Stream()
    small, large = Layer(rt, 70, 264, 520, seed=1), Layer(rt, 333, 520, 1032, seed=2)
    goes = [getattr(c, what)() for c in (small, large)]
    rt.set_stream(stream.ptr)
    graphs = []
    try:
        for c, go in zip((small, large), goes):
            go()
        rt.wait_idle()
        first = [c.b.read(free=False) for c in (small, large)]
        graphs = [hip_rt.Graph(stream, go) for go in goes]
        for turn in range(3):
            for c, graph in zip((small, large), graphs):
                for name, (addr, image, _) in c.b.outs.items():
                    if name not in ("w8", "w8s", "d8", "d8s"):
                        rt.memset(addr, 0x5A, raw(image).nbytes)
                graph.launch(stream)
                if turn == 1:
                    goes[0]()
            rt.wait_idle()
            for c, want in zip((small, large), first):
                for name, (addr, image, view) in c.b.outs.items():
                    r = raw(image)
                    r[:] = rt.read(addr, r.shape, r.dtype)
                    assert torch.equal(view.view(torch.uint8) if view.element_size() == 1 else view,
                                       want[name].view(torch.uint8) if view.element_size() == 1 else want[name]), (turn, name)
    finally:
        rt.wait_idle()
        for gr in graphs:
            gr.destroy()
        rt.set_stream(None)
        stream.destroy()
    for c in (small, large):
        for a in c.b.held:
            rt.free(a)


def test_capture_needs_the_scratch(rt):
    """A captured call whose scratch the handle does not hold yet is refused, and the handle still works."""
    with t0g.GpuRuntime.new(0) as own:
        c = Gated(own, 40, 72, 136)
        stream = hip_rt.Stream()
        ha, _ = c.b.out("h", (40, 72), BF16)
        dwa, _ = c.b.out("dwg", (72, 136), BF16)
        da, _ = c.b.inp(c.dh)
        d = t0g.gated_linear_backward_desc(da, c.xa, c.ga, c.ua, 40, 72, 136, dwg=dwa)
        own.set_stream(stream.ptr)

        def call():
            with pytest.raises(t0g.T0gError) as e:
                own.gated_linear_backward(d)
            assert e.value.code == t0g.ERR_INVALID_ARG and "capture" in str(e.value)

        hip_rt.Graph(stream, call).destroy()
        own.gated_linear_backward(d)
        own.wait_idle()
        own.set_stream(None)
        stream.destroy()


def test_same_results_every_time(rt):
    """Bit for bit, run after run, other calls in between."""
    first = None
    for turn in range(3):
        c = Layer(rt, 300, 520, 712, seed=4)
        c.train()()
        got = c.b.read()
        f8_gemm(rt, 40, 130, 1000, E4, E4, "row", F32)
        if first is None:
            first = got
        for name in got:
            assert torch.equal(got[name], first[name]), name
