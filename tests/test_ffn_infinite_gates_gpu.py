"""Gates that are infinite, not a number, or near the largest f32: the gated projections and their gradients against the
formulas in 64 bits, in which the same elements are infinite or not a number.

A gate is infinite where x and Wg multiply to more than f32 holds (2^120 by +-2^10, u untouched by a zero in Wu), and not a number in a feature
whose weights have one.  Finite elements: bounds as in test_ffn_gpu."""
import pytest
import torch

import t0g
from test_ffn_gpu import ACT, BF16, F32, HALF, TYPES, U, Bufs, act_of, data, near, rt   # noqa: F401

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def same(got, want, bound, what):
    """near(), with infinities where they have to be."""
    want = want.float().double()   # more than f32 holds is infinite
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got.double()), inf) and torch.equal(got.double()[inf], want[inf]), f"{what}: infinities"
    zero = torch.zeros_like(want)
    near(torch.where(inf, zero.to(got.dtype), got), torch.where(inf, zero, want), torch.where(inf, zero, bound), what)


class Case:
    def __init__(self, rt, rows, f, hidden, layout, act):   # noqa: F811
        self.rt, self.layout, self.act, self.sizes = rt, layout, act, (rows, f, hidden)
        g = torch.Generator().manual_seed(rows + f)
        self.x, self.dh = data(g, rows, hidden), data(g, rows, f)
        self.wg, self.wu = data(g, f, hidden, scale=hidden ** -0.5), data(g, f, hidden, scale=hidden ** -0.5)
        self.wg[:, 0] = self.wu[:, 0] = 0.0
        self.wg[1, 0], self.wg[f - 2, 0], self.wg[3, 5] = 2.0 ** 10, -2.0 ** 10, NAN
        self.x[rows // 2, 0] = 2.0 ** 120
        self.b = Bufs(rt)
        lay = (lambda w: w) if layout == "NT" else (lambda w: w.t().contiguous())
        (self.xa, _), (self.ga, _), (self.ua, _) = self.b.inp(self.x), self.b.inp(lay(self.wg)), self.b.inp(lay(self.wu))
        x, wg, wu = self.x.double(), self.wg.double(), self.wu.double()
        self.g, self.u = (x @ wg.t()).float().double(), x @ wu.t()
        assert int(torch.isinf(self.g).sum()) == 2 and int(torch.isnan(self.g[0]).sum()) == 1
        self.eg, self.eu = (2 * (hidden + 70) * U * (x.abs() @ w.abs().t()) for w in (wg.nan_to_num(), wu))

    def forward(self, out):
        rows, f, hidden = self.sizes
        ha, _ = self.b.out("h", (rows, f), out)
        ga, _ = self.b.out("gate", (rows, f), BF16)
        self.rt.gated_linear(t0g.gated_linear_desc(self.xa, self.ga, self.ua, ha, rows, f, hidden, transpose=self.layout, activation=self.act,
                                                   gate=ga, h_dtype=TYPES[out]))
        got = self.b.read()
        a, _ = act_of(self.act, self.g)
        h = a * self.u
        bound = (HALF[out] + 2.0 ** -20) * h.abs() + ACT[self.act][1] * self.eg * (self.u.abs() + self.eu) + a.abs() * self.eu
        same(got["h"], h, bound, "h")
        same(got["gate"], self.g, 2.0 ** -8 * self.g.abs() + 1.01 * self.eg, "gate")


@pytest.mark.parametrize("rows,f,hidden", [(1, 64, 64), (20, 72, 200), (40, 72, 136), (64, 64, 4096), (1000, 2731, 80), (2048, 4096, 64)])
@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_forward(rt, rows, f, hidden, layout, act):   # noqa: F811
    Case(rt, rows, f, hidden, layout, act).forward(F32 if act == "relu" else BF16)


def check_backward(got, c, g, u, eg, eu, dxt, dwt):
    act, dh, x, wg, wu = c.act, c.dh.double(), c.x.double(), c.wg.double(), c.wu.double()
    a, slope = act_of(act, g)
    if act == "relu":
        slope = torch.where(torch.isnan(g), g, slope)
    dg, du = dh * u * slope, dh * a
    # bf16 operands: infinite past its largest value
    dg, du = (torch.where(torch.isinf(d.float().to(BF16).double()), INF * d.sign(), d) for d in (dg, du))
    off_g = (2.0 ** -8 + 2.0 ** -18) * dg.abs() + 2.0 ** -20 * (dh * u).abs()
    off_u = (2.0 ** -8 + 2.0 ** -18) * du.abs()
    off_g = off_g + 1.01 * dh.abs() * (eu * ACT[act][1] + (u.abs() + eu) * ACT[act][2] * eg)
    off_u = off_u + 1.01 * dh.abs() * ACT[act][1] * eg
    if act == "relu":
        off_g = off_g + (dh * u).abs() * (g.abs() <= eg)
    for name, t, pairs in (("dx", dxt, ((dg, off_g, wg), (du, off_u, wu))), ("dwg", dwt, ((dg.t(), off_g.t(), x),)), ("dwu", dwt, ((du.t(), off_u.t(), x),))):
        v = sum(d @ m for d, _, m in pairs)
        terms = sum(d.shape[1] for d, _, m in pairs)
        bound = HALF[t] * v.abs() + sum(1.01 * (o @ m.abs()) + 2 * (terms + 70) * U * (d.abs() @ m.abs()) for d, o, m in pairs)
        y = got[name] if name == "dx" or c.layout == "NT" else got[name].t()
        # a bound that is not a number stands where the value is none
        same(y, v, torch.where(torch.isnan(v), torch.zeros_like(v), bound), name)


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,f,hidden", [(40, 72, 136), (1000, 600, 80)])
def test_backward_of_kept_gates(rt, rows, f, hidden, layout, act):   # noqa: F811
    c = Case(rt, rows, f, hidden, layout, act)
    c.x[:, 0] = 1.0
    g, u = (torch.randn(rows, f, generator=torch.Generator().manual_seed(s)).to(BF16) for s in (1, 2))
    c.wg.nan_to_num_(0.25)
    g[1, 5], g[2, 6], g[3, 7], g[4, 8], g[5, 9] = INF, -INF, NAN, 3.0e38, -3.0e38
    b = c.b = Bufs(rt)
    lay = (lambda w: w) if layout == "NT" else (lambda w: w.t().contiguous())
    (xa, _), (wga, _), (wua, _), (da, _), (ga, _), (ua, _) = (b.inp(t) for t in (c.x, lay(c.wg), lay(c.wu), c.dh, g, u))
    (dxa, _), (dga, _), (dua, _) = b.out("dx", c.x.shape, F32), b.out("dwg", lay(c.wg).shape, F32), b.out("dwu", lay(c.wu).shape, F32)
    f32 = t0g.F32
    rt.gated_linear_backward(t0g.gated_linear_backward_desc(da, xa, wga, wua, rows, f, hidden, transpose=layout, activation=act, gate=ga, up=ua,
                                                            dx=dxa, dwg=dga, dwu=dua, dx_dtype=f32, dw_dtype=f32))
    zero = torch.zeros(rows, f, dtype=torch.float64)
    check_backward(b.read(), c, g.double(), u.double(), zero, zero, F32, F32)


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,f,hidden", [(40, 72, 136), (1000, 2731, 80)])
def test_backward_with_gates_computed_again(rt, rows, f, hidden, layout, act):   # noqa: F811
    c = Case(rt, rows, f, hidden, layout, act)
    da, _ = c.b.inp(c.dh)
    shape = (f, hidden) if layout == "NT" else (hidden, f)
    (dxa, _), (dga, _), (dua, _) = c.b.out("dx", c.x.shape, F32), c.b.out("dwg", shape, F32), c.b.out("dwu", shape, F32)
    f32 = t0g.F32
    c.rt.gated_linear_backward(t0g.gated_linear_backward_desc(da, c.xa, c.ga, c.ua, rows, f, hidden, transpose=layout, activation=act, dx=dxa,
                                                              dwg=dga, dwu=dua, dx_dtype=f32, dw_dtype=f32))
    check_backward(c.b.read(), c, c.g, c.u, c.eg, c.eu, F32, F32)
