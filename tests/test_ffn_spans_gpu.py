"""The gated pair's gradients where the GEMMs do not take an operand as a whole: rows far apart, and [dgate | dup] of 2^31
elements and more with an odd number of features.  Bounds as in test_ffn_gpu; rows without a gradient add no error."""
import pytest
import torch

import t0g
from test_ffn_gpu import ACT, BF16, F32, HALF, TYPES, U, Bufs, act_of, data, near, raw, rt   # noqa: F401

pytestmark = pytest.mark.gpu


def check(got, x, wg, wu, dh, gate, up, dxt, dwt, layout):
    """gate, up: what the call was given, or None.  Weights as [features][hidden]; rows without a gradient left out of x and dh."""
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    rows, hidden = x.shape
    if gate is None:
        g, u = x @ wg.t(), x @ wu.t()
        eg, eu = (2 * (hidden + 70) * U * (x.abs() @ w.abs().t()) for w in (wg, wu))
    else:
        g, u = gate.double(), up.double()
        eg = eu = torch.zeros_like(g)
    a, slope = act_of("silu", g)
    dg, du = dh * u * slope, dh * a
    _, k, curve = ACT["silu"]
    og = (2.0 ** -8 + 2.0 ** -18) * dg.abs() + 2.0 ** -20 * (dh * u).abs() + 1.01 * dh.abs() * (eu * k + (u.abs() + eu) * curve * eg)
    ou = (2.0 ** -8 + 2.0 ** -18) * du.abs() + 1.01 * dh.abs() * k * eg
    f = wg.shape[0]
    for name, t, terms, pairs in (("dx", dxt, 2 * f, ((dg, og, wg), (du, ou, wu))), ("dwg", dwt, rows, ((dg.t(), og.t(), x),)),
                                  ("dwu", dwt, rows, ((du.t(), ou.t(), x),))):
        if name not in got:
            continue
        v = sum(d @ m for d, _, m in pairs)
        bound = HALF[t] * v.abs() + sum(1.01 * (o @ m.abs()) + 2 * (terms + 70) * U * (d.abs() @ m.abs()) for d, o, m in pairs)
        near(got[name] if name == "dx" or layout == "NT" else got[name].t(), v, bound, name)


@pytest.mark.parametrize("far", ["x", "w"])
@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("ld", [1_200_000_003, 1_200_000_000, 300_000_008])
@pytest.mark.parametrize("kept", [True, False])
def test_rows_far_apart(rt, far, layout, ld, kept):   # noqa: F811
    """x or both weights, side by side in one tensor, with rows that far apart."""
    g = torch.Generator().manual_seed(ld)
    n = 3 if ld > 1 << 30 else 9                      # rows of the far operand
    if far == "x":
        rows, f, hidden = n, 45, 72
    else:
        rows, f, hidden = 37, (n if layout == "NT" else 45), (72 if layout == "NT" else n)
    lay = (lambda w: w) if layout == "NT" else (lambda w: w.t().contiguous())
    x, dh = data(g, rows, hidden), data(g, rows, f)
    wg, wu = data(g, f, hidden, scale=hidden ** -0.5), data(g, f, hidden, scale=hidden ** -0.5)
    gate, up = (data(g, rows, f), data(g, rows, f)) if kept else (None, None)
    big = rt.alloc(((n - 1) * ld + 4096) * 2)
    try:
        b = Bufs(rt)
        (da, _), (ga, _), (ua, _) = b.inp(dh), b.inp(gate), b.inp(up)
        if far == "x":
            (wga, ldw), (wua, _) = b.inp(lay(wg)), b.inp(lay(wu))
            xa, ldx = big, ld
            for i in range(n):
                rt.write(big + 2 * i * ld, raw(x[i].clone()))
        else:
            xa, ldx = b.inp(x)
            wga, wua, ldw = big, big + 2 * 1000, ld
            for i in range(n):
                for at, w in ((wga, wg), (wua, wu)):
                    rt.write(at + 2 * i * ld, raw(lay(w)[i].clone()))
        shape = tuple(lay(wg).shape)
        (dxa, _), (dga, _), (dua, _) = b.out("dx", x.shape, BF16), b.out("dwg", shape, F32), b.out("dwu", shape, F32)
        d = t0g.gated_linear_backward_desc(da, xa, wga, wua, rows, f, hidden, transpose=layout, gate=ga, up=ua, dx=dxa, dwg=dga, dwu=dua, ldx=ldx,
                                           ldw=ldw, dw_dtype=t0g.F32)
        rt.gated_linear_backward(d)
        check(b.read(), x, wg, wu, dh, gate, up, BF16, F32, layout)
    finally:
        rt.wait_idle()
        rt.free(big)


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("kept", [True, False])
def test_many_rows_of_odd_features(rt, layout, kept):   # noqa: F811
    """[dgate | dup] of 1060000 rows of 2064 values, in three pieces.  Six rows have a gradient, on both sides of each
    piece's end."""
    rows, f, hidden = 1_060_000, 1025, 9
    end = ((1 << 30) - 1) // 2064 // 64 * 64
    some = [0, end - 1, end, 2 * end - 1, 2 * end, rows - 1]
    g = torch.Generator().manual_seed(rows)
    lay = (lambda w: w) if layout == "NT" else (lambda w: w.t().contiguous())
    x = data(g, rows, hidden)
    dh, gate, up = (data(g, len(some), f) for _ in range(3))
    wg, wu = data(g, f, hidden, scale=hidden ** -0.5), data(g, f, hidden, scale=hidden ** -0.5)
    held = [rt.alloc(rows * f * 2) for _ in range(3 if kept else 1)]
    try:
        for addr, t in zip(held, (dh, gate, up)):
            rt.memset(addr, 0, rows * f * 2)
            rt.wait_idle()
            for i, r in enumerate(some):
                rt.write(addr + 2 * r * f, raw(t[i].clone()))
        b = Bufs(rt)
        (xa, _), (wga, _), (wua, _) = b.inp(x), b.inp(lay(wg)), b.inp(lay(wu))
        shape = tuple(lay(wg).shape)
        (dxa, _), (dga, _), (dua, _) = b.out("dx", x.shape, F32), b.out("dwg", shape, BF16), b.out("dwu", shape, BF16)
        d = t0g.gated_linear_backward_desc(held[0], xa, wga, wua, rows, f, hidden, transpose=layout, gate=held[1] if kept else 0,
                                           up=held[2] if kept else 0, dx=dxa, dwg=dga, dwu=dua, dx_dtype=t0g.F32)
        rt.gated_linear_backward(d)
        got = b.read()
        left = torch.ones(rows, dtype=torch.bool)
        left[some] = False
        assert bool((got["dx"][left] == 0).all())
        got["dx"] = got["dx"][some]
        check(got, x[some], wg, wu, dh, gate if kept else None, up if kept else None, F32, BF16, layout)
    finally:
        rt.wait_idle()
        for addr in held:
            rt.free(addr)
