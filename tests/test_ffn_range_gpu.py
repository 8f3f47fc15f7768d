"""The norm and its gradients of rows whose squares f32 does not hold, against the definition in 64 bits.

Tolerances as for other rows (test_ffn_gpu), and below f32's and bf16's least normal values half a unit there for each
rounding: 2^-147 and 2^-133."""
import pytest
import torch

import t0g
from test_ffn_gpu import BF16, E4, F32, HALF, NORM_REL, TYPES, U, Bufs, blocks, check_f8, near, norm_of, rt   # noqa: F401

pytestmark = pytest.mark.gpu
LEAST = {F32: 2.0 ** -147, BF16: 2.0 ** -133}


def rows_of(g, sizes, hidden, dtype):
    """A row for each size, its values spread evenly up to it."""
    v = (torch.rand(len(sizes), hidden, generator=g, dtype=torch.float64) * 2 - 1) * torch.tensor(sizes, dtype=torch.float64)[:, None]
    return v.float().to(dtype)


@pytest.mark.parametrize("hidden", [1, 300, 512, 1001, 2048, 4096, 4099, 8192, 9001, 16384])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-19, 1e-5])
def test_norm_of_any_magnitude(rt, hidden, dtype, eps):   # noqa: F811
    g = torch.Generator().manual_seed(hidden)
    sizes = [1e20, 1.0, 1e-24, 3e38, 1e-36, 1e15, 1e-13, 1e17, 1e-44 if dtype == F32 else 1e-38]
    x = rows_of(g, sizes, hidden, dtype)
    if hidden > 1:
        x[0, ::2] = 0.0
    else:
        x[-1] = 1e-40   # not zero, whose norm with eps 0 is not a number
    w = 1 + 0.1 * torch.randn(1, hidden, generator=g)[0]
    b = Bufs(rt)
    (xa, _), (wa, _), (ya, _) = b.inp(x), b.inp(w, True), b.out("y", x.shape, F32)
    (sa, _), (za, _) = b.out("sum", x.shape, dtype), b.out("z", x.shape, BF16)
    (qa, _), (ca, _) = b.out("q", x.shape, E4), b.out("scales", (blocks(hidden), len(sizes)), F32)
    same = dict(eps=eps, x_dtype=TYPES[dtype], sum_dtype=TYPES[dtype], weight_dtype=t0g.F32)
    rt.rms_norm(t0g.rms_norm_desc(xa, wa, len(sizes), hidden, sum=sa, y=ya, q=qa, scales=ca, y_dtype=t0g.F32, **same))
    rt.rms_norm(t0g.rms_norm_desc(xa, 0, len(sizes), hidden, y=za, **same))
    got = b.read()
    assert torch.equal(got["sum"], x)
    y = norm_of(x, None, w, 0.0, eps)[2]
    near(got["y"], y, (U + NORM_REL) * y.abs() + 2 * LEAST[F32], "y")
    check_f8(got["q"], got["scales"], y, E4, slack=NORM_REL, what="q")
    z = norm_of(x, None, None, 0.0, eps)[2]
    near(got["z"], z, (HALF[BF16] + NORM_REL) * z.abs() + LEAST[BF16], "z")


@pytest.mark.parametrize("rows,hidden", [(8, 1), (9000, 40), (2500, 300), (3000, 1000), (2300, 2048), (1500, 4096), (40, 8192), (40, 9001),
                                         (300, 16384)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("amp,each", [(1.0, [1e20, 1.0, 1e-24, 3e38, 1e-36, 1e15, 1e-13]), (2.0 ** 61, [1e20, 1e-15, 1.0, 3e38, 1e13])])
def test_norm_backward_of_any_magnitude(rt, rows, hidden, dtype, amp, each):   # noqa: F811
    """Several rows to a workgroup, of magnitudes in turn."""
    g = torch.Generator().manual_seed(rows + hidden)
    x = rows_of(g, [each[i % len(each)] for i in range(rows)], hidden, dtype)
    dy = (torch.randn(rows, hidden, generator=g) * amp).to(dtype)
    w = (1 + 0.1 * torch.randn(1, hidden, generator=g)[0]).to(dtype)
    b, t = Bufs(rt), TYPES[dtype]
    (ya, _), (xa, _), (wa, _) = b.inp(dy), b.inp(x), b.inp(w, True)
    (dxa, _), (dwa, _) = b.out("dx", x.shape, F32), b.out("dw", (1, hidden), F32)
    rt.rms_norm_backward(t0g.rms_norm_backward_desc(ya, xa, wa, rows, hidden, eps=0.0, dx=dxa, dw=dwa, dy_dtype=t, x_dtype=t, weight_dtype=t,
                                                    dx_dtype=t0g.F32))
    got = b.read()
    s, rho, _ = norm_of(x, None, None, 0.0, 0.0)
    n, gr = s * rho, dy.double() * w.double()
    want = rho * (gr - n * (gr * n).mean(1, keepdim=True))
    size = rho * (gr.abs() + n.abs() * (gr * n).abs().mean(1, keepdim=True))
    near(got["dx"], want, U * want.abs() + 2 * NORM_REL * size + 2 * LEAST[F32], "dx")
    each = dy.double() * n
    near(got["dw"], each.sum(0, keepdim=True), (U + NORM_REL + (rows + 34) * U) * each.abs().sum(0, keepdim=True), "dw")


@pytest.mark.parametrize("hidden", [300, 4096, 9001])
@pytest.mark.parametrize("size,weight", [(1e-12, 1e-26), (1e-20, 1e-24), (1e13, 1e25), (1e30, 1e30), (1e-30, 1e36)])
def test_norm_in_8_bits_of_weights_of_any_magnitude(rt, hidden, size, weight):   # noqa: F811
    """x times the weight, without the norm's factor, is not f32's."""
    g = torch.Generator().manual_seed(hidden)
    x, w = rows_of(g, [size] * 3, hidden, F32), rows_of(g, [weight], hidden, F32)[0]
    b = Bufs(rt)
    (xa, _), (wa, _), (ya, _) = b.inp(x), b.inp(w, True), b.out("y", x.shape, F32)
    (qa, _), (ca, _) = b.out("q", x.shape, E4), b.out("scales", (blocks(hidden), 3), F32)
    f = t0g.F32
    rt.rms_norm(t0g.rms_norm_desc(xa, wa, 3, hidden, eps=0.0, y=ya, q=qa, scales=ca, x_dtype=f, weight_dtype=f, y_dtype=f))
    got, y = b.read(), norm_of(x, None, w, 0.0, 0.0)[2]
    near(got["y"], y, (U + NORM_REL) * y.abs() + 2 * LEAST[F32], "y")
    check_f8(got["q"], got["scales"], y, E4, slack=NORM_REL, what="q")
