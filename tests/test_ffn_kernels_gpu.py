"""The feed-forward layer's calls at the sizes that decide which kernel runs and which of its loops: every tile of the
products in every type, operands that are copied in front of the large tiles, the loops over several rows of a workgroup and
over several blocks in flight.  What is checked, and how exactly, as in test_ffn_gpu, whose functions run here at these sizes.

Products of more than 32 rows take 256x256 tiles (a bf16 result in 256 or more of them; gated 256x128), else 128-row tiles
where 64-row ones would take more than 1.6 times as many rounds of 512."""
import pytest
import torch

import t0g
import test_ffn_gpu as base
from test_ffn_gpu import BF16, E4, E5, F32, HALF, NORM_REL, TYPES, U, Bufs, Gated, blocks, check_f8, data, near, norm_of, raw, rt   # noqa: F401

pytestmark = pytest.mark.gpu
PAIRS = [(E4, E4), (E4, E5), (E5, E4), (E5, E5)]


# ---- products ---------------------------------------------------------------------------
@pytest.mark.parametrize("m,n,k", [(2048, 4096, 272), (2000, 4090, 333)])   # 512 tiles of 128x128, 1024 of 64x128
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("at,bt", PAIRS)
@pytest.mark.parametrize("out", [BF16, F32])
def test_f8_in_128_row_tiles(rt, m, n, k, block, at, bt, out):   # noqa: F811
    base.f8_gemm(rt, m, n, k, at, bt, block, out)


@pytest.mark.parametrize("m,n,k", [(4096, 4096, 272), (3900, 4200, 333)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("at,bt", PAIRS)
def test_f8_in_256_row_tiles(rt, m, n, k, block, at, bt):   # noqa: F811
    base.f8_gemm(rt, m, n, k, at, bt, block, BF16)


@pytest.mark.parametrize("m,n", [(4096, 4096), (2048, 4096), (100, 300)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("pad,offset", [(3, 1), (16, 16), (5, 0)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_f8_of_rows_apart(rt, m, n, block, pad, offset, out):   # noqa: F811
    base.f8_gemm(rt, m, n, 400, E4, E4, block, out, pad, offset)


@pytest.mark.parametrize("m", [33, 100, 300])
@pytest.mark.parametrize("at,bt", PAIRS)
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("out", [BF16, F32])
def test_f8_in_64_row_tiles_and_slices(rt, m, at, bt, block, out):   # noqa: F811
    base.f8_gemm(rt, m, 300, 2100, at, bt, block, out)


@pytest.mark.parametrize("m", [1, 5, 16, 17, 32])
@pytest.mark.parametrize("n,k", [(200, 4096), (130, 4200), (40, 8300)])   # more than the blocks in flight of all waves
@pytest.mark.parametrize("at,bt", PAIRS)
@pytest.mark.parametrize("block", ["row", "tile"])
def test_f8_of_few_rows(rt, m, n, k, at, bt, block):   # noqa: F811
    base.f8_gemm(rt, m, n, k, at, bt, block, F32 if m % 2 else BF16)


@pytest.mark.parametrize("rows,f,hidden", [(1000, 2731, 200), (1500, 2100, 77), (1024, 2048 + 64, 136)])   # 128x64
@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act,out,keep,pad,offset,apart", [("silu", BF16, True, 0, 0, False), ("gelu", F32, False, 3, 1, True),
                                                           ("relu", BF16, True, 8, 8, False)])
def test_gated_in_128_row_tiles(rt, rows, f, hidden, layout, act, out, keep, pad, offset, apart):   # noqa: F811
    c = Gated(rt, rows, f, hidden, layout, act, pad, offset, apart)
    c.forward(keep, out)
    c.free()


@pytest.mark.parametrize("rows,f,hidden", [(1000, 2731, 200), (1500, 2100, 77), (2048, 4096, 64)])
@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("act,pad,offset,apart,types", [("silu", 0, 0, False, (BF16, BF16, BF16)), ("gelu", 3, 1, True, (F32, F32, BF16)),
                                                        ("relu", 8, 8, False, (BF16, BF16, F32))])
def test_gated_backward_computed_again_in_128_row_tiles(rt, rows, f, hidden, layout, act, pad, offset, apart, types):   # noqa: F811
    Gated(rt, rows, f, hidden, layout, act, pad, offset, apart, seed=3).backward(False, dht=types[0], dxt=types[1], dwt=types[2])


# ---- rows -------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,hidden", [(5000, 512), (5000, 200), (2100, 2048), (2100, 4096), (1100, 8192), (600, 9008)])
@pytest.mark.parametrize("xt,yt,wt,st", [(BF16, BF16, BF16, BF16), (BF16, BF16, None, None), (F32, BF16, BF16, F32)])
def test_norm_backward_of_several_rows_to_a_workgroup(rt, rows, hidden, xt, yt, wt, st):   # noqa: F811
    base.test_norm_backward(rt, rows, hidden, xt, yt, wt, st, *((0, 0) if rows * hidden > 1 << 22 else (8, 8)))


def test_norm_of_several_rows_to_a_wave(rt):   # noqa: F811
    """More rows than the largest launch has waves for."""
    rows, hidden = (1 << 22) + 1000, 8
    x = data(torch.Generator().manual_seed(1), rows, hidden)
    b = Bufs(rt)
    (xa, _), (ya, _) = b.inp(x), b.out("y", x.shape, BF16)
    rt.rms_norm(t0g.rms_norm_desc(xa, 0, rows, hidden, y=ya))
    y = norm_of(x, None, None, 0.0, 1e-6)[2]
    near(b.read()["y"], y, (HALF[BF16] + NORM_REL) * y.abs(), "y")


@pytest.mark.parametrize("hidden", [520, 521])
def test_norm_of_several_rows_to_a_workgroup(rt, hidden):   # noqa: F811
    """Rows of ordinary and of large values 2^20 rows apart, which a workgroup takes one after another; zeros between them."""
    step, rows = 1 << 20, (1 << 20) + 300
    some = [0, 1, 2, 299, step, step + 1, step + 2, rows - 1]
    x = data(torch.Generator().manual_seed(hidden), len(some), hidden)
    for i, size in enumerate([1.0, 1e25, 1.0, 1e25, 1e25, 1e25, 1.0, 1.0]):
        x[i] = (x[i].float() * size).to(BF16)
    xa, ya = rt.alloc(rows * hidden * 2), rt.alloc(rows * hidden * 2)
    try:
        rt.memset(xa, 0, rows * hidden * 2)
        rt.memset(ya, 0x55, rows * hidden * 2)
        for i, r in enumerate(some):
            rt.write(xa + 2 * r * hidden, raw(x[i].clone()))
        rt.rms_norm(t0g.rms_norm_desc(xa, 0, rows, hidden, y=ya))
        y = norm_of(x, None, None, 0.0, 1e-6)[2]
        for i, r in enumerate(some):
            got = torch.from_numpy(rt.read(ya + 2 * r * hidden, (hidden,), "int16")).view(BF16)
            near(got, y[i], (HALF[BF16] + NORM_REL) * y[i].abs(), f"row {r}")
        for r in (3, 298, 300, step - 1, step + 3, rows - 2):
            assert not rt.read(ya + 2 * r * hidden, (hidden,), "int16").any(), r
    finally:
        rt.wait_idle()
        rt.free(xa)
        rt.free(ya)


@pytest.mark.parametrize("hidden", [7, 300, 1000, 4096, 9001])
@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("qt", [E4, E5])
def test_norm_with_an_f32_residual_in_8_bits(rt, hidden, xt, qt):   # noqa: F811
    """s is the f32 sum, off by half a unit of itself, also where x and the residual cancel."""
    g = torch.Generator().manual_seed(hidden)
    x, r, w = data(g, 5, hidden, xt, 2.0), data(g, 5, hidden, F32, 2.0), data(g, 1, hidden, F32)[0]
    r[:, ::7] = -x[:, ::7].float() * (1 + 2.0 ** -10)
    b = Bufs(rt)
    (xa, _), (ra, _), (wa, _) = b.inp(x), b.inp(r), b.inp(w, True)
    (sa, _), (ya, _) = b.out("sum", x.shape, F32), b.out("y", x.shape, BF16)
    (qa, _), (ca, _) = b.out("q", x.shape, qt), b.out("scales", (blocks(hidden), 5), F32)
    f = t0g.F32
    rt.rms_norm(t0g.rms_norm_desc(xa, wa, 5, hidden, residual=ra, sum=sa, y=ya, q=qa, scales=ca, x_dtype=TYPES[xt], residual_dtype=f,
                                  weight_dtype=f, sum_dtype=f, q_dtype=TYPES[qt]))
    got = b.read()
    s, _, y = norm_of(x, r, w, 0.0, 1e-6)
    near(got["sum"], s, U * s.abs(), "sum")
    near(got["y"], y, (HALF[BF16] + NORM_REL + U) * y.abs(), "y")
    check_f8(got["q"], got["scales"], y, qt, slack=NORM_REL + U, what="q")


@pytest.mark.parametrize("rows,cols,want", [((1 << 22) + 3000, 8, "q"), ((1 << 22) + 3000, 7, "q"), ((1 << 23) + 3000, 2, "qt")])
def test_quantize_of_more_rows_than_a_launch_has(rt, rows, cols, want):   # noqa: F811
    x = data(torch.Generator().manual_seed(rows), rows, cols)
    b = Bufs(rt)
    xa, _ = b.inp(x)
    if want == "q":
        (qa, _), (ca, _) = b.out("q", (rows, cols), E4), b.out("scales", (1, rows), F32)
        d = t0g.fp8_quantize_desc(xa, qa, ca, rows, cols)
    else:
        (qa, _), (ca, _) = b.out("q", (cols, rows), E4), b.out("scales", (blocks(rows), cols), F32)
        d = t0g.fp8_quantize_desc(xa, 0, 0, rows, cols, qt=qa, scales_t=ca)
    rt.fp8_quantize(d)
    got = b.read()
    check_f8(got["q"], got["scales"], x.double() if want == "q" else x.double().t(), E4, what=want)


# ---- ends of rows -----------------------------------------------------------------------
ENDS = [n + r for n in (504, 520, 2040, 2048, 4088, 4096, 8184, 8192, 16376) for r in range(1, 9)]


@pytest.mark.parametrize("hidden", ENDS)
@pytest.mark.parametrize("xt,rt_,wt,yt,pad,offset", [(BF16, BF16, BF16, BF16, 0, 0), (F32, F32, F32, F32, 3, 1)])
def test_norm_at_every_end(rt, hidden, xt, rt_, wt, yt, pad, offset):   # noqa: F811
    """Last pieces of every length, on both sides of each kernel's limit."""
    base.test_norm(rt, 3, hidden, xt, rt_, wt, yt, pad, offset)


@pytest.mark.parametrize("hidden", ENDS)
@pytest.mark.parametrize("xt,yt,wt,st,pad,offset", [(BF16, BF16, BF16, BF16, 0, 0), (F32, BF16, F32, F32, 5, 1)])
def test_norm_backward_at_every_end(rt, hidden, xt, yt, wt, st, pad, offset):   # noqa: F811
    base.test_norm_backward(rt, 5, hidden, xt, yt, wt, st, pad, offset)


@pytest.mark.parametrize("cols", [n + r for n in (120, 248, 2040) for r in range(1, 17)])
@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("block", ["row", "tile"])
def test_quantize_at_every_end(rt, cols, xt, block):   # noqa: F811
    base.test_quantize(rt, 130 + cols % 16, cols, xt, E4, block, "q qt", 3, 1)


@pytest.mark.parametrize("n", range(57, 74))
@pytest.mark.parametrize("layout", ["NT", "NN"])
def test_gated_at_every_end(rt, n, layout):   # noqa: F811
    c = Gated(rt, n, n + 3, n + 7, layout, "silu", 3, 1, apart=True)
    c.forward(True)
    c.free()
    Gated(rt, n, n + 3, n + 7, layout, "silu", 1, 0, apart=True).backward(n % 2 == 0)


@pytest.mark.parametrize("rows", [1, 40, 2048])
@pytest.mark.parametrize("layout", ["NT", "NN"])
def test_gated_of_one_weight(rt, rows, layout):   # noqa: F811
    """Both projections by the same array."""
    f, hidden = (4096, 64) if rows == 2048 else (72, 136)
    c = Gated(rt, rows, f, hidden, layout, "silu", apart=True)
    c.wu, c.ua, c.u, c.eu = c.wg, c.ga, c.g, c.eg
    c.forward(True)
    if rows != 2048:
        c.backward(False)
    else:
        c.free()
