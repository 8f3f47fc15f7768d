"""8-bit products with values and scales that are infinite, zero or not a number: the same elements of the result are as in 64 bits, in
every kernel, and the others are untouched by them."""
import pytest
import torch

import t0g
from test_ffn_gpu import BF16, E4, E5, F32, HALF, TYPES, U, Bufs, blocks, f8_operand, largest8, spread, rt   # noqa: F401
from test_ffn_infinite_gates_gpu import same

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("m,n,k", [(6, 40, 300), (30, 200, 4200), (60, 300, 512), (90, 300, 2100), (2048, 4096, 272), (4096, 4096, 144)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("at,bt", [(E5, E4), (E4, E5), (E4, E4)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_special_values(rt, m, n, k, block, at, bt, out):   # noqa: F811
    g, tile = torch.Generator().manual_seed(m + k), block == "tile"
    (a, sa), (b, sb) = f8_operand(g, m, k, at, False), f8_operand(g, n, k, bt, tile)
    for v in (a, b):   # no zeros but the ones set below: an infinity times zero is none
        v.copy_(torch.where(v.float() == 0, torch.ones(()), v.float()).to(v.dtype))
    a.view(torch.uint8)[1, k - 1] = 0x7F                       # not a number, in both types
    b.view(torch.uint8)[3, 7] = 0xFF
    sa[0, 2], sa[blocks(k) - 1, 3], sa[:, 4] = INF, NAN, 0.0
    if at == E5:
        a.view(torch.uint8)[5, 130 % k] = 0x7C                 # infinities
    if bt == E5:
        b.view(torch.uint8)[6, 9] = 0xFC
    bufs = Bufs(rt)
    (aa, _), (ba, _), (sa_, _), (sb_, _) = bufs.inp(a), bufs.inp(b), bufs.inp(sa), bufs.inp(sb)
    ca, _ = bufs.out("c", (m, n), out)
    rt.fp8_gemm(t0g.fp8_gemm_desc(aa, sa_, ba, sb_, ca, m, n, k, a_dtype=TYPES[at], b_dtype=TYPES[bt],
                                  b_block=t0g.BLOCK_TILE if tile else t0g.BLOCK_ROW, out_dtype=TYPES[out]))
    got = bufs.read()["c"]
    # the definition: a block's products first, then the scales
    want = torch.zeros(m, n, dtype=torch.float64)
    bs = sb.double() if not tile else sb.double().repeat_interleave(128, dim=1)[:, :n]
    for i in range(blocks(k)):
        c = slice(128 * i, min(k, 128 * i + 128))
        want += sa[i].double()[:, None] * bs[i][None, :] * (a[:, c].double() @ b[:, c].double().t().contiguous())
    clean = lambda v, s, t: v.double().nan_to_num(0.0, 0.0, 0.0).abs() * spread(s.double().nan_to_num(0.0, 0.0, 0.0), v.shape, t)   # noqa: E731
    av, bv = clean(a, sa, False), clean(b, sb, tile)
    bound = 2 * (min(k, 128) + blocks(k) + 70) * U * (av @ bv.t())
    if out == BF16:
        bound += 7 * 2.0 ** -13 * (largest8(av) @ largest8(bv).t())
    bound = HALF[out] * (want.abs() + bound) + bound
    same(got, want, torch.where(torch.isnan(bound), torch.zeros_like(bound), bound), f"{m}x{n}x{k}")
