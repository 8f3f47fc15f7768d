"""8-bit values whose quotient lies on a border between two roundings go to the even neighbour, as in 64 bits.

For bf16 values a and amax = b, both of 8 significant bits, most a / b is either on a border (a number of at most 6
bits) or at least 1 / (2 b c) with b < 2^8, c < 2^6, that is 2^-14 of itself, away from every one; in f32 the quotient is
off by 2^-23 at most, so the 8 bits are determined and are compared bit for bit."""
import pytest
import torch

import t0g
from test_ffn_gpu import BF16, E4, E5, F32, MOST, TYPES, Bufs, blocks, data, rt, scales_of, spread   # noqa: F401

pytestmark = pytest.mark.gpu


def quotients(v, dtype, tile=False):
    """v most / amax in 64 bits: the product of two 8-bit numbers is exact, and a quotient on a border as well."""
    s = scales_of(v, dtype, tile) * MOST[dtype]
    return v * MOST[dtype] / spread(s, v.shape, tile)


def on_border(u, dtype):
    """Halfway between two neighbours of the type: f32's rounding of the quotient moved either way gives both."""
    u = u.float().double()
    up, down = ((u * (1 + s * 2.0 ** -20)).float().to(dtype).double() for s in (1, -1))
    return (up != down) & (u == (up + down) / 2)


def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("qt", [E4, E5])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("rows,cols", [(130, 4096), (200, 1001)])
def test_quantize_on_borders(rt, rows, cols, block, qt, xt):   # noqa: F811
    """f32 values that bf16 holds have the same quotients."""
    tile = block == "tile"
    x = data(torch.Generator().manual_seed(rows), rows, cols, BF16, 2.0)
    x[3, 5], x[4, 5] = 0.0, -0.0
    if not tile:   # one scale for a tile's 16384 values may leave none
        assert int(on_border(quotients(x.double(), qt), qt).sum()) >= 20
    both = {}
    for want in ("q", "q qt", "qt"):
        b = Bufs(rt)
        xa, _ = b.inp(x.to(xt))
        kw = dict(q=0, scales=0)
        if "q" in want.split():
            kw["q"], _ = b.out("q", (rows, cols), qt)
            kw["scales"], _ = b.out("scales", (blocks(cols), blocks(rows) if tile else rows), F32)
        if "qt" in want.split():
            kw["qt"], _ = b.out("qt", (cols, rows), qt)
            kw["scales_t"], _ = b.out("scales_t", (blocks(rows), blocks(cols) if tile else cols), F32)
        q, scales = kw.pop("q"), kw.pop("scales")
        rt.fp8_quantize(t0g.fp8_quantize_desc(xa, q, scales, rows, cols, x_dtype=TYPES[xt], q_dtype=TYPES[qt],
                                              block=t0g.BLOCK_TILE if tile else t0g.BLOCK_ROW, **kw))
        both[want] = b.read()
    for name, v in (("q", x.double()), ("qt", x.double().t())):
        want = quotients(v, qt, tile).float().to(qt)
        for got in both.values():
            if name in got:
                wrong = bits(got[name]) != bits(want)
                assert not bool(wrong.any()), f"{name}: {int(wrong.sum())} of {want.numel()} values"


@pytest.mark.parametrize("hidden", [384, 1000, 4096, 8200])
@pytest.mark.parametrize("qt", [E4, E5])
@pytest.mark.parametrize("wt,woff", [(None, 0.0), (BF16, 0.0), (F32, 0.0), (F32, 1.0)])
def test_norm_on_borders(rt, hidden, qt, wt, woff):   # noqa: F811
    """The norm's factor leaves the quotients, which are x (w + offset) most / amax: of 16 significant bits above and below (w + offset:
    of 8, in f32 as well), so that one that is on no border is 2^-22 of itself away and f32's rounding does not matter."""
    g = torch.Generator().manual_seed(hidden)
    rows = 300
    x = data(g, rows, hidden, BF16, 2.0)
    w = (1 + 0.1 * data(g, 1, hidden, F32)[0]).to(BF16) if wt else None
    if woff:
        w = (w.float() - woff).to(BF16)
        w = torch.where((w.float() + woff).to(BF16).float() == w.float() + woff, w, torch.zeros_like(w))
    b = Bufs(rt)
    (xa, _), (wa, _) = b.inp(x), b.inp(w.to(wt) if wt else None, True)
    (qa, _), (ca, _) = b.out("q", x.shape, qt), b.out("scales", (blocks(hidden), rows), F32)
    rt.rms_norm(t0g.rms_norm_desc(xa, wa, rows, hidden, q=qa, scales=ca, weight_offset=woff, weight_dtype=TYPES[wt or BF16], q_dtype=TYPES[qt]))
    u = quotients(x.double() * ((w.double() + woff) if wt else 1.0), qt)
    assert int(on_border(u, qt).sum()) >= 3
    wrong = bits(b.read()["q"]) != bits(u.float().to(qt))
    assert not bool(wrong.any()), f"{int(wrong.sum())} of {u.numel()} values"
