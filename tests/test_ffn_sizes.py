"""Host side of the feed-forward layer's calls at their limits: the calls and their scratch queries refuse the same.  No GPU
needed."""
import pytest

import t0g
from test_ffn import call, refused

FAR = [i << 46 for i in range(1, 12)]   # arrays of any size do not meet


def gemm(m, n, k=64, **kw):
    return t0g.fp8_gemm_desc(*FAR[:5], m, n, k, **kw)


def gated(rows, features, hidden=64, **kw):
    return t0g.gated_linear_desc(*FAR[:4], rows, features, hidden, **kw)


def gated_backward(rows, features, hidden=64, **kw):
    return t0g.gated_linear_backward_desc(*FAR[:4], rows, features, hidden, dx=FAR[6], dwg=FAR[7], dwu=FAR[8], **kw)


def taken(d):
    """By the scratch query, and by the call up to its missing device."""
    t0g.ffn_scratch_size(d)
    with pytest.raises(t0g.T0gError, match="device is NULL"):
        call(d)


@pytest.mark.parametrize("over,below", [
    (gemm(1 << 20, 1 << 18), gemm((1 << 20) - 256, 1 << 18)),                                         # 2^22 tiles of 256 x 256
    (gemm(1 << 20, 1 << 16, out_dtype=t0g.F32), gemm((1 << 20) - 128, 1 << 16, out_dtype=t0g.F32)),   # of 128 x 128
    (gated(1 << 22, 1 << 15), gated((1 << 22) - 256, 1 << 15)),                                       # of 256 x 128
    (gated(1 << 25, 1 << 10), gated((1 << 25) - 256, 1 << 9)),                                        # x past 2^30 elements: of 128 x 64
    (gated_backward(1 << 20, 1 << 15), gated_backward((1 << 20) - 128, 1 << 15)),
])
def test_number_of_tiles(over, below):
    refused(over, "bad size")
    taken(below)


def test_backward_of_kept_products_has_no_tiles():
    d = gated_backward(1 << 20, 1 << 15, gate=FAR[9], up=FAR[10])
    taken(d)


# ---- scratch, to the byte ---------------------------------------------------------------
@pytest.mark.parametrize("m,n,k,kw,size", [
    (64, 512, 304, {}, 0),                                                  # whole 16-byte pieces, few stages of K
    (33, 512, 300, {}, 12800 + 512 * 384),                                  # both copied: rows of 384, each array to 256 bytes
    (64, 512, 300, {}, (64 + 512) * 384),
    (64, 512, 304, dict(lda=305), 64 * 384),                                # a's rows are not aligned
    (64, 512, 304, dict(a=FAR[0] + 8), 64 * 384),
    (64, 512, 304, dict(ldb=312), 512 * 384),
    (64, 512, 4096, {}, 8 * 64 * 512 * 4),                                  # eight slices of four stages
    (64, 510, 4100, {}, (64 + 510) * 4224 + 7 * 64 * 512 * 4),              # seven of five, planes of whole pieces of 4
    (2048, 4096, 304, {}, 0),
    (2048, 4096, 333, dict(out_dtype=t0g.F32), (2048 + 4096) * 384),
    (32, 512, 300, {}, 0),                                                  # few rows: no copy
])
def test_gemm_scratch(m, n, k, kw, size):
    d = gemm(m, n, k)
    for name, v in kw.items():
        setattr(d, name, v)
    assert t0g.ffn_scratch_size(d) == size


@pytest.mark.parametrize("hidden,rows,groups", [
    (512, 3, 1), (512, 100000, 1024), (513, 3, 3), (513, 100000, 1024), (2048, 1023, 1023), (2049, 100000, 1024), (4096, 100000, 1024),
    (4097, 100000, 512), (8192, 511, 511), (8192, 100000, 512), (8193, 100000, 256), (16384, 3, 3), (500, 4096, 1024), (500, 4000, 1000),
    (1, 1, 1), (1, 0, 0),
])
def test_norm_backward_scratch(hidden, rows, groups):
    """A row of dw for each workgroup (four rows to one up to 512 values), of whole pieces of 8."""
    d = t0g.rms_norm_backward_desc(*FAR[:3], rows, hidden, dx=FAR[4], dw=FAR[5])
    assert t0g.ffn_scratch_size(d) == groups * ((hidden + 7) // 8 * 8) * 4
    d.dw = 0
    assert t0g.ffn_scratch_size(d) == 0


def test_gated_scratch():
    assert t0g.ffn_scratch_size(gated(32, 512, 77)) == 0                     # few rows, NT
    assert t0g.ffn_scratch_size(gated(64, 512, 80)) == 0
    assert t0g.ffn_scratch_size(gated(64, 512, 77)) == (64 + 2 * 512) * 256  # rows of 128 values
    assert t0g.ffn_scratch_size(gated(64, 512, 77, ldw=80)) == (64 + 2 * 512) * 256
    assert t0g.ffn_scratch_size(gated(64, 512, 80, ldx=81)) == 64 * 256
    # 8 tiles, 64 stages of K in sixteen slices, two f32 planes each
    assert t0g.ffn_scratch_size(gated(64, 512, 4096)) == 16 * 2 * 64 * 512 * 4


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("kw", [dict(ldx=1 << 31), dict(ldw=1 << 31), dict(ldw=(1 << 32) - 1, ldx=(1 << 32) - 1)])
def test_backward_of_operands_that_no_memory_holds(layout, kw):
    """Refused before a product for each of their pieces is laid out."""
    rows, f, hidden = 1 << 24, (1 << 20) + 1, (1 << 20) + 1
    far = [i << 59 for i in range(1, 12)]
    d = t0g.gated_linear_backward_desc(*far[:4], rows, f, hidden, transpose=layout, gate=far[9], up=far[10], dx=far[6], dwg=far[7], dwu=far[8], **kw)
    refused(d, "bad size")
    d.rows, d.features, d.hidden = 300, 45, 9
    taken(d)
