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
