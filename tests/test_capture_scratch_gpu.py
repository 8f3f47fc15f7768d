"""Graphs captured from a handle's calls, replayed after larger calls made the handle's scratch buffers grow: the
blocks that the captured calls were given stay, so every replay gives the eager result's bits."""
import numpy as np
import pytest

import oracle as o
import t0g
from hip_rt import Graph, Stream

pytestmark = pytest.mark.gpu


def replays_after_growth(prepare):
    """prepare(h): (the call to capture, its output's address and size, a call that needs a larger scratch)."""
    h = t0g.GpuRuntime.new(0)
    s, g = Stream(), None
    try:
        h.set_stream(s.ptr)
        call, out, size, larger = prepare(h)
        call()
        h.wait_idle()
        want = h.read(out, (size,), np.uint8)
        g = Graph(s, call)
        before = t0g.device_alloc_count()
        larger()
        h.wait_idle()
        assert t0g.device_alloc_count() > before, "the larger call's scratch is not larger"
        filled = [h.alloc(n << 20) for n in (1, 2, 4, 8, 16, 32)]
        for n, addr in zip((1, 2, 4, 8, 16, 32), filled):
            h.memset(addr, 0xFF, n << 20)
        for replay in range(3):
            h.memset(out, 0xFF, size)
            g.launch(s)
            h.wait_idle()
            assert np.array_equal(h.read(out, (size,), np.uint8), want), f"replay {replay}"
            larger()
            h.wait_idle()
        h.set_stream(None)
    finally:
        if g is not None:
            g.destroy()
        h.close()
        s.destroy()


def bf16(h, rows, cols, seed):
    return h.upload(o.rand_bf16_lcg(rows * cols, seed))


@pytest.mark.parametrize("m,n,k,split", [(128, 4096, 4096, 2), (256, 512, 8192, 8), (100, 333, 5001, 4)])
def test_split_k_workspace(m, n, k, split):
    def prepare(h):
        a, b, c = bf16(h, m, k, 1), bf16(h, n, k, 2), h.alloc(m * n * 4)
        la, lb, lc = bf16(h, 2048, 4096, 3), bf16(h, 2048, 4096, 4), h.alloc(2048 * 2048 * 4)
        return (lambda: h.gemm(a, b, c, m, n, k, split_k=split), c, m * n * 4,
                lambda: h.gemm(la, lb, lc, 2048, 2048, 4096, split_k=8))
    replays_after_growth(prepare)


def test_group_workspaces():
    """Each stream of a group has a workspace of its own."""
    def prepare(h):
        m, n, k = 128, 512, 4096
        a, b, c = bf16(h, m, k, 5), bf16(h, n, k, 6), h.alloc(3 * m * n * 4)
        la, lb, lc = bf16(h, 1024, 4096, 7), bf16(h, 1024, 4096, 8), h.alloc(3 * 1024 * 1024 * 4)
        small = [t0g.gemm_desc(a, b, c + i * m * n * 4, m, n, k, split_k=4) for i in range(3)]
        large = [t0g.gemm_desc(la, lb, lc + i * 1024 * 1024 * 4, 1024, 1024, 4096, split_k=8) for i in range(3)]
        return lambda: h.gemm_group(small), c, 3 * m * n * 4, lambda: h.gemm_group(large)
    replays_after_growth(prepare)


def test_conversion_scratch():
    """An f32 layer whose operands are converted first."""
    def prepare(h):
        m, k, n = 2048, 2048, 512
        rng = np.random.default_rng(9)
        x, w = (h.upload(rng.uniform(-0.5, 0.5, s).astype(np.float32)) for s in ((m, k), (k, n)))
        y = h.alloc(m * n * 4)
        lx, lw = (h.upload(rng.uniform(-0.5, 0.5, s).astype(np.float32)) for s in ((4096, 2048), (2048, 4096)))
        ly = h.alloc(4096 * 4096 * 4)
        return (lambda: h.matmul_f32(x, w, y, m, k, n), y, m * n * 4, lambda: h.matmul_f32(lx, lw, ly, 4096, 2048, 4096))
    replays_after_growth(prepare)
