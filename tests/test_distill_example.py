"""The example that trains a small model from a larger one's logits (t0-gpu_amd/examples/distill_head.py): on the
GPU, and on a stand-in for the runtime in numpy that holds the losses' definitions."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "t0-gpu_amd", "examples"))
import distill_head
import t0g


def _softmax(z):
    e = np.exp(z - z.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


class Numpy:
    """The runtime's calls that the example makes; an address is a buffer's number."""

    def __init__(self):
        self.mem, self.live, self.last = {}, set(), 0

    def alloc(self, nbytes):
        self.last += 1
        self.live.add(self.last)
        return self.last

    def free(self, addr):
        self.live.remove(addr)

    def wait_idle(self):
        pass

    def write(self, addr, array):
        self.mem[addr] = array.copy()

    def read(self, addr, shape, dtype):
        return self.mem[addr].reshape(shape).astype(dtype)

    def f32_to_bf16(self, src, dst, n):
        u = self.mem[src].view(np.uint32)
        self.mem[dst] = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)

    def gemm(self, a, b, c, m, n, k, **kw):
        assert kw["transpose"] == "NT"
        self.mem[c] = self.mem[a].reshape(m, k) @ self.mem[b].reshape(n, k).T

    def head(self, d):
        x = self.mem[d.x].reshape(d.rows, d.hidden).astype(np.float64)
        w = self.mem[d.w].reshape(d.vocab, d.hidden).astype(np.float64)
        return x, w, d.logit_scale * (x @ w.T)

    def linear_cross_entropy(self, d):
        z = self.head(d)[2]
        self.mem[d.loss] = -np.log(_softmax(z)[np.arange(d.rows), self.mem[d.labels]])

    def linear_distill(self, dd):
        d, tau = dd.head, dd.temperature
        x, w, z = self.head(d)
        labels, tokens = self.mem[d.labels], self.mem[dd.tokens]
        p, pt, q = _softmax(z), _softmax(z / tau), _softmax(self.mem[dd.teacher].astype(np.float64) / tau)
        loss, g = np.zeros(d.rows), np.zeros_like(z)
        for t in range(d.rows):
            if labels[t] < 0:
                continue
            a, b = dd.label_weight, dd.distill_weight
            loss[t] = -a * np.log(p[t, labels[t]]) + b * tau ** 2 * (q[t] * np.log(q[t] / pt[t, tokens[t]])).sum()
            g[t] = a * p[t] + b * tau * pt[t]
            g[t, labels[t]] -= a
            g[t, tokens[t]] -= b * tau * q[t]
        g *= d.loss_scale * d.logit_scale
        self.mem[d.loss], self.mem[d.dx], self.mem[d.dw] = loss, g @ w, g.T @ x


def test_trains_on_the_definitions():
    rt = Numpy()
    losses, before, after = distill_head.run(rt, steps=40, log=lambda m: None)
    assert abs(before - np.log(1000)) < 0.05      # a head of small weights: every token alike
    assert after < before - 1 and losses[-1] < 0.7 * losses[0], (before, after, losses[0], losses[-1])
    assert not rt.live


@pytest.mark.gpu
def test_trains_on_the_gpu():
    """The same run on the device.  Its first loss and the first score come from equal inputs: f32 losses of logits
    that are exact to 2^-24 (128 + 2) sum |x||w| / 11 < 1e-3; later steps differ by bf16 roundings of G that Adam
    can enlarge, so of those only what training has to reach is asked."""
    _, before_np, _ = distill_head.run(Numpy(), steps=0, log=lambda m: None)
    first_np = distill_head.run(Numpy(), steps=1, log=lambda m: None)[0][0]
    with t0g.GpuRuntime.new(0) as rt:
        losses, before, after = distill_head.run(rt, steps=40)
    assert abs(before - before_np) < 1e-3 and abs(losses[0] - first_np) < 1e-3 * first_np
    assert after < before - 1 and losses[-1] < 0.7 * losses[0], (before, after, losses[0], losses[-1])
