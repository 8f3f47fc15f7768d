#!/usr/bin/env python3
"""A small next-token model taught by a larger one, on one MI355X.

Teacher and student are a table of token vectors and a head onto the vocabulary.  The teacher's
logits come from one GEMM and its `top` largest of each position are kept; the student's step is one
t0g_linear_distill (divergence from those at a temperature, and the cross entropy of the next tokens),
which gives the loss and the gradients of its hidden states and of its head.  Tokens that neither
has trained on are scored with t0g_linear_cross_entropy.  Each step ignores some positions
(label -1 and no teacher's token), as padding would be.

    python3 distill_head.py --steps 60
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import t0g


class Adam:
    """f32 master weights on the host."""

    def __init__(self, w, lr):
        self.w, self.lr, self.t = w, lr, 0
        self.m, self.v = np.zeros_like(w), np.zeros_like(w)

    def step(self, g):
        self.t += 1
        self.m += 0.1 * (g - self.m)
        self.v += 0.01 * (g * g - self.v)
        m, v = self.m / (1 - 0.9 ** self.t), self.v / (1 - 0.99 ** self.t)
        self.w -= self.lr * m / (np.sqrt(v) + 1e-8)


class Device:
    """The few device buffers the loop needs, each allocated once."""

    def __init__(self, rt):
        self.rt, self.held = rt, {}

    def buf(self, name, nbytes):
        addr, size = self.held.get(name, (0, 0))
        if size < nbytes:
            if addr:
                self.rt.free(addr)
            addr = self.rt.alloc(nbytes)
            self.held[name] = (addr, nbytes)
        return addr

    def put(self, name, array):
        addr = self.buf(name, array.nbytes)
        self.rt.write(addr, array)
        return addr

    def bf16(self, name, array):
        """f32 values as bf16, converted on the device."""
        src = self.put(name + ".f32", np.ascontiguousarray(array, dtype=np.float32))
        dst = self.buf(name, array.size * 2)
        self.rt.f32_to_bf16(src, dst, array.size)
        return dst

    def close(self):
        for addr, _ in self.held.values():
            self.rt.free(addr)


class Bigrams:
    """The teacher: p(next | token) = softmax(table[token] head^T)."""

    def __init__(self, dev, vocab, width, rng):
        self.dev, self.vocab, self.width, self.rng = dev, vocab, width, rng
        self.table = rng.standard_normal((vocab, width), dtype=np.float32)
        self.head = dev.bf16("teacher.head", 3.0 * width ** -0.5 * rng.standard_normal((vocab, width), dtype=np.float32))

    def logits(self, tokens):
        n = len(tokens)
        x = self.dev.bf16("teacher.x", self.table[tokens])
        z = self.dev.buf("teacher.z", 4 * n * self.vocab)
        self.dev.rt.gemm(x, self.head, z, n, self.vocab, self.width, transpose="NT", out_dtype=t0g.F32)
        self.dev.rt.wait_idle()
        return self.dev.rt.read(z, (n, self.vocab), np.float32)

    def batch(self, n):
        """n tokens, the teacher's logits after them and a next token drawn from those."""
        tokens = self.rng.integers(0, self.vocab, n)
        z = self.logits(tokens)
        drawn = np.argmax(z + self.rng.gumbel(size=z.shape), axis=1)
        return tokens, z, drawn.astype(np.int64)


def run(rt, steps=60, rows=512, vocab=1000, width=128, teacher_width=32, top=32, temperature=2.0, lr=0.05, seed=1, log=print):
    """Trains for `steps` steps: (divergence-and-label loss a step, cross entropy of unseen tokens before and after)."""
    rng = np.random.default_rng(seed)
    dev = Device(rt)
    teacher = Bigrams(dev, vocab, teacher_width, rng)
    table = Adam(rng.standard_normal((vocab, width), dtype=np.float32), lr)
    head = Adam(0.1 * rng.standard_normal((vocab, width), dtype=np.float32), lr)
    held_tokens, _, held_next = teacher.batch(4 * rows)

    def score():
        n = len(held_tokens)
        loss = dev.buf("score", 4 * n)
        d = t0g.linear_ce_desc(dev.bf16("held.x", table.w[held_tokens]), dev.bf16("head", head.w), dev.put("held.next", held_next),
                               loss, n, vocab, width, logit_scale=width ** -0.5)
        rt.linear_cross_entropy(d)
        rt.wait_idle()
        return float(rt.read(loss, (n,), np.float32).mean(dtype=np.float64))

    def step():
        tokens, z, labels = teacher.batch(rows)
        best = np.argpartition(z, vocab - top, axis=1)[:, vocab - top:]
        kept = np.take_along_axis(z, best, axis=1)
        ignored = rng.random(rows) < 0.1
        labels[ignored], best[ignored] = -1, -1
        counted = rows - int(ignored.sum())
        out = dev.buf("loss", 4 * rows), dev.buf("dx", 4 * rows * width), dev.buf("dw", 4 * vocab * width)
        d = t0g.linear_distill_desc(dev.bf16("x", table.w[tokens]), dev.bf16("head", head.w), dev.put("kept", kept),
                                    dev.put("best", best.astype(np.int64)), out[0], rows, vocab, width, top,
                                    temperature=temperature, labels=dev.put("labels", labels), label_weight=0.5,
                                    distill_weight=0.5, dx=out[1], dw=out[2], dx_dtype=t0g.F32, dw_dtype=t0g.F32,
                                    loss_scale=1.0 / counted, logit_scale=width ** -0.5)
        rt.linear_distill(d)
        rt.wait_idle()
        loss, dx = rt.read(out[0], (rows,), np.float32), rt.read(out[1], (rows, width), np.float32)
        g = np.zeros_like(table.w)
        np.add.at(g, tokens, dx)
        table.step(g)
        head.step(rt.read(out[2], (vocab, width), np.float32))
        return float(loss.sum(dtype=np.float64)) / counted

    try:
        before, losses = score(), []
        log(f"unseen tokens: {before:.3f} nats before training")
        for i in range(steps):
            losses.append(step())
            if i % 10 == 0 or i == steps - 1:
                log(f"step {i:3d}: loss {losses[-1]:.3f}")
        after = score()
        log(f"unseen tokens: {after:.3f} nats after training, {np.log(vocab):.3f} by chance")
        return losses, before, after
    finally:
        rt.wait_idle()
        dev.close()


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--rows", type=int, default=512)
    p.add_argument("--vocab", type=int, default=1000)
    a = p.parse_args()
    with t0g.GpuRuntime.new(0) as runtime:
        run(runtime, steps=a.steps, rows=a.rows, vocab=a.vocab)
