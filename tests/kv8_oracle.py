"""The 8-bit K/V cache and its attention from their definitions, in 64 bits on the CPU (torch
tensors): what tests/test_gpu_kv8.py holds the kernels to."""
import math

import numpy as np
import torch

BLOCK = 64


def quantise(x):
    """x [64, D] fp16: codes float64, the scale fp32, and the block's values in fp16, as the cache
    gives them back (one fp32 product, rounded).  127 x / a is formed in 64 bits: its value is
    halfway between two codes only where the real number is."""
    x = x.double()
    if not bool(torch.isfinite(x).all()):
        return torch.zeros_like(x), float("nan"), torch.full_like(x, math.nan).half()
    a = max(float(x.abs().max()), 2.0 ** -24)
    codes = torch.round(x * 127 / a)
    scale = np.float32(a) / np.float32(127)
    return codes, float(scale), (codes.float() * torch.tensor(scale)).half()


class Head:
    """One head of one sequence: x [len, D] fp16 as given; values [len, D] as the cache holds them
    (full blocks: code * scale with the fp32 scale in 64 bits; open block: x)."""

    def __init__(self, x):
        self.x, self.n = x, x.shape[0]
        parts, self.codes, self.scales, read = [], [], [], []
        for i in range(self.n // BLOCK):
            c, s, r = quantise(x[i * BLOCK:(i + 1) * BLOCK])
            self.codes.append(c)
            self.scales.append(s)
            parts.append(c * s)
            read.append(r)
        rest = x[self.n // BLOCK * BLOCK:]
        self.steps = torch.cat([torch.full((BLOCK,), s, dtype=torch.float64) for s in self.scales] +
                               [torch.ones(len(rest), dtype=torch.float64)])  # of a key's values: v / step is what is multiplied
        self.values = torch.cat(parts + [rest.double()])
        self.read = torch.cat(read + [rest])  # fp16, bit for bit

    def summary(self, i):
        """The 8-bit sum of block i's codes and its fp32 scale."""
        c = self.codes[i].sum(0)
        big = max(float(c.abs().max()), 1.0)
        m = torch.round(127 * c / big)
        scale = (np.float32(self.scales[i]) * np.float32(big)) * np.float32(1.0 / (BLOCK * 127))
        return m, np.float32(scale)


def attend(q, K, V, steps, keys, scale, gate=None):
    """q [D], K, V [n, D] values in 64 bits, keys: the positions seen (a list, repeats count).  The
    output in 64 bits and the most that a kernel with fp16 weights and fp32 sums may be off,
    element by element, the output's own rounding included:
      weights       a rounding to fp16: 2^-11 of each.  What is rounded is p_j step_j in units where the
                    largest of a row is 2^12 or more, and what is multiplied v_j / step_j.  Below 2^-14
                    fp16's steps are 2^-24, so a weight may be off by 2^-25 whatever its size: that
                    is 2^-37 of the largest p_j step_j, times |v_j| / step_j, summed over the keys
      scores        an fp32 dot of D terms, the factor and log2 of the value scale: (D + 8) 2^-24 of
                    sum |q k| scale; and of the score itself, twice; exp2's argument and result: 2^-21
      sums          n terms in fp32: n 2^-23 at the most
      output        2^-11 of it, and half of fp16's smallest step; the gate 2^-20
    A weight's relative error e moves the output by at most e sum(p |v|), and as much again through
    the denominator (which is summed before the rounding: all but the first 2^-11)."""
    D = q.shape[0]
    if not keys:
        return torch.zeros(D, dtype=torch.float64), torch.full((D,), 2.0 ** -25, dtype=torch.float64)
    k, v, q, step = K[keys], V[keys], q.double(), steps[keys]
    s = (k @ q) * scale
    p = torch.exp(s - s.max())
    p = p / p.sum()
    o = p @ v
    size = p @ v.abs()
    ds = (D + 8) * 2.0 ** -24 * float((k.abs() @ q.abs()).max()) * scale + 2 ** -23 * float(s.abs().max()) + 2.0 ** -21
    tol = (2.0 ** -11 + 2 * (math.expm1(ds) + len(keys) * 2.0 ** -23)) * size
    tol = tol + 2.0 ** -37 * float((p * step).max()) * (v.abs() / step[:, None]).sum(0)
    if gate is not None:
        g = 1 / (1 + torch.exp(-gate.double()))
        o, tol = o * g, (tol + 2.0 ** -20 * o.abs()) * g
    return o, tol + 2.0 ** -11 * (o.abs() + tol) + 2.0 ** -25


def select(q, head, pos, top, first, recent, pages=None, scored=None):
    """q [G, D] fp16 of one group, head: Head of its keys; the blocks that the query at `pos` keeps.
    pages: which blocks have one; scored: blocks from this one on have no score."""
    if pos < 0:
        return []
    a = q.double().abs().max()
    ok = bool(torch.isfinite(q.double()).all())
    qc = torch.round(127 * q.double() / max(float(a), 2.0 ** -24)) if ok else torch.zeros_like(q.double())
    own, ranked = pos // BLOCK, []
    for i in range(own + 1):
        if i < first or i >= own - recent:
            rank = (2, np.float32(0))
        elif scored is not None and i >= scored:
            rank = (0, np.float32(0))
        elif pages is not None and not pages[i]:
            rank = (1, np.float32(-np.inf))
        else:
            m, scale = head.summary(i)
            score = np.float32(float((qc @ m).max())) * scale
            rank = (1, np.float32(-np.inf) if np.isnan(score) else score)
        ranked.append((rank[0], rank[1], -i))
    return sorted(-r[2] for r in sorted(ranked, reverse=True)[:top])
