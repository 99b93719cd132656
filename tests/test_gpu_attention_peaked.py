"""Attention over the cache where few tokens carry a row: in some pages of every head a
key answers one of the head's queries, through columns and a page's scale of its own.
A wrong scale, a column or a page that is left out then moves the output by far more
than it may be off; test_attention_inputs.py shows that, without a GPU.

Tolerance beside the BF16 rounding of the output: a score's sum of D products errs by at
most (D + 1) 2^-24 times the sum of their magnitudes, its exponent by 2^-22 of itself, a
probability in two BF16 parts by 2^-16, and the sums, of at most 1024 terms in a chain,
by 2^-14; numerator and denominator."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, load
from test_gpu_attention import E4M3, PAGE, Decode, close, e4m3

pytestmark = pytest.mark.gpu

CASES = [(17, 1, 64, [2048]), (32, 8, 128, [2048]), (14, 2, 64, [2048]), (32, 8, 128, [2000, 4096]),
         (17, 1, 64, [4000, 500]), (16, 2, 128, [1420, 4052, 2600, 0, 3333, 1]), (14, 2, 64, [20000]),
         (8, 8, 64, [640, 64, 1200] * 11)]


class Peaked(Decode):
    def __init__(self, heads, kv, dim, lengths):
        super().__init__(heads + dim + sum(lengths), lengths, heads, kv, dim, size=1.0)
        rng, group = np.random.default_rng(len(lengths)), heads // kv
        for row, n in enumerate(lengths):
            for j in range(-(-n // PAGE)):
                page = self.table[row, j]
                for h in range(kv):
                    if rng.random() > 0.3 and n > 3 * PAGE:
                        continue
                    q = self.q[row, h * group + rng.integers(group)] * (rng.random(dim) < 0.5)
                    target = np.log(n) + rng.uniform(-3, 1)
                    size = target * dim ** 0.5 / (np.abs(q).sum() * float(self.cache.s[page, h, 0]))
                    slot = rng.integers(min(PAGE, n - PAGE * j))
                    self.cache.k[page, h, slot] = e4m3(np.sign(q) * min(size, 15.0))

    def want(self, key_scale=None, value_scale=None, columns=None, without=None):
        """Outputs and tolerances; the arguments plant mistakes: one scale for all pages, the
        first columns alone, pages left out."""
        c, group = self.cache, self.heads // self.kv
        columns = columns or self.dim
        out, err = np.zeros((self.m, self.heads, self.dim)), np.zeros((self.m, self.heads, self.dim))
        for i, n in enumerate(self.lengths):
            t = np.arange(n)
            if without is not None:
                t = t[~without(t // PAGE)]
            if not len(t):
                continue
            at, slot = self.table[i, t // PAGE], t % PAGE
            for h in range(self.heads):
                ks, vs = (np.full(len(t), float(x)) if x is not None else c.s[at, h // group, w].astype(np.float64)
                          for w, x in enumerate((key_scale, value_scale)))
                k = E4M3[c.k[at, h // group, slot]] * ks[:, None]
                v = E4M3[c.v[at, h // group, slot]] * vs[:, None]
                terms = k[:, :columns] * self.q[i, h, :columns].astype(np.float64) * self.dim ** -0.5
                s = terms.sum(1)
                p = np.exp(s - s.max())
                off = (self.dim + 1) * 2.0 ** -24 * np.abs(terms).sum(1).max() + 2.0 ** -22 * np.abs(s).max()
                out[i, h] = p @ v / p.sum()
                err[i, h] = 2 * (off + 2.0 ** -16 + 2.0 ** -14) * (p @ np.abs(v)) / p.sum()
        return out, err


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


@pytest.mark.parametrize("heads, kv, dim, lengths", CASES)
def test_decode(env, heads, kv, dim, lengths):
    c = Peaked(heads, kv, dim, lengths)
    close(c.run(env), *c.want())
