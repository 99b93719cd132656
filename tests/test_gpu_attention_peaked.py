"""Attention where few tokens carry a row: over the cache, in some pages of every head a
key answers one of the head's queries, through columns and a page's scale of its own; in
prompts, scores spread over several units.  A wrong scale, a column, a page or a few
keys that are left out then move the output by far more than it may be off;
test_attention_inputs.py shows that, without a GPU.

Tolerance beside the BF16 rounding of the output: a score's sum of D products errs by at
most (D + 1) 2^-24 times the sum of their magnitudes, its exponent by 2^-22 of itself, a
probability in two BF16 parts by 2^-16, and the sums, of at most 1024 terms in a chain,
by 2^-14; numerator and denominator.  In prompts a probability is off by 2^-8, and so
is their sum, beside 2048 terms in a chain."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, load
from test_gpu_attention import E4M3, PAGE, Decode, Prefill, close, e4m3

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


PROMPTS = [(8, 2, 128, [1100]), (7, 1, 64, [700, 1, 450]), (4, 4, 64, [2000]), (1, 1, 128, [1500])]


class Spread(Prefill):
    def __init__(self, heads, kv, dim, rows):
        super().__init__(heads + dim + sum(rows), rows, heads, kv, dim, size=3.0)

    def want(self, scale=None, columns=None, without=None, heads_on=0, values_on=0):
        """As Peaked.want: also another head's keys, and other columns' values."""
        columns = columns or self.dim
        out, err = np.zeros((self.m, self.heads, self.dim)), np.zeros((self.m, self.heads, self.dim))
        group = self.heads // self.kv
        for lo, hi in zip(self.starts, self.starts[1:]):
            n = hi - lo
            if not n:
                continue
            unseen = np.triu(np.ones((n, n), bool), 1)
            if without is not None:
                unseen[:, without(np.arange(n))] = True
                unseen[np.arange(n), np.arange(n)] = False
            for h in range(self.heads):
                q = self.q[lo:hi, h, :columns].astype(np.float64) * self.dim ** -0.5
                k = self.k[lo:hi, (h // group + heads_on) % self.kv, :columns].astype(np.float64)
                v = np.roll(self.v[lo:hi, h // group].astype(np.float64), values_on, 1)
                s = q @ k.T
                off = (self.dim + 1) * 2.0 ** -24 * (np.abs(q) @ np.abs(k).T).max() + 2.0 ** -22 * np.abs(s).max()
                p = np.exp(np.where(unseen, -np.inf, s - np.where(unseen, -np.inf, s).max(1, keepdims=True)))
                total = p.sum(1, keepdims=True)
                out[lo:hi, h] = p @ v / total
                err[lo:hi, h] = 2 * (off + 2.0 ** -8 + 2.0 ** -13) * (p @ np.abs(v)) / total
        return out, err


@pytest.mark.parametrize("heads, kv, dim, rows", PROMPTS)
@pytest.mark.parametrize("empty", [0, 300])   # workgroups of 128 and of 256 rows
def test_prompts(env, heads, kv, dim, rows, empty):
    c = Spread(heads, kv, dim, [*rows, *[0] * empty])
    close(c.run(env), *c.want())
