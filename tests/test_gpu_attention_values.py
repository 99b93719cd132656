"""Attention at the ends of f32: scores that overflow, and rows that see nothing.
(Inputs, 64-bit forms and tolerances: test_gpu_attention.py.)"""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, load
from test_gpu_attention import PAGE, Decode, Prefill, bf16, close

pytestmark = pytest.mark.gpu

LARGE = bf16(np.float32(3e38))[0]


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


def overflowing(c, row, pages=None):
    """The keys of a row's pages (all of them by default) give its queries scores
    that overflow f32 downwards: 3e38 * -32 * 64 * scale."""
    c.q[row, :, 0] = LARGE
    mine = c.table[row][c.table[row] >= 0]
    for at in mine if pages is None else mine[pages]:
        c.cache.k[at, :, :, 0], c.cache.s[at, :, 0] = 0xE0, 64.0


# one page, several of one workgroup, splits and joins of both kinds (of up to 16 splits, of more), ranked rows
@pytest.mark.parametrize("n, others", [(5, 0), (64, 3), (300, 0), (300, 40), (1500, 0), (8000, 1), (8000, 12), (1500, 100)])
@pytest.mark.parametrize("heads, kv, dim", [(8, 2, 128), (7, 1, 64)])
def test_decode_rows_whose_scores_all_overflow(env, n, others, heads, kv, dim):
    """The softmax of nothing but -inf is NaN, as in attention of prompts; a row
    that sees no token is 0."""
    c = Decode(n + others, [n, n, 0, n, *[n // 2 + 1] * others], heads, kv, dim)
    clean = c.run(env)
    c.q[1, :, 0] = 0            # a row's queries are its own: the others' pages stay
    overflowing(c, 0)
    c.table[3] = -1             # no page
    got = c.run(env)
    assert np.isnan(got[0]).all()
    assert np.all(got[2:4] == 0)
    assert np.array_equal(got[4:], clean[4:])
    c.q[0] = 0
    close(got[1:], *(a[1:] for a in c.want()))


@pytest.mark.parametrize("n", [200, 3000, 9000])
@pytest.mark.parametrize("finite", [[0], [1], [-1]])
def test_decode_one_page_of_finite_scores(env, n, finite):
    """Waves and splits whose scores all overflow weigh nothing beside one page's,
    and neither do pages that are not there."""
    c = Decode(n, [n, n], 4, 1, 128)
    count = -(-n // PAGE)
    keep = finite[0] % count
    overflowing(c, 0, [i for i in range(count) if i != keep])
    c.cache.k[c.table[0, keep], ..., 0] = 0
    c.table[1, [i for i in range(count) if i != keep]] = c.cache.pages
    c.check(env)


@pytest.mark.parametrize("n", [1, 40, 100, 700])
def test_prompt_rows_whose_scores_all_overflow(env, n):
    c = Prefill(n, [n + 70, 9], 4, 2, 64)
    clean = c.run(env)
    c.q[:n, :, 0], c.k[:n, :, 0] = LARGE, -LARGE
    c.q[n:n + 70, :, 0] = 0
    got = c.run(env)
    assert np.isnan(got[:n]).all()
    assert np.array_equal(got[n + 70:], clean[n + 70:])
    want, err = c.want()
    close(got[n:], want[n:], err[n:])


@pytest.mark.parametrize("n", [70, 3000])
def test_a_score_that_overflows_upwards(env, n):
    """+inf minus +inf: the row, and no other, is NaN."""
    c = Decode(n, [n, n], 4, 2, 64)
    clean = c.run(env)
    c.q[0, :, 0] = LARGE
    c.cache.k[c.table[0, n // PAGE], 0, 3, 0], c.cache.s[c.table[0, n // PAGE], 0, 0] = 0x70, 64.0
    c.cache.k[c.table[0], 1, :, 0] = 0      # the other head's stay finite
    got = c.run(env)
    assert np.isnan(got[0, :2]).all() and np.isfinite(got[0, 2:]).all()
    assert np.array_equal(got[1], clean[1])

    p = Prefill(n, [min(n, 700), 30], 4, 2, 64)
    at = 50
    p.q[at:, 1, 0], p.k[:, 0, 0] = LARGE, 0
    p.k[at, 0, 0] = LARGE
    p.q[:, 0, 0] = 0
    got = p.run(env)
    assert np.isnan(got[at:p.rows[0], 1]).all()
    got[at:p.rows[0], 1] = 0
    assert np.isfinite(got).all()
