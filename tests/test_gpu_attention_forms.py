"""Attention of prompts in workgroups of 128 and of 256 rows: which of the two runs
depends on how many a batch can have, and empty sequences count as one.  Attention
over the cache in the orders that its workgroups take rows and splits in.
(Inputs, 64-bit forms and tolerances: test_gpu_attention.py.)"""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, load
from test_gpu_attention import F32, PAGE, Decode, Prefill, bf16, close

pytestmark = pytest.mark.gpu

LAYOUTS = [(4, 1, 128), (2, 2, 64), (7, 1, 64), (8, 2, 128)]
SIZES = pytest.mark.parametrize("empty", [0, 300])


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


@SIZES
@pytest.mark.parametrize("heads, kv, dim", LAYOUTS)
@pytest.mark.parametrize("rows", [[1], [63, 0, 64, 65], [257, 130], [1100, 5]])
def test_prefill(env, heads, kv, dim, rows, empty):
    Prefill(len(rows) + heads, [*rows, *[0] * empty], heads, kv, dim, lead=1, behind=3).check(env)


@pytest.mark.parametrize("heads, kv, dim", [(32, 8, 128), (32, 32, 64)])
def test_prefill_fills_the_card(env, heads, kv, dim):
    Prefill(1, [2100], heads, kv, dim).check(env, starts=False)


@SIZES
@pytest.mark.parametrize("heads, kv, dim", LAYOUTS)
@pytest.mark.parametrize("n", [64, 127, 128, 129, 192, 513, 1500])
def test_every_key_counts_once(env, heads, kv, dim, n, empty):
    c = Prefill(2, [n, 5, *[0] * empty], heads, kv, dim)
    c.q[:] = 0
    c.v = np.random.default_rng(n).integers(-8, 9, c.v.shape).astype(F32)
    close(c.run(env), *c.want(exact=True))


@SIZES
@pytest.mark.parametrize("step", [30.0, -30.0, 9.0])
def test_scores_far_apart(env, step, empty):
    """The running maximum moves at every group of keys, or never again; what a
    row does not see is far above what it does."""
    c = Prefill(3, [500, *[0] * empty], 2, 1, 128)
    c.q[:] = 0
    c.k[:] = 0
    c.q[..., 0] = 1.0
    c.k[:, 0, 0] = bf16(np.arange(500) // 8 * step)
    # groups of eight equal scores: each probability is 1 or at most e^-9, and a sum's weight beside it below 2^-9
    got = c.run(env, scale=1.0)
    want, err = c.want(scale=1.0)
    close(got, want, err)


@SIZES
@pytest.mark.parametrize("heads, kv, dim", [(4, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("n, at", [(100, 99), (300, 70), (300, 200), (700, 400), (64, 0)])
def test_what_is_not_seen_does_not_count(env, heads, kv, dim, n, at, empty):
    c = Prefill(4, [n, 40, *[0] * empty], heads, kv, dim)
    clean = c.run(env)
    for which, x in ((c.v, np.nan), (c.v, np.inf), (c.v, -np.inf), (c.k, np.nan), (c.k, np.inf)):
        kept = which[at].copy()
        which[at, 0, 3] = x
        got = c.run(env)
        assert np.array_equal(got[:at], clean[:at])
        assert np.array_equal(got[n:], clean[n:])
        if np.isnan(x) or which is c.v:
            close(got, *c.want())
        which[at] = kept


@SIZES
@pytest.mark.parametrize("n", [40, 100])
def test_scores_of_minus_infinity_weigh_nothing(env, n, empty):
    """The first n keys' scores overflow f32 downwards."""
    c = Prefill(5, [n + 70, *[0] * empty], 4, 2, 64)
    c.q[:, :, 0], c.k[:n, :, 0], c.k[n:, :, 0] = bf16(np.float32(3e38)), bf16(np.float32(-3e38)), 0
    want, err = c.want()
    close(c.run(env)[n:], want[n:], err[n:])


@pytest.mark.parametrize("heads, kv, dim, m, most, width", [
    (16, 8, 128, 64, 900, None), (16, 8, 128, 33, 1100, None), (8, 8, 64, 16, 2050, None), (6, 3, 64, 50, 700, 70),
    (32, 8, 128, 8, 4096, None), (34, 2, 64, 20, 1500, None),          # ranked a lane each
    (8, 8, 128, 65, 600, None), (8, 8, 64, 200, 600, 12), (5, 5, 128, 256, 520, None),  # by the workgroup
    (8, 8, 64, 257, 600, None), (8, 8, 64, 64, 200, None), (2, 2, 64, 100, 2100, None)])  # in the order they have
def test_decode_orders(env, heads, kv, dim, m, most, width):
    """All kinds of lengths, many alike, none, negative ones and some beyond the table."""
    rng = np.random.default_rng(m)
    lengths = rng.integers(0, most + 1, m)
    lengths[rng.integers(0, m, m // 4)] = most // 2
    lengths[::7] = 0
    lengths[1], lengths[-1] = most, 1
    c = Decode(m, lengths.tolist(), heads, kv, dim, width=width)
    c.lengths[0] = -5
    if width is None:
        c.lengths[1] = c.width * PAGE + 100
        page = c.table[1, -1]   # its last page, seen to the end
        c.cache.k[page], c.cache.v[page] = 0x30, 0x31
    c.check(env)


def test_decode_orders_one_length(env):
    for n in (0, 640):
        c = Decode(1, [640] * 40, 8, 8, 64)
        c.lengths = [n] * 40
        c.check(env)


def test_decode_scores_of_minus_infinity_weigh_nothing(env):
    """A page's scores overflow f32 downwards."""
    c = Decode(2, [200, 130], 4, 2, 64)
    c.q[:, :, 0] = bf16(np.float32(3e38))
    c.cache.k[..., 0] = 0
    for row, page in ((0, 0), (1, 1)):
        at = c.table[row, page]
        c.cache.k[at, :, :, 0], c.cache.s[at, :, 0] = 0xF0, 64.0
    c.check(env)
