"""Attention at the ends of f32: scores that overflow, rows that see nothing, and
heads whose squares leave f32.
(Inputs, 64-bit forms and tolerances: test_gpu_attention.py.)"""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, load
from test_gpu_attention import F32, PAGE, Decode, Prefill, bf16, bf16_bits, close, dev, e4m3, from_bits, rope_table

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


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [np.uint16, np.float32])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("power, eps", [(0, 0.0), (-55, 0.0), (-64, 0.0), (-70, 0.0), (-100, 0.0), (-125, 0.0), (40, 0.0),
                                        (66, 0.0), (100, 0.0), (120, 1e-6), (-70, 2.0 ** -140), (-60, 2.0 ** -118),
                                        (-60, 1e-6), (-125, 1e-38), (0, 1e30), (30, 1e18), (0, 3e38), (100, 3e38)])
def test_heads_of_any_size_are_normalised(env, dim, dtype, packed, power, eps):
    """The squares' mean of finite heads may lie anywhere, below f32's normal numbers and above its largest."""
    mod, s, _ = env
    rng = np.random.default_rng(dim)
    heads, kv, m = 6, 2, 5
    x = np.ldexp(bf16(rng.standard_normal((m, heads + 2 * kv, dim))), power).astype(F32)
    x[1] = 0
    x[1, :, 3] = np.ldexp(F32(1.5), power)
    if dtype == np.uint16:
        x = bf16(x)   # subnormal ones have fewer bits
    gain, rope = [(1 + 0.3 * rng.standard_normal(dim)).astype(F32) for _ in range(2)], rope_table(m, dim)
    q, k = (dev(s, np.zeros(m * n * dim, np.uint16)) for n in (heads, kv))
    kw = dict(starts=dev(s, np.array([0, m], np.int32))) if packed else dict(past=dev(s, np.arange(m, dtype=np.int32)))
    mod.prepare_qk(s, dev(s, bf16_bits(x) if dtype == np.uint16 else x), heads, kv, dim, dev(s, rope), q,
                   q_gain=dev(s, gain[0]), k_gain=dev(s, gain[1]), k_out=k, eps=eps, **kw)
    for out, part, g in ((q, x[:, :heads], gain[0]), (k, x[:, heads:heads + kv], gain[1])):
        n = part.astype(np.float64)
        n = n / np.sqrt((n ** 2).mean(2, keepdims=True) + float(F32(eps))) * g.astype(np.float64)
        c, t, a, b = (z.astype(np.float64) for z in (rope[:, None, :dim // 2], rope[:, None, dim // 2:],
                                                     n[..., :dim // 2], n[..., dim // 2:]))
        want = np.concatenate([a * c - b * t, b * c + a * t], 2)
        size = np.concatenate([abs(a * c) + abs(b * t), abs(b * c) + abs(a * t)], 2)
        # below 2^-126 bf16's steps no longer shrink
        close(from_bits(out.to_host_vec(s)).reshape(want.shape), want, 2.0 ** -19 * size + 2.0 ** -134)


def test_a_head_of_zeros_without_eps(env):
    """0 / 0, as the formula has it; with any eps it is 0."""
    mod, s, _ = env
    x, rope, gain = dev(s, np.zeros(2 * 3 * 64, F32)), dev(s, rope_table(2, 64)), dev(s, np.ones(64, F32))
    out = dev(s, np.ones(2 * 64, np.uint16))
    for eps in (0.0, 1e-45, 1e-6):
        mod.prepare_qk(s, x, 1, 1, 64, rope, out, q_gain=gain, eps=eps)
        got = from_bits(out.to_host_vec(s))
        assert np.isnan(got).all() if eps == 0 else np.all(got == 0)


@pytest.mark.parametrize("heads, kv, dim", [(7, 1, 128), (14, 2, 64)])
@pytest.mark.parametrize("lengths", [[64], [500], [130, 500, 63], [4000, 2500]])
def test_decode_weights_have_more_bits_than_bf16(env, heads, kv, dim, lengths):
    """Two kinds of tokens whose values almost cancel: what is left shows the weights'
    roundings, which all tokens of a kind share.

    A weight in two BF16 parts is off by 2^-16, its exponent (below 2^3 here) by 2^-21 and
    v_exp_f32 by 2^-23; a sum has at most 512 terms in a chain (a wave's tokens, then the
    waves' and the splits' parts), so 2^-15. Numerator and denominator: 2^-13 of sum p |v|."""
    c = Decode(len(lengths) + sum(lengths), lengths, heads, kv, dim)
    c.cache.s[:] = 1
    c.q[:] = 0
    c.q[:, :, 0] = bf16(np.linspace(0.1, 2.2, heads))
    c.cache.k[:], c.cache.v[:] = 0, e4m3(-np.arange(dim) / dim)   # by column
    c.cache.k[:, :, ::2, 0], c.cache.v[:, :, ::2] = e4m3(-1.0), e4m3(1.0)
    want, err = c.want(scale=1.0)
    size = err / (2.0 ** -7 + 2.0 ** -9)
    assert np.all((np.abs(want) / size).min(2) < 2.0 ** -5)   # some column nearly cancels
    close(c.run(env, scale=1.0), want, 2.0 ** -13 * size)
