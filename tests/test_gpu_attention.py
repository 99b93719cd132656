"""Attention between the qkv and the o projection against plain 64-bit forms:
head norms, rotation and the append to the paged 8-bit cache, attention of whole
prompts, attention over the cache and copies of pages, at the sizes, masks and
values where they can go wrong.

Tolerances.  A BF16 output is off by at most 2^-8 of its value beside the error
err of what was rounded: |got - want| <= 2^-8 (|want| + err) + err.
* prepare_qk: a sum of squares in a tree over 64 or 128 terms, v_rsq_f32 (one
  unit), three products and a rotation: fewer than 32 roundings of 2^-24, so err is
  2^-19 (|a cos| + |b sin|).  A code is off by half a step of e4m3: 2^-4 of the
  value, or 2^-10 of the scale among the subnormals.
* Attention: each probability is off by 2^-8 (BF16) and by twice the error of
  its score, and so is their sum: err is (2 * 2^-8 + d) sum p |v| / sum p.  A
  score's sums of 64 or 128 products err by at most 129 * 2^-24 times the sum of their
  magnitudes, which the inputs keep below 2^6 (2^-11), the exponent by 2^-24 of itself
  (below 2^7), the f32 sums over at most 2^13 keys by 2^-11: d = 2^-9 covers them.
* With equal scores and whole-numbered values every probability is 1 and every
  sum exact: err is 2^-22 of the quotient, which a wrong key or length exceeds."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, DeviceBuffer, Graph, KvCache, load

pytestmark = pytest.mark.gpu

F32 = np.float32
PAGE = 64


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


def dev(s, a):
    return DeviceBuffer.from_host(s, np.ascontiguousarray(a).reshape(-1))


def bf16_bits(a):
    a = np.ascontiguousarray(a, F32)
    u = a.view(np.uint32).astype(np.uint64)
    return np.where(np.isnan(a), 0x7FC0, (u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bits(b):
    return (b.astype(np.uint32) << 16).view(F32)


def bf16(a):
    return from_bits(bf16_bits(a))


def values(buf, s):
    a = buf.to_host_vec(s)
    return from_bits(a) if a.dtype == np.uint16 else a


def close(got, want, err):
    """Within a BF16 rounding of want +- err; the same NaN and infinities."""
    got = got.astype(np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:4]
    odd = ~fine & ~np.isnan(want)
    assert np.array_equal(got[odd], want[odd])
    bound = 2.0 ** -8 * (np.abs(want) + err) + err
    bad = fine & ~(np.abs(got - np.where(fine, want, 0)) <= np.where(fine, bound, np.inf))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], bound[bad][:4])


# ------------------------------------------------------------------ e4m3
def _table():
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


E4M3 = _table()
STEPS = E4M3[:127]  # the non-negative ones, rising


def e4m3(x):
    """Codes of values up to 448, nearest, ties to the even code; NaN where not finite."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(STEPS, a), 1, 126)
    lo = hi - 1
    up = (a - STEPS[lo] > STEPS[hi] - a) | ((a - STEPS[lo] == STEPS[hi] - a) & (hi % 2 == 0))
    code = np.where(up, hi, lo) | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def scale_for(top):
    with np.errstate(divide="ignore"):
        return np.exp2(np.maximum(np.ceil(np.log2(np.asarray(top, np.float64) / 448.0)), -100.0))


def test_e4m3_table_rounds_to_itself():
    ok = ~np.isnan(E4M3)
    assert np.array_equal(e4m3(E4M3[ok]), np.arange(256)[ok])


class Cache:
    """One layer on the host: keys and values as [pages, kv, 64, dim]."""

    def __init__(self, rng, pages, kv, dim, fill=0x7F):
        self.pages, self.kv, self.dim = pages, kv, dim
        self.k = np.full((pages, kv, PAGE, dim), fill, np.uint8)   # NaN where nothing was written
        self.v = self.k.copy()
        self.s = np.exp2(rng.integers(-6, -2, (pages, kv, 2))).astype(F32)

    def random(self, rng):
        draw = lambda: rng.integers(0, 256, self.k.shape).astype(np.uint8)  # noqa: E731
        self.k, self.v = draw(), draw()
        for a in (self.k, self.v):
            a[(a & 127) >= 0x58] &= 0xCF   # up to 15 and without NaN
        return self

    def codes(self):
        k, v = self.k.reshape(self.pages, self.kv, -1), self.v.transpose(0, 1, 3, 2).reshape(self.pages, self.kv, -1)
        return np.stack([k, v], 2)

    def put(self, s):
        return KvCache.over(dev(s, self.codes()), dev(s, self.s), 1, self.pages, self.kv, self.dim)

    def read(self, cache, s):
        c = cache.codes.to_host_vec(s).reshape(self.pages, self.kv, 2, -1)
        k = c[:, :, 0].reshape(self.k.shape)
        v = c[:, :, 1].reshape(self.pages, self.kv, self.dim, PAGE).transpose(0, 1, 3, 2)
        return k, v, cache.scales.to_host_vec(s).reshape(self.s.shape)


# ------------------------------------------------------------------ prepare_qk
def rope_table(rows, dim):
    a = np.arange(rows)[:, None] * 1e4 ** (-np.arange(dim // 2) * 2.0 / dim)
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(F32)


class Prepare:
    def __init__(self, seed, rows, past, heads, kv, dim, lead=0, behind=0, width=None, norm=True, gap=0):
        rng = self.rng = np.random.default_rng(seed)
        self.rows, self.past, self.heads, self.kv, self.dim = rows, past, heads, kv, dim
        self.m = lead + sum(rows) + behind
        self.starts = np.concatenate([[lead], lead + np.cumsum(rows)]).astype(np.int32)
        self.x = bf16(rng.standard_normal((self.m, heads + 2 * kv, dim)))
        self.x[:, :, 5::31] *= 8
        self.gains = [1 + 0.3 * rng.standard_normal(dim).astype(F32) if norm else None for _ in range(2)]
        self.rope = rope_table(max([1, *(p + n for p, n in zip(past, rows))]) - gap, dim)
        counts = [-(-(p + n) // PAGE) for p, n in zip(past, rows)]
        self.width = max(1, *counts) if width is None else width
        self.cache = Cache(rng, sum(counts) + 2, kv, dim)
        order, self.table = rng.permutation(self.cache.pages), np.full((len(rows), max(1, *counts)), -1, np.int32)
        at = 0
        for i, c in enumerate(counts):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.table = np.ascontiguousarray(self.table[:, :self.width])
        for i, p in enumerate(past):   # earlier tokens
            for t in range(min(p, self.width * PAGE)):
                page = self.table[i, t // PAGE]
                self.cache.k[page, :, t % PAGE] = rng.integers(0, 0x70, (kv, dim))
                self.cache.v[page, :, t % PAGE] = rng.integers(0x80, 0xF0, (kv, dim))

    def rotated(self, which, rows, positions):
        """n rotated in 64 bits, and the sum of magnitudes."""
        lo, hi = (0, self.heads) if which == 0 else (self.heads, self.heads + self.kv)
        x = self.x[rows, lo:hi].astype(np.float64)
        if self.gains[which] is not None:
            x = x / np.sqrt((x ** 2).mean(2, keepdims=True) + 1e-6) * self.gains[which].astype(np.float64)
        half = self.dim // 2
        known = (positions < len(self.rope))[:, None, None]
        turn = self.rope[np.minimum(positions, len(self.rope) - 1)].astype(np.float64)[:, None]
        c, s, a, b = turn[..., :half], turn[..., half:], x[..., :half], x[..., half:]
        out = np.concatenate([a * c - b * s, b * c + a * s], 2)
        size = np.concatenate([abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)], 2)
        return np.where(known, out, np.nan), size

    def run(self, env, dtype=np.uint16, fused=True, outs=True, cached=True, one_row=False, stream=None):
        mod, s, _ = env
        s = stream or s
        put = lambda a: dev(s, bf16_bits(a) if dtype == np.uint16 else a.astype(F32))  # noqa: E731
        h, kv = self.heads, self.kv
        kw = {}
        if fused:
            q = put(self.x)
        else:
            q, kw["k"], kw["v"] = put(self.x[:, :h]), put(self.x[:, h:h + kv]), put(self.x[:, h + kv:])
        full = lambda heads: dev(s, np.full(self.m * heads * self.dim, 0x4242, np.uint16))  # noqa: E731
        self.q_out, self.k_out, self.v_out = full(h), full(kv), full(kv)
        if outs:
            kw.update(k_out=self.k_out, v_out=self.v_out)
        for name, gain in zip(("q_gain", "k_gain"), self.gains):
            if gain is not None:
                kw[name] = dev(s, gain)
        if cached:
            self.held = self.cache.put(s)
            kw.update(cache=self.held, table=dev(s, self.table))
        if any(self.past):
            kw["past"] = dev(s, np.array(self.past, np.int32))
        if not one_row:
            kw["starts"] = dev(s, self.starts)
        mod.prepare_qk(s, q, h, kv, self.dim, dev(s, self.rope), self.q_out, **kw)
        return s

    def check(self, s, outs=True, cached=True):
        m, h, kv, dim = self.m, self.heads, self.kv, self.dim
        shape = lambda b, heads: b.to_host_vec(s).reshape(m, heads, dim)  # noqa: E731
        q, k, v = shape(self.q_out, h), shape(self.k_out, kv), shape(self.v_out, kv)
        touched = np.zeros(m, bool)
        codes_k, codes_v, scales = self.cache.read(self.held, s) if cached else (None,) * 3
        want_k, want_v, want_s = self.cache.k.copy(), self.cache.v.copy(), self.cache.s.copy()
        new = np.zeros(want_k.shape, bool)
        for i, (n, p) in enumerate(zip(self.rows, self.past)):
            rows = np.arange(self.starts[i], self.starts[i] + n)
            touched[rows] = True
            pos = p + np.arange(n)
            want, size = self.rotated(0, rows, pos)
            close(from_bits(q[rows]), want, 2.0 ** -19 * size)
            y, size = self.rotated(1, rows, pos)
            if outs:
                close(from_bits(k[rows]), y, 2.0 ** -19 * size)
                assert np.array_equal(v[rows], bf16_bits(self.x[rows, h + kv:]))
            if not cached or n == 0:
                continue
            value = self.x[rows, h + kv:].astype(np.float64)
            for page in range(p // PAGE, (p + n - 1) // PAGE + 1):
                if page >= self.width or not 0 <= self.table[i, page] < self.cache.pages:
                    continue
                at, lo, hi = self.table[i, page], max(p, page * PAGE), min(p + n, (page + 1) * PAGE)
                a, b = lo - page * PAGE, hi - page * PAGE
                for which, (z, zs) in enumerate(((y, size), (value, 0 * value))):
                    part = np.where(np.isfinite(z[lo - p:hi - p]), z[lo - p:hi - p], 0)
                    need = scale_for(np.abs(part).max((0, 2)))
                    was = want_s[at, :, which].astype(np.float64) if a else np.zeros(kv)
                    now = np.maximum(need, was)
                    want_s[at, :, which] = now
                    codes = want_k if which == 0 else want_v
                    codes[at, :, :a] = e4m3(E4M3[codes[at, :, :a]] * (was / now)[:, None, None])
                    got = (codes_k if which == 0 else codes_v)[at, :, a:b].transpose(1, 0, 2)
                    new[at, :, a:b] = True
                    bad = ~np.isfinite(z[lo - p:hi - p])
                    assert np.all((got[bad] & 127) == 127)
                    dec, step = E4M3[got] * now[None, :, None], now[None, :, None]
                    bound = np.maximum(2.0 ** -4 * np.abs(part), 2.0 ** -10 * step) + 2.0 ** -18 * zs[lo - p:hi - p]
                    assert np.all((np.abs(dec - part) <= bound)[~bad])
        for got in (q, k, v) if outs else (q,):
            assert np.all(got[~touched] == 0x4242)
        if not outs:
            assert np.all(k == 0x4242) and np.all(v == 0x4242)
        if cached:
            assert np.array_equal(scales.astype(np.float64), want_s.astype(np.float64))
            assert np.array_equal(codes_k[~new], want_k[~new])
            assert np.array_equal(codes_v[~new], want_v[~new])


LAYOUTS = [(4, 4, 128), (32, 8, 128), (14, 2, 64), (5, 1, 128), (3, 3, 64)]


@pytest.mark.parametrize("heads, kv, dim", LAYOUTS)
@pytest.mark.parametrize("rows, past", [([1], [0]), ([1, 1, 1], [63, 64, 700]), ([64], [0]), ([65, 0, 1], [1, 5, 127]),
                                        ([130, 62, 3], [0, 2, 62]), ([7], [61])])
@pytest.mark.parametrize("dtype, fused", [(np.uint16, True), (np.float32, False)])
def test_prepare(env, heads, kv, dim, rows, past, dtype, fused):
    c = Prepare(hash((heads, dim, sum(rows))) % 1000, rows, past, heads, kv, dim)
    c.check(c.run(env, dtype, fused))


@pytest.mark.parametrize("m", [1, 3, 200])
def test_prepare_one_row_each(env, m):
    rng = np.random.default_rng(m)
    c = Prepare(m, [1] * m, rng.integers(0, 300, m).tolist(), 8, 2, 128)
    c.check(c.run(env, one_row=True, outs=False), outs=False)


def test_prepare_many_sequences(env):
    rng = np.random.default_rng(5)
    rows = rng.integers(0, 6, 301).tolist()
    c = Prepare(7, rows, rng.integers(0, 200, 301).tolist(), 4, 1, 64)
    c.check(c.run(env))


def test_prepare_leaves_rows_of_no_sequence(env):
    c = Prepare(11, [3, 70], [0, 9], 4, 2, 128, lead=2, behind=5)
    c.check(c.run(env))


def test_prepare_without_norm_outputs_or_cache(env):
    c = Prepare(12, [67], [3], 6, 3, 64, norm=False)
    c.check(c.run(env, np.float32, cached=False), cached=False)
    c.check(c.run(env, outs=False), outs=False)


def test_prepare_position_behind_the_rotations(env):
    c = Prepare(13, [5], [60], 2, 1, 128, gap=2)
    c.check(c.run(env))


def test_prepare_beyond_the_table_and_bad_pages(env):
    c = Prepare(14, [100, 10], [40, 0], 2, 2, 128, width=1)
    c.check(c.run(env))
    c = Prepare(15, [100, 10], [40, 0], 2, 2, 128)
    c.table[0, 0], c.table[1, 0] = -1, c.cache.pages
    c.check(c.run(env))


@pytest.mark.parametrize("grow", [0.0, 1e-30, 1.0, 100.0, 1e30])
def test_prepare_scale_grows(env, grow):
    c = Prepare(16, [9], [30], 4, 2, 128, norm=False)
    c.x *= F32(grow)
    c.x = bf16(c.x)
    c.check(c.run(env))


def test_prepare_values_that_are_not_finite(env):
    c = Prepare(17, [70], [10], 4, 2, 128, norm=False)
    kv = c.x[:, 4:]
    kv[3, 2, 7], kv[40, 3, 100], kv[69, 0, 1] = np.nan, np.inf, -np.inf
    c.x[5, 0, 9] = np.nan
    c.check(c.run(env))


def test_prepare_twice_is_once(env):
    c = Prepare(18, [9, 80], [30, 5], 4, 2, 128)
    s = c.run(env)
    first = [b.to_host_vec(s) for b in (c.q_out, c.held.codes, c.held.scales)]
    held = c.held
    c.cache.put = lambda _: held
    c.run(env)
    assert all(np.array_equal(a, b.to_host_vec(s)) for a, b in zip(first, (c.q_out, held.codes, held.scales)))


# ------------------------------------------------------------------ attention of prompts
def softmax_sums(scores, v):
    """o and sum p |v| / sum p of scores [..., q, k] (-inf: not seen) and v [k, d]."""
    top = scores.max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        p = np.exp(scores - np.where(np.isneginf(top), 0, top))
        total = p.sum(-1, keepdims=True)
        seen = ~np.isneginf(scores)
        o = np.zeros(scores.shape[:-1] + v.shape[-1:])
        bad = ~np.isfinite(v)
        o += np.matmul(p, np.where(bad, 0, v))
        for j in np.unique(np.argwhere(bad)[:, 0]):
            o += np.where(seen[..., j, None], p[..., j, None] * np.where(bad[j], v[j], 0.0), 0.0)
        size = np.matmul(p, np.where(bad, 0, np.abs(v)))
        return o / total, np.nan_to_num(size / total, posinf=0.0)


class Prefill:
    def __init__(self, seed, rows, heads, kv, dim, lead=0, behind=0, size=1.0):
        rng = np.random.default_rng(seed)
        self.rows, self.heads, self.kv, self.dim = rows, heads, kv, dim
        self.m = lead + sum(rows) + behind
        self.starts = np.concatenate([[lead], lead + np.cumsum(rows)]).astype(np.int32)
        self.q = bf16(size * rng.standard_normal((self.m, heads, dim)))
        self.k = bf16(rng.standard_normal((self.m, kv, dim)))
        self.v = bf16(rng.standard_normal((self.m, kv, dim)))

    def run(self, env, dtype=np.uint16, starts=True, strided=False, scale=None, stream=None):
        mod, s, _ = env
        s = stream or s
        out = dev(s, np.full(self.m * self.heads * self.dim, 0x4242 if dtype == np.uint16 else 7.0, dtype))
        v, kw = dev(s, bf16_bits(self.v)), {}
        if strided:
            wide = np.zeros((self.m, 3 * self.kv, self.dim), F32)
            wide[:, self.kv:2 * self.kv] = self.v
            whole = dev(s, bf16_bits(wide))
            n = self.kv * self.dim
            v, kw = DeviceBuffer.view_of(whole, n, (self.m - 1) * 3 * n + n), {"v_stride": 3 * n}
        mod.attention_prefill(s, dev(s, bf16_bits(self.q)), dev(s, bf16_bits(self.k)), v, self.heads, self.kv, self.dim,
                              out, starts=dev(s, self.starts) if starts else None, scale=scale, **kw)
        return values(out, s).reshape(self.m, self.heads, self.dim)

    def want(self, scale=None, exact=False):
        out, err = np.full((self.m, self.heads, self.dim), np.nan), np.zeros((self.m, self.heads, self.dim))
        group = self.heads // self.kv
        for lo, hi in zip(self.starts, self.starts[1:]):
            n = hi - lo
            if n == 0:
                continue
            later = np.triu(np.ones((n, n), bool), 1)
            for h in range(self.heads):
                k, v = self.k[lo:hi, h // group].astype(np.float64), self.v[lo:hi, h // group].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    s = self.q[lo:hi, h].astype(np.float64) @ k.T * (self.dim ** -0.5 if scale is None else scale)
                s[later] = -np.inf
                out[lo:hi, h], err[lo:hi, h] = softmax_sums(s, v)
        return out, 2.0 ** -22 * np.abs(np.nan_to_num(out)) if exact else (2.0 ** -7 + 2.0 ** -9) * err

    def check(self, env, **kw):
        got = self.run(env, **kw)
        want, err = self.want(kw.get("scale"))
        inside = np.zeros(self.m, bool)
        inside[self.starts[0]:self.starts[-1]] = True
        close(got[inside], want[inside], err[inside])
        left = values_of(kw.get("dtype", np.uint16))
        assert np.all(got[~inside] == left)


def values_of(dtype):
    return from_bits(np.array([0x4242], np.uint16))[0] if dtype == np.uint16 else F32(7.0)


@pytest.mark.parametrize("heads, kv, dim", [*LAYOUTS, (16, 1, 64), (24, 1, 128), (6, 2, 128)])
@pytest.mark.parametrize("rows", [[1], [2, 0, 1, 33], [63, 64, 65], [257]])
def test_prefill(env, heads, kv, dim, rows):
    Prefill(hash((heads, dim, sum(rows))) % 1000, rows, heads, kv, dim).check(env)


@pytest.mark.parametrize("dtype, strided, starts", [(np.float32, False, True), (np.uint16, True, False)])
def test_prefill_outputs_and_strides(env, dtype, strided, starts):
    Prefill(3, [130], 8, 2, 128).check(env, dtype=dtype, strided=strided, starts=starts)
    Prefill(4, [70], 4, 4, 64).check(env, dtype=dtype, strided=strided, starts=starts, scale=0.3)


def test_prefill_leaves_rows_of_no_sequence(env):
    Prefill(5, [40, 0, 0, 90], 4, 2, 128, lead=3, behind=70).check(env)


def test_prefill_many_sequences(env):
    rows = np.random.default_rng(6).integers(0, 9, 200).tolist()
    Prefill(6, rows, 4, 2, 64).check(env)


@pytest.mark.parametrize("rows", [[1500], [700, 1, 900]])
@pytest.mark.parametrize("heads, kv, dim", [(4, 1, 128), (2, 2, 64), (7, 1, 64)])
def test_prefill_longer(env, rows, heads, kv, dim):
    Prefill(7, rows, heads, kv, dim).check(env)


@pytest.mark.parametrize("heads, kv, dim", [(4, 1, 128), (3, 1, 64), (1, 1, 128)])
@pytest.mark.parametrize("n", [1, 31, 64, 200, 513, 2100])
def test_prefill_counts_every_key_once(env, heads, kv, dim, n):
    c = Prefill(8, [n, 5], heads, kv, dim)
    c.q[:] = 0
    c.v = np.random.default_rng(n).integers(-8, 9, c.v.shape).astype(F32)
    close(c.run(env), *c.want(exact=True))


@pytest.mark.parametrize("rising", [True, False])
def test_prefill_scores_far_apart(env, rising):
    """Each key's score 30 above or below the one before: the running maximum
    moves at every key, or never again."""
    c = Prefill(9, [150], 2, 1, 128)
    c.q[:] = 0
    c.k[:] = 0
    c.q[..., 0] = 1.0
    c.k[:, 0, 0] = bf16((np.arange(150) if rising else -np.arange(150)) * 30.0)
    got = c.run(env, scale=1.0)
    want, _ = c.want(scale=1.0)
    # a key's neighbours weigh e^-30: below a unit of f32
    close(got, want, 2.0 ** -20 * np.abs(want) + 1e-6)


@pytest.mark.parametrize("heads, kv, dim", [(4, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("n, at", [(100, 99), (100, 50), (300, 70), (64, 0), (5, 3)])
def test_prefill_what_is_not_seen_does_not_count(env, heads, kv, dim, n, at):
    c = Prefill(10, [n, 40], heads, kv, dim)
    clean = c.run(env)
    for which, x in ((c.v, np.nan), (c.v, np.inf), (c.k, np.nan)):
        kept = which[at].copy()
        which[at, 0, 3] = x
        if x == np.inf:
            which[at, 0, 4] = -np.inf
        got = c.run(env)
        assert np.array_equal(got[:at], clean[:at])
        assert np.array_equal(got[n:], clean[n:])
        close(got, *c.want())
        which[at] = kept


def test_prefill_query_that_is_not_finite(env):
    c = Prefill(11, [90], 4, 2, 64)
    clean = c.run(env)
    c.q[30, 1, 5] = np.nan
    got = c.run(env)
    assert np.isnan(got[30, 1]).all()
    got[30, 1] = clean[30, 1]
    assert np.array_equal(got, clean)


# ------------------------------------------------------------------ attention over the cache
class Decode:
    def __init__(self, seed, lengths, heads, kv, dim, width=None, size=0.25):
        rng = np.random.default_rng(seed)
        self.lengths, self.heads, self.kv, self.dim = lengths, heads, kv, dim
        self.m = len(lengths)
        counts = [-(-max(n, 0) // PAGE) for n in lengths]
        self.width = max([1, *counts]) if width is None else width
        self.cache = Cache(rng, sum(counts) + 3, kv, dim).random(rng)
        self.q = bf16(size * rng.standard_normal((self.m, heads, dim)))
        order = rng.permutation(self.cache.pages)
        self.table, at = np.full((self.m, self.width), -1, np.int32), 0
        for i, c in enumerate(counts):
            c = min(c, self.width)
            self.table[i, :c] = order[at:at + c]
            at += c
        # behind the last token: NaN codes
        for i, n in enumerate(lengths):
            if 0 < n < self.width * PAGE and n % PAGE:
                page = self.table[i, n // PAGE]
                self.cache.k[page, :, n % PAGE:] = 0x7F
                self.cache.v[page, :, n % PAGE:] = 0xFF

    def run(self, env, dtype=np.uint16, scale=None, stream=None):
        mod, s, _ = env
        s = stream or s
        out = dev(s, np.full(self.m * self.heads * self.dim, 7, dtype))
        mod.attention_decode(s, dev(s, bf16_bits(self.q)), self.cache.put(s), dev(s, np.array(self.lengths, np.int32)),
                             dev(s, self.table), self.heads, out, scale=scale)
        return values(out, s).reshape(self.m, self.heads, self.dim)

    def want(self, scale=None, exact=False):
        c, group = self.cache, self.heads // self.kv
        k, v = (E4M3[a] * c.s[:, :, i, None, None].astype(np.float64) for i, a in enumerate((c.k, c.v)))
        out, err = np.zeros((self.m, self.heads, self.dim)), np.zeros((self.m, self.heads, self.dim))
        for i, n in enumerate(self.lengths):
            n = min(max(n, 0), self.width * PAGE)
            at = self.table[i, np.arange(n) // PAGE]
            ok = (at >= 0) & (at < c.pages)
            at, slot = at[ok], (np.arange(n) % PAGE)[ok]
            if len(at) == 0:
                continue
            for h in range(self.heads):
                with np.errstate(invalid="ignore"):
                    s = k[at, h // group, slot] @ self.q[i, h].astype(np.float64)
                s = s[None] * (self.dim ** -0.5 if scale is None else scale)
                o, size = softmax_sums(s, v[at, h // group, slot])
                out[i, h], err[i, h] = o[0], size[0]
        return out, 2.0 ** -22 * np.abs(np.nan_to_num(out)) if exact else (2.0 ** -7 + 2.0 ** -9) * err

    def check(self, env, **kw):
        close(self.run(env, **kw), *self.want(kw.get("scale")))


@pytest.mark.parametrize("heads, kv, dim", [*LAYOUTS, (16, 1, 64), (40, 1, 128), (17, 1, 64)])
@pytest.mark.parametrize("lengths", [[1], [0, 63, 64, 65], [700, 3, 0, 129], [2048]])
def test_decode(env, heads, kv, dim, lengths):
    Decode(hash((heads, dim, sum(lengths))) % 1000, lengths, heads, kv, dim).check(env)


@pytest.mark.parametrize("dtype", [np.float32, np.uint16])
def test_decode_outputs(env, dtype):
    Decode(2, [300, 5, 1000], 8, 2, 128).check(env, dtype=dtype, scale=0.05)


def test_decode_wide_table_and_lengths_beyond_it(env):
    Decode(3, [30, 0, 500], 8, 2, 128, width=700).check(env)
    Decode(4, [500, -7, 64], 8, 2, 64, width=3).check(env)


def test_decode_many_rows(env):
    Decode(5, np.random.default_rng(5).integers(0, 200, 300).tolist(), 8, 2, 128).check(env)


def test_decode_pages_out_of_range_are_not_seen(env):
    c = Decode(6, [300, 64, 130], 8, 2, 128)
    c.table[0, 2], c.table[1, 0], c.table[2, 2] = -5, c.cache.pages, 1 << 30
    c.check(env)


@pytest.mark.parametrize("heads, kv, dim", [(4, 1, 128), (3, 1, 64)])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 64, 200, 1000, 8000])
def test_decode_counts_every_token_once(env, heads, kv, dim, n):
    c = Decode(7, [n, 5, 0], heads, kv, dim)
    c.q[:] = 0
    c.cache.v = e4m3(np.random.default_rng(n).integers(-8, 9, c.cache.v.shape) * 1.0)
    close(c.run(env), *c.want(exact=True))


@pytest.mark.parametrize("n", [500, 3000])
def test_decode_scores_far_apart(env, n):
    c = Decode(8, [n, n], 4, 1, 128)
    c.q[:], c.cache.k[:] = 0, 0
    c.q[0, :, 0], c.q[1, :, 0] = 1.0, -1.0
    for t in range(n):   # pages' scores rise (and fall, for the second row) by 16 or 32 each
        for r in range(2):
            page = c.table[r, t // PAGE]
            c.cache.s[page, :, 0] = 1.0
            c.cache.k[page, :, t % PAGE, 0] = e4m3(16.0 * (t // PAGE // 2))
    c.check(env, scale=1.0)


def test_decode_codes_that_are_nan(env):
    c = Decode(9, [200, 200, 100], 4, 2, 128)
    c.cache.k[c.table[0, 1], 0, 5, 9] = 0x7F
    c.cache.v[c.table[1, 3], 1, 2, 77] = 0xFF
    got = c.run(env)
    assert np.isnan(got[0, :2]).all() and np.isnan(got[1, 2:, 77]).all()
    close(got, *c.want())


def test_decode_rows_of_one_sequence(env):
    """Draft tokens: three rows of one sequence's pages."""
    c = Decode(10, [203, 201, 202], 8, 2, 128)
    c.table[1:] = c.table[0]
    c.check(env)


# ------------------------------------------------------------------ pages
@pytest.mark.parametrize("layers, pages, kv, dim, n", [(1, 2, 1, 64, 1), (3, 40, 3, 128, 17), (36, 9, 8, 128, 4),
                                                       (2, 300, 5, 64, 150)])
def test_copy_pages(env, layers, pages, kv, dim, n):
    mod, s, _ = env
    rng = np.random.default_rng(n)
    codes = rng.integers(0, 256, (layers, pages, kv * 2 * PAGE * dim), dtype=np.uint8)
    scales = rng.standard_normal((layers, pages, kv * 2)).astype(F32)
    at = rng.permutation(pages).astype(np.int32)
    src, dst = at[:n].copy(), at[n:2 * n].copy()
    if n > 4:
        src[1], dst[2] = -1, pages      # skipped
    cache = KvCache.over(dev(s, codes), dev(s, scales), layers, pages, kv, dim)
    mod.copy_pages(s, cache, dev(s, src), dev(s, dst))
    for a, b in zip(src, dst):
        if 0 <= a < pages and 0 <= b < pages:
            codes[:, b], scales[:, b] = codes[:, a], scales[:, a]
    assert np.array_equal(cache.codes.to_host_vec(s), codes.reshape(-1))
    assert np.array_equal(cache.scales.to_host_vec(s), scales.reshape(-1))


def test_replays(env):
    """A captured append and attention, replayed with new rows and lengths while
    other work runs between."""
    mod, _, ctx = env
    s = ctx.new_stream()
    heads, kv, dim, m, width = 8, 2, 128, 3, 40
    rng = np.random.default_rng(0)
    mod.reserve_workspace(mod.attention_decode_workspace_bytes(m, heads, kv, dim, width), s)
    cache = [KvCache(1, 130, kv, dim) for _ in range(2)]
    table = dev(s, rng.permutation(130)[:m * width].astype(np.int32))
    rope = dev(s, rope_table(width * PAGE, dim))
    x, past, lengths = DeviceBuffer(m * 12 * dim, np.float32), DeviceBuffer(m, np.int32), DeviceBuffer(m, np.int32)
    q, out = ([DeviceBuffer(m * heads * dim, np.uint16) for _ in range(2)] for _ in range(2))

    def step(i):
        mod.prepare_qk(s, x, heads, kv, dim, rope, q[i], past=past, cache=cache[i], table=table)
        mod.attention_decode(s, q[i], cache[i], lengths, table, heads, out[i])

    with Graph(s) as g:
        step(0)
    for t in range(130):
        x.copy_from_host(s, rng.standard_normal(m * 12 * dim).astype(F32) * (1 + t % 7))
        past.copy_from_host(s, np.array([t, 0, 2 * t], np.int32))
        lengths.copy_from_host(s, np.array([t + 1, 1, 2 * t + 1], np.int32))
        g.launch()
        step(1)
        s.synchronize()
        for a, b in ((q[0], q[1]), (out[0], out[1]), (cache[0].codes, cache[1].codes)):
            assert np.array_equal(a.to_host_vec(s), b.to_host_vec(s)), t
