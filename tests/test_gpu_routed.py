"""The routed layers against plain 64-bit forms: the router, the routed
experts' MLP and the adapters beside a projection, at the sizes, masks and
values where they can go wrong.

Tolerances.  A BF16 output is the f32 value rounded to 8 significant bits, a
relative error of at most 2^-8, so |got - want| <= 2^-8 (|want| + err) + err
with err the f32 value's own error.
* Router: a weight is a chain of a handful of f32 roundings, exp among them,
  and a sum over at most 1024 terms in a tree: 2^-19 relative covers it.
* Experts: err adds, per slot, 2^-18 of the sum of the magnitudes of its terms
  (f32 sums), 2^-16 of the row's largest |y| (y may be held in 16 bits against
  its block's largest), and for every act value whose quotient lies within
  127 * 2^-18 of a half-integer a whole code step times its weight: f32 cannot
  tell which side it falls on.
* Adapters: 2^-16 of the sums of magnitudes (f32 sums of up to 4096 products,
  and h carried as two BF16 parts)."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, DeviceBuffer, Graph, load
from inferrous_amd._lib import lib

pytestmark = pytest.mark.gpu

F32 = np.float32
INF, NAN = np.inf, np.nan


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


def dev(s, a):
    return DeviceBuffer.from_host(s, a)


def bf16_bits(a):
    u = np.ascontiguousarray(a, F32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bits(b):
    return (b.astype(np.uint32) << 16).view(F32)


def bf16(a):
    return from_bits(bf16_bits(a))


def values(buf, s):
    a = buf.to_host_vec(s)
    return from_bits(a) if a.dtype == np.uint16 else a


def close_bf16(got, want, err):
    bound = 2.0 ** -8 * (np.abs(want) + err) + err
    bad = ~(np.abs(got.astype(np.float64) - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], bound[bad][:4])


# ------------------------------------------------------------------ router
def route_oracle(x, k, score, bias, groups, top_groups, group_top, renorm, scale):
    """ids, weights in 64 bits, and whether f32 could choose otherwise (two of
    the values compared are within 4e-6 of their size, but not equal)."""
    m, e = x.shape
    ids, weights, near = np.full((m, k), -1, np.int32), np.zeros((m, k)), np.zeros(m, bool)

    def close(a, b):
        return a != b and abs(a - b) < 4e-6 * max(abs(a), abs(b))

    for r in range(m):
        row = np.where(np.isnan(x[r]), -INF, x[r].astype(np.float64))
        live = row > -INF
        if score == "softmax":
            top = row.max()
            if top == -INF:
                s = np.zeros(e)
            elif top == INF:
                s = (row == INF) / np.sum(row == INF)
            else:
                s = np.exp(row - top)
                s /= s.sum()
        else:
            with np.errstate(over="ignore"):
                s = 1.0 / (1.0 + np.exp(-row))
        s = np.where(s < 2.0 ** -126, 0.0, s)  # scores are held in f32
        c = s + (bias.astype(np.float64) if bias is not None else 0.0)
        c = np.where(live & ~np.isnan(c), c, -INF)
        if groups > 1:
            best = -np.sort(-c.reshape(groups, -1), axis=1)
            gs = best[:, 0].copy()
            if group_top == 2 and best.shape[1] > 1:
                gs = gs + np.where(best[:, 1] > -INF, best[:, 1], 0.0)
            order = np.argsort(-gs, kind="stable")
            if top_groups < groups:
                near[r] |= close(gs[order[top_groups - 1]], gs[order[top_groups]])
            keep = np.zeros(groups, bool)
            keep[order[:top_groups]] = True
            c = np.where(np.repeat(keep, e // groups), c, -INF)
        order = np.argsort(-c, kind="stable")[:k + 1]
        near[r] |= any(close(c[a], c[b]) for a, b in zip(order, order[1:]))
        chosen = [i for i in order[:k] if c[i] > -INF]
        ids[r, :len(chosen)] = chosen
        w = s[chosen]
        if renorm:
            w = w / w.sum() if w.sum() > 0 else 0 * w
        weights[r, :len(chosen)] = w * scale
    return ids, weights, near


def run_route(env, x, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0,
              b16=False, stream=None):
    mod, s, _ = env
    s = stream or s
    m, e = x.shape
    ids, w = dev(s, np.full(m * k, 77, np.int32)), dev(s, np.full(m * k, NAN, F32))
    mod.route_experts(s, dev(s, bf16_bits(x) if b16 else x.astype(F32)), e, ids, w, score=score,
                      bias=None if bias is None else dev(s, bias.astype(F32)), groups=groups, top_groups=top_groups,
                      group_top=group_top, renorm=renorm, scale=scale)
    return ids.to_host_vec(s).reshape(m, k), w.to_host_vec(s).reshape(m, k)


def check_route(env, x, k, b16=False, **kw):
    args = dict(score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0)
    args.update(kw)
    x = bf16(x) if b16 else x.astype(F32)
    bias = None if args["bias"] is None else args["bias"].astype(F32)
    ids, weights, near = route_oracle(x, k, **{**args, "bias": bias})
    got_ids, got = run_route(env, x, k, b16=b16, **args)
    ok = ~near
    # where f32 cannot tell the order, equally good experts' weights
    if args["bias"] is None and args["top_groups"] == args["groups"]:
        assert np.all(np.abs(got[near] - weights[near]) <= 1e-5 * np.abs(weights[near]))
    assert np.array_equal(got_ids[ok], ids[ok])
    assert np.all(np.abs(got[ok] - weights[ok]) <= 2.0 ** -19 * np.abs(weights[ok]) + 1e-37)


@pytest.mark.parametrize("e, k", [(1, 1), (2, 1), (2, 2), (8, 2), (60, 6), (63, 63), (64, 8), (65, 64), (128, 8),
                                  (129, 3), (256, 8), (384, 6), (512, 8), (513, 9), (1000, 10), (1024, 64)])
@pytest.mark.parametrize("m", [1, 5, 130])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(env, e, k, m, score):
    rng = np.random.default_rng(e * 131 + k + m)
    check_route(env, rng.standard_normal((m, e)) * 2, k, score=score, renorm=m != 5, scale=1.0 if m == 1 else 2.5,
                b16=m == 130)


@pytest.mark.parametrize("e, groups, top_groups, k", [
    (64, 8, 3, 8), (256, 8, 4, 8), (60, 6, 3, 7), (12, 12, 5, 5), (64, 64, 9, 9), (96, 2, 1, 48), (1024, 4, 2, 16),
    (32, 4, 4, 8), (130, 13, 2, 20)])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups_and_bias(env, e, groups, top_groups, k, group_top, score):
    rng = np.random.default_rng(e + groups + group_top)
    x = rng.standard_normal((40, e)) * 2
    x[7, ::3] = -INF
    check_route(env, x, k, score=score, bias=rng.standard_normal(e) * 0.3, groups=groups, top_groups=top_groups,
                group_top=group_top)


@pytest.mark.parametrize("e, groups, top_groups, group_top, k", [
    (16, 1, 1, 1, 3), (16, 8, 3, 2, 5), (32, 4, 2, 1, 9), (64, 16, 7, 2, 16), (128, 1, 1, 1, 8), (256, 8, 4, 2, 8),
    (256, 2, 1, 2, 16), (256, 32, 9, 2, 8), (240, 8, 4, 2, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_many_rows(env, e, groups, top_groups, group_top, k, score):
    """Enough rows for several to a wave; ties, masks and infinities among them."""
    rng = np.random.default_rng(e + groups)
    x = rng.standard_normal((2051, e)) * 2
    x[5] = -INF
    x[6] = NAN
    x[7, 1:] = -INF
    x[8] = 0.0
    x[9] = np.repeat(np.arange(e // 4), 4) * -0.25
    x[10, ::3] = INF
    x[11, : e // 2] = -INF
    x[12, ::2] = -INF
    x[2050, e - 1] = 9.0
    check_route(env, x, k, score=score, bias=rng.standard_normal(e) * 0.3 if score == "sigmoid" else None,
                groups=groups, top_groups=top_groups, group_top=group_top, renorm=k != 9, scale=2.5, b16=e == 64)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_ties_masks_and_infinities(env, score, groups):
    e, k = 32, 6
    x = np.zeros((16, e))
    x[1] = -INF                                   # nothing left
    x[2] = NAN
    x[3, 1:] = -INF                               # one expert left
    x[4] = np.repeat(np.arange(8), 4) * 0.5       # ties in fours
    x[5] = -x[4]
    x[6, [3, 9, 30]] = INF
    x[7] = np.finfo(F32).min                      # the lowest value is a logit like any other
    x[8, 5] = NAN
    x[9] = -INF
    x[9, [4, 31]] = np.finfo(F32).min, np.finfo(F32).max
    x[10] = np.where(np.arange(e) % 2, 60.0, -60.0)
    x[11, :8] = -INF                              # a whole group out
    x[12] = -200.0
    x[13, ::2] = -0.0
    for top_groups in ([1] if groups == 1 else [2, 4]):
        for group_top in (1, 2):
            for renorm in (True, False):
                check_route(env, x, k, score=score, groups=groups, top_groups=top_groups, group_top=group_top,
                            renorm=renorm)


def test_route_bias_puts_experts_out(env):
    rng = np.random.default_rng(5)
    bias = np.zeros(40)
    bias[3], bias[4], bias[5] = -INF, NAN, INF
    x = rng.standard_normal((9, 40))
    with np.errstate(invalid="ignore"):
        check_route(env, x, 5, score="sigmoid", bias=bias)


def test_route_on_another_stream_and_replayed(env):
    """Every replay of a captured router gives the eager result."""
    mod, s, ctx = env
    rng = np.random.default_rng(8)
    x = rng.standard_normal((100, 256)).astype(F32)
    other = ctx.new_stream()
    want = run_route(env, x, 8, stream=other)
    assert np.array_equal(want[0], run_route(env, x, 8)[0])
    lx, ids, w = dev(s, x), dev(s, np.zeros(800, np.int32)), dev(s, np.zeros(800, F32))
    graph = Graph(s)
    with graph:
        mod.route_experts(s, lx, 256, ids, w)
    for turn in range(3):
        lx.copy_from_host(s, np.roll(x, turn, 0))
        graph.launch(s)
        s.synchronize()
        eager = run_route(env, np.roll(x, turn, 0), 8)
        assert np.array_equal(ids.to_host_vec(s).reshape(100, 8), eager[0])
        assert np.array_equal(w.to_host_vec(s).reshape(100, 8), eager[1])


# ------------------------------------------------------------------ experts
class Experts:
    """Inputs of an experts_mlp call, and its 64-bit outputs with their error bound."""

    def __init__(self, m, k, e, h, f, seed=0, residual=False, ids=None):
        rng = np.random.default_rng(seed)
        self.m, self.k, self.e, self.h, self.f = m, k, e, h, f
        self.q = rng.integers(-127, 128, (m, h)).astype(np.int8)
        self.asc = (0.02 * (0.5 + rng.random(m))).astype(F32)
        if ids is None:
            ids = np.stack([rng.permutation(max(e, k))[:k] for _ in range(m)]) if m else np.zeros((0, k))
            ids = np.where(ids < e, ids, -1)
        self.ids = np.asarray(ids, np.int32).reshape(m, k)
        self.weights = rng.random((m, k)).astype(F32)
        self.wg, self.wu = (rng.integers(-127, 128, (e, f, h)).astype(np.int8) for _ in range(2))
        self.wd = rng.integers(-127, 128, (e, h, f)).astype(np.int8)
        size = 1.0 / (73.0 * 73.0 * 0.02 * h ** 0.5)
        self.sg, self.su = ((size * 73.0 * (0.5 + rng.random((e, f)))).astype(F32) for _ in range(2))
        self.sd = ((0.5 + rng.random((e, h))) / (73.0 * f ** 0.5)).astype(F32)
        self.residual = rng.standard_normal((m, h)).astype(F32) if residual else None

    def run(self, env, dtype=np.uint16, stream=None):
        mod, s, _ = env
        s = stream or s
        out = dev(s, np.full(self.m * self.h, 1, dtype))
        d = [dev(s, a) for a in (self.q, self.asc, self.ids, self.weights, self.wg, self.sg, self.wu, self.su,
                                 self.wd, self.sd)]
        res = dev(s, self.residual) if self.residual is not None else None
        mod.experts_mlp(s, d[0], d[1], self.h, d[2], d[3], *d[4:], self.e, out, residual=res)
        return values(out, s).reshape(self.m, self.h)

    def want(self):
        out = np.zeros((self.m, self.h)) if self.residual is None else self.residual.astype(np.float64)
        err = 2.0 ** -18 * np.abs(out)
        x = self.q.astype(np.float64) * self.asc.astype(np.float64)[:, None]
        for e in range(self.e):
            for j in range(self.k):
                t = np.flatnonzero(self.ids[:, j] == e)
                if not len(t):
                    continue
                gate = x[t] @ (self.wg[e].astype(np.float64) * self.sg[e].astype(np.float64)[:, None]).T
                up = x[t] @ (self.wu[e].astype(np.float64) * self.su[e].astype(np.float64)[:, None]).T
                with np.errstate(over="ignore"):
                    act = gate / (1.0 + np.exp(-gate)) * up
                held, doubt = np.zeros_like(act), np.zeros_like(act)
                for c in range(0, self.f, 128):
                    p = act[:, c:c + 128]
                    step = np.maximum(np.abs(p).max(1, keepdims=True), 1e-8) / 127.0
                    v = p / step
                    held[:, c:c + 128] = np.rint(v).clip(-127, 127) * step
                    doubt[:, c:c + 128] = (np.abs(v - np.floor(v) - 0.5) < 127 * 2.0 ** -18) * step
                wd = self.wd[e].astype(np.float64) * self.sd[e].astype(np.float64)[:, None]
                y, w = held @ wd.T, self.weights[t, j].astype(np.float64)[:, None]
                out[t] += w * y
                err[t] += np.abs(w) * (2.0 ** -18 * (np.abs(held) @ np.abs(wd).T) + doubt @ np.abs(wd).T
                                       + 2.0 ** -16 * np.abs(y).max(1, keepdims=True))
        return out, err

    def check(self, env, dtype=np.uint16):
        close_bf16(self.run(env, dtype), *self.want())


@pytest.mark.parametrize("m, k, e, h, f", [
    (1, 1, 1, 16, 16), (1, 8, 64, 256, 128), (1, 3, 5, 4096, 256), (1, 20, 24, 1040, 1168), (2, 2, 4, 144, 400), (3, 8, 8, 128, 2064),
    (4, 6, 16, 1040, 240), (7, 2, 3, 272, 144), (16, 8, 32, 512, 192), (33, 2, 4, 2000, 720), (64, 4, 128, 256, 384),
    (65, 1, 2, 512, 256), (130, 3, 5, 784, 272), (300, 2, 3, 384, 640), (600, 4, 6, 256, 128), (1100, 2, 2, 144, 272),
    (257, 1, 1, 640, 1024), (40, 7, 1000, 32, 48), (1000, 6, 1024, 48, 16)])
def test_experts(env, m, k, e, h, f):
    Experts(m, k, e, h, f, seed=m + e).check(env)


@pytest.mark.parametrize("m", [1, 5, 200])
def test_experts_residual_in_f32(env, m):
    Experts(m, 3, 6, 272, 208, seed=m, residual=True).check(env, F32)


@pytest.mark.parametrize("m", [1, 6, 150, 900])
def test_experts_slots_without_an_expert(env, m):
    """Ids outside the experts are skipped; a row with none gets zeros (or its residual)."""
    rng = np.random.default_rng(m)
    ids = np.stack([rng.permutation(8)[:3] for _ in range(m)]).astype(np.int32)
    ids[rng.random((m, 3)) < 0.3] = -1
    ids[0] = [-1, 8, 2 ** 31 - 1]
    for residual in (False, True):
        c = Experts(m, 3, 8, 160, 144, seed=m, residual=residual, ids=ids)
        got = c.run(env)
        close_bf16(got, *c.want())
        assert np.array_equal(got[0], bf16(c.residual[0]) if residual else np.zeros(160, F32))
    Experts(m, 3, 8, 160, 144, seed=m, ids=np.full((m, 3), -1)).check(env)


@pytest.mark.parametrize("m, e", [(300, 4), (40, 64), (130, 3)])
def test_experts_all_rows_to_one(env, m, e):
    """Every row meets the same expert; the others have none."""
    Experts(m, 1, e, 256, 144, seed=e, ids=np.full((m, 1), e - 1)).check(env)


@pytest.mark.parametrize("m", [2, 400])
def test_experts_expert_met_twice(env, m):
    """A row may name one expert in two slots."""
    Experts(m, 2, 3, 128, 128, seed=m, ids=np.tile([2, 2], (m, 1))).check(env)


@pytest.mark.parametrize("m", [1, 300])
def test_experts_non_finite_rows(env, m):
    """An infinite or NaN row scale reaches its own row only; zero rows give zeros."""
    c = Experts(m, 2, 4, 144, 144, seed=3)
    base = c.run(env)
    c.asc[0] = NAN
    bad = c.run(env)
    assert np.array_equal(bad[1:], base[1:])
    c.asc[0] = INF
    bad = c.run(env)
    assert np.array_equal(bad[1:], base[1:]) and not np.isfinite(bad[0]).all()
    c.asc[0] = 0.0
    assert np.array_equal(c.run(env)[0], np.zeros(144, F32))


@pytest.mark.parametrize("m", [1, 40, 700])
def test_experts_non_finite_scales_stay_in_their_columns(env, m):
    """An infinite or NaN scale of one output column reaches that column only."""
    c = Experts(m, 2, 3, 192, 144, seed=6, ids=np.tile([1, 2], (m, 1)))
    want, err = c.want()
    c.sd[2, 5], c.sd[1, 70], c.sd[2, 191] = INF, NAN, -INF
    got = c.run(env)
    bad = [5, 70, 191]
    assert not np.isfinite(got[:, bad]).any() and np.isnan(got[:, 70]).all()
    rest = np.setdiff1d(np.arange(192), bad)
    close_bf16(got[:, rest], want[:, rest], err[:, rest])


@pytest.mark.parametrize("m", [1, 70])
def test_experts_same_bits_again_and_on_another_stream(env, m):
    c = Experts(m, 4, 8, 512, 256, seed=9)
    first = c.run(env)
    for _ in range(3):
        assert np.array_equal(c.run(env), first)
    assert np.array_equal(c.run(env, stream=env[2].new_stream()), first)


@pytest.mark.parametrize("m", [1, 48])
def test_experts_replayed(env, m):
    """A captured call follows new ids, weights and rows at every replay."""
    mod, s, _ = env
    cs = [Experts(m, 4, 8, 512, 256, seed=9 + i) for i in range(3)]
    c = cs[0]
    mod.reserve_workspace(lib().w8a8_experts_mlp_workspace_bytes(m, 4, 8, 512, 256), s)
    q, asc, ids, w = (dev(s, a) for a in (c.q, c.asc, c.ids, c.weights))
    mats = [dev(s, a) for a in (c.wg, c.sg, c.wu, c.su, c.wd, c.sd)]
    out = dev(s, np.zeros(m * 512, np.uint16))
    graph = Graph(s)
    with graph:
        mod.experts_mlp(s, q, asc, 512, ids, w, *mats, 8, out)
    for n in cs + cs:
        for buf, a in ((q, n.q), (asc, n.asc), (ids, n.ids), (w, n.weights)):
            buf.copy_from_host(s, a)
        graph.launch(s)
        s.synchronize()
        n.wg, n.sg, n.wu, n.su, n.wd, n.sd = c.wg, c.sg, c.wu, c.su, c.wd, c.sd
        assert np.array_equal(values(out, s).reshape(m, 512), n.run(env))


# ------------------------------------------------------------------ adapters
class Adapters:
    def __init__(self, m, n, k, rank, count, seed=0, residual=False, ids=None):
        rng = np.random.default_rng(seed)
        self.m, self.n, self.k, self.rank, self.count = m, n, k, rank, count
        self.x = bf16(rng.standard_normal((m, k)).astype(F32))
        self.asc = (np.abs(self.x).max(1).clip(1e-8) / 127).astype(F32)
        self.q = np.rint(self.x / self.asc[:, None]).clip(-127, 127).astype(np.int8)
        self.w = rng.integers(-127, 128, (n, k)).astype(np.int8)
        self.ws = ((0.5 + rng.random(n)) / (73.0 * k ** 0.5)).astype(F32)
        self.ids = (rng.integers(-1, count, m) if ids is None else np.asarray(ids)).astype(np.int32)
        self.a = bf16(rng.standard_normal((count, rank, k)).astype(F32) * F32(k ** -0.5))
        self.b = bf16(rng.standard_normal((count, n, rank)).astype(F32) * F32(0.5 * rank ** -0.5))
        self.scaling = (0.5 + rng.random(count)).astype(F32)
        self.residual = rng.standard_normal((m, n)).astype(F32) if residual else None

    def run(self, env, dtype=np.uint16, x_bf16=False, stream=None):
        mod, s, _ = env
        s = stream or s
        out = dev(s, np.full(self.m * self.n, 1, dtype))
        res = dev(s, self.residual) if self.residual is not None else None
        x = dev(s, bf16_bits(self.x) if x_bf16 else self.x)
        q, asc, w, ws, ids, a, b, sc = (dev(s, v) for v in (self.q, self.asc, self.w, self.ws, self.ids,
                                                            bf16_bits(self.a), bf16_bits(self.b), self.scaling))
        mod.linear_adapters(s, q, asc, w, ws, self.k, x, ids, a, b, sc, out, residual=res)
        return values(out, s).reshape(self.m, self.n)

    def want(self):
        base = (self.q.astype(np.float64) @ self.w.astype(np.float64).T) * self.asc[:, None].astype(np.float64) \
            * self.ws.astype(np.float64)
        out, err = base.copy(), 2.0 ** -22 * np.abs(base)
        if self.residual is not None:
            out += self.residual
            err += 2.0 ** -22 * np.abs(out)
        x = bf16(self.x).astype(np.float64)
        for a in range(self.count):
            t = np.flatnonzero(self.ids == a)
            if len(t):
                A, B, sc = self.a[a].astype(np.float64), self.b[a].astype(np.float64), float(self.scaling[a])
                out[t] += sc * (x[t] @ A.T) @ B.T
                err[t] += 2.0 ** -16 * sc * (np.abs(x[t]) @ np.abs(A).T) @ np.abs(B).T
        return out, err

    def check(self, env, dtype=np.uint16, x_bf16=False):
        close_bf16(self.run(env, dtype, x_bf16), *self.want())


@pytest.mark.parametrize("m, n, k, rank, count", [
    (1, 1, 16, 8, 1), (1, 33, 64, 8, 2), (1, 4096, 4096, 16, 3), (1, 515, 2000, 64, 4), (1, 7, 5136, 256, 2), (64, 96, 4096, 128, 5), (2, 300, 512, 24, 3), (2, 33, 4112, 256, 2), (3, 1030, 2064, 40, 5), (4, 515, 1008, 16, 3), (4, 8200, 4096, 8, 2),
    (5, 1023, 784, 16, 7), (8, 256, 4096, 256, 2), (16, 640, 1024, 32, 40), (33, 129, 272, 128, 5),
    (64, 700, 1040, 40, 64), (65, 257, 128, 8, 3), (130, 500, 2000, 72, 9), (300, 320, 640, 16, 4),
    (513, 193, 400, 64, 1)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_adapters(env, m, n, k, rank, count, x_bf16):
    Adapters(m, n, k, rank, count, seed=m + n).check(env, x_bf16=x_bf16)


@pytest.mark.parametrize("m, n, k, rank, count", [
    (600, 1024, 1040, 256, 2), (1500, 520, 528, 128, 3), (2100, 999, 400, 72, 1), (1100, 264, 2048, 200, 8),
    (5000, 130, 144, 256, 3)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_adapters_where_the_tiles_lead(env, m, n, k, rank, count, x_bf16):
    """Enough work for the sorted rows: runs of one adapter, many in one tile, rows
    with none at the end, odd columns, both types of x and of out."""
    rng = np.random.default_rng(m)
    ids = np.where(np.arange(m) < 2 * m // 3, 0, np.arange(m) % (count + 1) - 1)
    ids = rng.permutation(ids) if x_bf16 else ids
    Adapters(m, n, k, rank, count, seed=m + n, ids=ids, residual=x_bf16).check(env, F32 if x_bf16 else np.uint16,
                                                                                x_bf16=x_bf16)


def test_adapters_in_tiles_without_any(env):
    """No row has an adapter: the projection, bit for bit."""
    mod, s, _ = env
    c = Adapters(900, 512, 512, 256, 3, seed=4, ids=np.full(900, -1))
    out = dev(s, np.zeros(900 * 512, np.uint16))
    mod.linear(s, None, *(dev(s, v) for v in (c.q, c.asc, c.w, c.ws)), 512, out)
    assert np.array_equal(c.run(env), values(out, s).reshape(900, 512))


def test_adapters_in_tiles_keep_rows_apart(env):
    """A NaN adapter reaches its own rows only, rows without one equal the projection,
    and the same call gives the same bits."""
    mod, s, _ = env
    m, n, k = 900, 512, 512
    ids = np.arange(m) % 4 - 1
    c = Adapters(m, n, k, 256, 3, seed=4, ids=ids)
    base = c.run(env)
    assert np.array_equal(c.run(env), base)
    out = dev(s, np.zeros(m * n, np.uint16))
    mod.linear(s, None, *(dev(s, v) for v in (c.q, c.asc, c.w, c.ws)), k, out)
    assert np.array_equal(base[ids < 0], values(out, s).reshape(m, n)[ids < 0])
    c.b[2], c.a[2, 5] = NAN, INF
    got = c.run(env)
    assert np.array_equal(got[ids != 2], base[ids != 2]) and not np.isfinite(got[ids == 2]).any()


@pytest.mark.parametrize("m", [1, 9, 140])
def test_adapters_residual_in_f32(env, m):
    Adapters(m, 333, 400, 16, 3, seed=m, residual=True).check(env, F32)


@pytest.mark.parametrize("m", [1, 6, 200])
def test_rows_without_an_adapter_are_the_projection(env, m):
    """Ids outside the adapters leave w8a8_linear's output, bit for bit."""
    mod, s, _ = env
    ids = np.resize([-1, 4, 2 ** 31 - 1, -2 ** 31], m)
    c = Adapters(m, 301, 528, 16, 4, seed=m, ids=ids)
    out = dev(s, np.zeros(m * 301, np.uint16))
    mod.linear(s, None, *(dev(s, v) for v in (c.q, c.asc, c.w, c.ws)), 528, out)
    assert np.array_equal(c.run(env), values(out, s).reshape(m, 301))


@pytest.mark.parametrize("m", [12, 200])
def test_adapters_in_runs_and_alone(env, m):
    """Rows in runs, rows in turn, one adapter for all, and one odd row among them."""
    for ids in (np.arange(m) * 5 // m, np.arange(m) % 5, np.full(m, 3), np.where(np.arange(m) == m // 2, 1, 4),
                np.where(np.arange(m) == m - 1, 0, -1)):
        Adapters(m, 160, 256, 24, 5, seed=m, ids=ids).check(env)


def test_adapters_round_f32_rows_to_bf16(env):
    c = Adapters(7, 96, 128, 8, 2, seed=1)
    c.x = (c.x * (1 + 2.0 ** -10)).astype(F32)
    c.check(env)


@pytest.mark.parametrize("m", [3, 140])
def test_adapter_with_non_finite_values_stays_with_its_rows(env, m):
    """A NaN or infinite adapter, or row, reaches no other row."""
    c = Adapters(m, 130, 256, 16, 3, seed=4, ids=np.arange(m) % 4 - 1)
    base = c.run(env)
    c.b[2], c.a[2, 5] = NAN, INF
    got = c.run(env)
    assert np.array_equal(got[c.ids != 2], base[c.ids != 2]) and not np.isfinite(got[c.ids == 2]).any()
    c = Adapters(m, 130, 256, 16, 3, seed=4, ids=np.arange(m) % 4 - 1)
    c.x[1] = NAN
    got = c.run(env)
    rest = np.arange(m) != 1
    assert np.array_equal(got[rest], base[rest]) and np.isnan(got[1]).all()


def test_adapters_same_bits_again_and_on_another_stream(env):
    for m in (1, 20, 150):
        c = Adapters(m, 500, 1024, 16, 6, seed=m)
        first = c.run(env)
        assert all(np.array_equal(c.run(env), first) for _ in range(3))
        assert np.array_equal(c.run(env, stream=env[2].new_stream()), first)


@pytest.mark.parametrize("m", [1, 40])
def test_adapters_replayed(env, m):
    mod, s, _ = env
    c = Adapters(m, 320, 512, 16, 6, seed=m)
    mod.reserve_workspace(lib().w8a8_linear_adapters_workspace_bytes(m, 320, 512, 16, 6), s)
    q, asc, w, ws, x, ids, a, b, sc = (dev(s, v) for v in (c.q, c.asc, c.w, c.ws, bf16_bits(c.x), c.ids,
                                                           bf16_bits(c.a), bf16_bits(c.b), c.scaling))
    out = dev(s, np.zeros(m * 320, np.uint16))
    graph = Graph(s)
    with graph:
        mod.linear_adapters(s, q, asc, w, ws, 512, x, ids, a, b, sc, out)
    for turn in range(4):
        c.ids = np.roll(c.ids, 1) if m > 1 else np.array([turn - 1], np.int32)
        ids.copy_from_host(s, c.ids)
        graph.launch(s)
        s.synchronize()
        assert np.array_equal(values(out, s).reshape(m, 320), c.run(env, x_bf16=True))
