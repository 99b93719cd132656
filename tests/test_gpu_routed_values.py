"""The routed layers' values where a form could lose them: an output column much
larger than its neighbours, codes at exact ties, infinite scales and weights, and
adapter sums whose last bits count.  Every form has to give the definition's
value, whatever the number of rows that chose it."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, DeviceBuffer, W8A8Error, load
from test_gpu_routed import Adapters, Experts, bf16, bf16_bits, close_bf16, from_bits, values

pytestmark = pytest.mark.gpu

F32 = np.float32
INF = np.inf


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


# Rows at which experts_mlp runs slot by slot, and expert by expert in tiles of 32, 64, 128
# and 256 rows.
ROWS = [1, 5, 70, 130, 300, 900]


@pytest.mark.parametrize("m", ROWS)
def test_experts_large_columns_cost_their_neighbours_nothing(env, m):
    """Columns 3000 and 100,000 times their neighbours: an output column depends on
    its own scale alone, so the others keep the bound that they had without."""
    c = Experts(m, 2, 3, 192, 144, seed=m)
    want, err = c.want()
    c.sd[:, 5] *= 3000.0
    c.sd[:, 70] *= 1e5
    rest = np.setdiff1d(np.arange(192), [5, 70])
    close_bf16(c.run(env)[:, rest], want[:, rest], err[:, rest])


@pytest.mark.parametrize("m", ROWS)
def test_experts_codes_round_ties_to_even(env, m):
    """act exactly at the half-way points of its codes, for a scale that is no power
    of two: gate is 32, whose sigmoid is 1 in f32, and up k + 1/2 times the scale.
    The codes' products are exact, so the outputs are the definition's in BF16."""
    h, f = 128, 128
    c = Experts(m, 1, 1, h, f, ids=np.zeros((m, 1), np.int32))
    c.q[:] = 0
    c.q[:, :2] = 1                                # column 0 of gate's rows, column 1 of up's
    c.asc[:], c.weights[:] = 1.0, 1.0
    c.wg[:], c.wu[:], c.wd[:] = 0, 0, 0
    c.wg[0, :, 0] = 32
    c.sg[:], c.sd[:] = 1.0, 1.0
    steps = np.arange(f) % 63 + 0.5               # act in units of the scale
    steps[1::2] *= -1
    steps[0] = 127.0                              # act's largest: the scale is 3 exactly
    c.wu[0, :, 1] = 2 * steps
    c.wu[0, 0, 1] = 127
    c.su[:] = 3.0 / 64.0                          # 32 * 2 steps * 3 / 64 = 3 steps
    c.su[0, 0] = 3.0 / 32.0
    c.wd[0, np.arange(h), np.arange(f)] = 1       # output column i is code i's value
    assert np.array_equal(c.run(env), np.tile(bf16(3.0 * np.rint(steps)), (m, 1)))


@pytest.mark.parametrize("m", ROWS)
def test_experts_act_is_held_in_f32(env, m):
    """One act value to each group of 128 columns, gates from -60 to 20, less its 64-bit
    value as the residual: what is left is act's error.  exp 1 unit and a rounding, a
    reciprocal 1 unit, and eight products, quotients and sums of half a unit: 12 *
    2^-24 of the value, below 2^-20."""
    gates = np.array([-60, -55, -47, -38, -33, -27, -21, -16, -11, -7, -3, -1, 1, 4, 9, 20], np.float64)
    h, f = 16, 16 * 128
    c = Experts(m, 1, 1, h, f, residual=True, ids=np.zeros((m, 1), np.int32))
    c.q[:], c.wg[:], c.wu[:], c.wd[:] = 0, 0, 0, 0
    c.q[:, 0] = 1
    c.asc[:], c.weights[:], c.sg[:], c.sd[:] = 1.0, 1.0, 1.0, 1.0
    c.wg[0, ::128, 0], c.wu[0, ::128, 0] = gates, 1
    silu = gates / (1.0 + np.exp(-gates))
    c.su[0, ::128] = 2.0 ** -np.floor(np.log2(np.abs(silu)))   # act between 1 and 2
    c.wd[0, np.arange(h), np.arange(h) * 128] = 1
    act = silu * c.su[0, ::128].astype(np.float64)
    c.residual[:] = -act
    assert np.all(np.abs(c.run(env)) <= 2.0 ** -20 * np.abs(act))


@pytest.mark.parametrize("m", ROWS)
def test_experts_infinite_column_scale(env, m):
    """y = ws_down * a finite sum: an infinite scale of one column gives an infinity of
    the sum's sign, in every form, and leaves the other columns alone."""
    c = Experts(m, 2, 3, 192, 144, seed=m + 1, ids=np.tile([1, 2], (m, 1)))
    want, err = c.want()
    c.sd[1, 5] = 0.0                              # column 5 of expert 2 alone
    w5, e5 = c.want()
    c.sd[1, 5], c.sd[2, 5] = 1.0, INF
    got = c.run(env)
    sure = np.abs(w5[:, 5]) > e5[:, 5]
    assert sure.mean() > 0.9
    assert np.array_equal(got[sure, 5], np.where(w5[sure, 5] > 0, INF, -INF))
    rest = np.arange(192) != 5
    close_bf16(got[:, rest], want[:, rest], err[:, rest])


@pytest.mark.parametrize("m", ROWS)
def test_experts_infinite_weight(env, m):
    """An infinite weight of one slot gives infinities of its product's signs."""
    c = Experts(m, 2, 3, 192, 144, seed=m + 2, ids=np.tile([1, 2], (m, 1)))
    want, err = c.want()
    w = c.weights[0].copy()
    c.weights[0] = 1.0, 0.0
    one, bound = (v[0] for v in c.want())
    c.weights[0] = INF, w[1]
    got = c.run(env)
    sure = np.abs(one) > bound
    assert sure.mean() > 0.9
    assert np.array_equal(got[0, sure], np.where(one[sure] > 0, INF, -INF))
    close_bf16(got[1:], want[1:], err[1:])


# ------------------------------------------------------------------ adapters
# rows, columns, width, rank, adapters: row by row (one kernel, and two), with the rows sorted
# by adapter and tiles of 128 and of 256.
ADAPTED = [(1, 40, 64, 8, 2), (4, 40, 64, 8, 2), (30, 130, 272, 16, 3), (900, 512, 512, 256, 3),
           (4096, 3088, 144, 16, 4)]


def bare(m, n, k, rank, count):
    """Rows of adapter r % count whose projection is 0 and whose h is x[0] alone."""
    c = Adapters(m, n, k, rank, count, ids=np.arange(m) % count)
    c.x[:], c.w[:], c.a[:], c.b[:], c.scaling[:] = 0, 0, 0, 0, 1.0
    c.q[:] = 0
    c.x[:, 0], c.a[:, :, 0] = 1.0, 1.0
    return c


@pytest.mark.parametrize("m, n, k, rank, count", ADAPTED)
def test_adapters_keep_every_bit_of_h(env, m, n, k, rank, count):
    """h[i] = 1 + 2^-9 + 2^-e less h[7] = 1 + 2^-9: what is left is h's last bits."""
    e = np.array([12, 15, 18, 20, 23])
    c = bare(m, n, k, rank, count)
    c.x[:, 1:3] = 1.0
    c.a[:, :, 1], c.a[:, :5, 2] = 2.0 ** -9, 2.0 ** -e.astype(F32)
    i = np.arange(n) % 5
    c.b[:, np.arange(n), i], c.b[:, :, 7] = 1.0, -1.0
    assert np.array_equal(c.run(env), np.tile(2.0 ** -e[i].astype(F32), (m, 1)))


@pytest.mark.parametrize("m, n, k, rank, count", ADAPTED)
@pytest.mark.parametrize("what", ["x", "a", "b", "scaling", "largest"])
def test_adapters_infinities(env, m, n, k, rank, count, what):
    """An infinity of x, A, B or the scaling gives infinities of the products' signs in
    its rows, and h may be the largest f32; the other rows keep their values."""
    c = bare(m, n, k, rank, count)
    sign = np.where(np.arange(n) % 3 == 1, -1.0, 1.0).astype(F32)
    c.b[:] = sign[None, :, None]
    mine = np.arange(m) == 0 if what in ("x", "largest") else c.ids == 0
    want = np.where(mine[:, None], INF, float(rank)) * sign
    if what == "x":
        c.x[0, 0] = INF
    elif what == "a":
        c.a[0, 3, 0] = INF
    elif what == "b":
        c.b[0, 7, 5] = INF
        want = np.tile(rank * sign, (m, 1))
        want[mine, 7] = INF
    elif what == "scaling":
        c.scaling[0] = -INF
        want[mine] = -want[mine]
    else:  # less than 2^128, but no BF16 value between
        c.x[0, :3] = 255 * 2.0 ** 120, 2.0 ** 119, 255 * 2.0 ** 110
        c.x[1:, 1:3] = 0.0
        c.a[:, :, :3] = 0.0
        c.a[:, 2, :3] = 1.0
        c.b[:, :, :] = (sign * 2.0 ** -100)[None, :, None]
        want = np.zeros((m, n))
        want[0] = (255 * 2.0 ** 20 + 2.0 ** 19 + 255 * 2.0 ** 10) * sign
        want[1:] = 2.0 ** -100 * sign
        want = bf16(want)
    with np.errstate(invalid="ignore"):
        got = c.run(env)
    assert np.array_equal(got, want.astype(F32))


# ------------------------------------------------------------------ workspaces
def test_a_refused_allocation_is_no_later_calls_error(env):
    """An allocation that cannot be had raises, and the launch after it does not report
    its error once more."""
    with pytest.raises(W8A8Error):
        DeviceBuffer(1 << 50, np.uint8)
    Experts(3, 2, 4, 64, 48).check(env)


# ------------------------------------------------------------------ limits
def test_experts_at_the_most_slots(env):
    """2^24 rows of one slot, the documented limit: a period of rows again and again,
    each with the outputs of its first."""
    mod, s, _ = env
    m, period, h, f, e = 1 << 24, 1 << 12, 16, 16, 5
    c = Experts(period, 1, e, h, f, seed=7)
    c.ids = np.random.default_rng(8).integers(-1, e, (period, 1)).astype(np.int32)
    want, err = c.want()
    rows = [np.tile(a, (m // period,) + (1,) * (a.ndim - 1)) for a in (c.q, c.asc, c.ids, c.weights)]
    q, asc, ids, weights = (DeviceBuffer.from_host(s, a) for a in rows)
    mats = [DeviceBuffer.from_host(s, a) for a in (c.wg, c.sg, c.wu, c.su, c.wd, c.sd)]
    out = DeviceBuffer(m * h, np.uint16)
    mod.experts_mlp(s, q, asc, h, ids, weights, *mats, e, out)
    got = out.to_host_vec(s).reshape(-1, period * h)
    close_bf16(from_bits(got[0]).reshape(period, h), want, err)
    assert (got == got[0]).all()


def at_the_end(s, count, part):
    """A buffer of `count` parts, zeros but for the last one."""
    buf = DeviceBuffer(count * part.size, part.dtype)
    DeviceBuffer.view_of(buf, (count - 1) * part.size, part.size).copy_from_host(s, part.reshape(-1))
    return buf


@pytest.mark.parametrize("m", [2, 200])
def test_experts_weights_past_four_gib(env, m):
    """The last of 270 experts of 4096 x 4096: its weights lie above 2^32 bytes."""
    mod, s, _ = env
    h = f = 4096
    e = 270
    c = Experts(m, 1, 1, h, f, seed=m, ids=np.zeros((m, 1), np.int32))
    mats = [at_the_end(s, e, a) for a in (c.wg, c.sg, c.wu, c.su, c.wd, c.sd)]
    assert len(mats[0]) > 1 << 32
    q, asc, ids, weights = (DeviceBuffer.from_host(s, a) for a in (c.q, c.asc, np.full(m, e - 1, np.int32), c.weights))
    out = DeviceBuffer(m * h, np.uint16)
    mod.experts_mlp(s, q, asc, h, ids, weights, *mats, e, out)
    close_bf16(values(out, s).reshape(m, h), *c.want())


@pytest.mark.parametrize("m", [4, 40, 4000])
def test_adapters_past_four_gib(env, m):
    """The last of 1023 adapters of rank 256, rows again and again: row by row and with the
    rows sorted, every row has the outputs of its first."""
    mod, s, _ = env
    n = k = 8320
    count, rank, period = 1023, 256, 4
    c = Adapters(period, n, k, rank, 1, seed=m, ids=[0, -1, 0, 0])
    a, b = at_the_end(s, count, bf16_bits(c.a)), at_the_end(s, count, bf16_bits(c.b))
    assert a.nbytes > 1 << 32 and b.nbytes > 1 << 32
    scaling = at_the_end(s, count, c.scaling)
    reps = m // period
    q, asc, x, ids = (DeviceBuffer.from_host(s, np.concatenate([v] * reps)) for v in (
        c.q, c.asc, bf16_bits(c.x), np.where(c.ids == 0, count - 1, -1).astype(np.int32)))
    out = DeviceBuffer(m * n, np.uint16)
    mod.linear_adapters(s, q, asc, DeviceBuffer.from_host(s, c.w), DeviceBuffer.from_host(s, c.ws), k, x, ids, a, b,
                        scaling, out)
    got = values(out, s).reshape(reps, period, n)
    close_bf16(got[0], *c.want())
    assert (got == got[0]).all()
