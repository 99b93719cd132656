"""Every form of experts_mlp and linear_adapters that the host rules choose, at
small shapes: each case says which form it has to take (asked from the library,
so that a changed rule cannot move it elsewhere unseen), and is checked against
the 64-bit definition.  The same forms replayed from graphs with new ids."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from inferrous_amd import CudaContext, DeviceBuffer, Graph, load
from inferrous_amd._lib import OUT_I32, PATH_AUTO, lib
from test_gpu_routed import Adapters, Experts, bf16_bits, close_bf16, values

pytestmark = pytest.mark.gpu

F32 = np.float32


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


def form(op, *shape):
    got = (ctypes.c_int32 * 8)()
    assert getattr(lib(), f"w8a8_diag_{op}_form")(*shape, got, 8) == 0
    return list(got)


# ------------------------------------------------------------------ experts
SLOTS, TILES = 1, 2

# (rows, slots a row, experts, hidden, inner): tile rows, gate / up and down with four stages.
# Hidden and inner of whole 128s, and with 16 more: K tails.
EXPERT_FORMS = [
    ((70, 2, 16, 128, 128), 32, 1, 1),
    ((70, 2, 16, 256, 256), 32, 1, 1),
    ((90, 2, 16, 1152, 640), 32, 1, 1),
    ((200, 3, 130, 256, 256), 32, 0, 1),
    ((200, 3, 130, 512, 128), 32, 1, 0),
    ((200, 3, 130, 512, 256), 32, 0, 0),
    ((200, 3, 130, 768, 384), 32, 0, 0),
    ((150, 2, 8, 256, 128), 64, 0, 0),
    ((150, 2, 8, 640, 384), 64, 0, 0),
    ((300, 2, 6, 128, 256), 128, 0, 0),
    ((300, 2, 6, 512, 640), 128, 0, 0),
    ((600, 1, 3, 256, 128), 256, 0, 0),
    ((600, 1, 3, 384, 512), 256, 0, 0),
]


@pytest.mark.parametrize("shape, bt, gate_deep, down_deep", EXPERT_FORMS)
@pytest.mark.parametrize("hidden_tail, inter_tail", [(0, 0), (16, 0), (0, 112), (64, 48)])
def test_experts_forms(env, shape, bt, gate_deep, down_deep, hidden_tail, inter_tail):
    m, k, e, h, f = shape
    h, f = h - hidden_tail, f - inter_tail
    got = form("experts", m, k, e, h, f)
    assert [got[0], got[1], *got[4:]] == [TILES, bt, gate_deep, down_deep, hidden_tail > 0, inter_tail > 0]
    Experts(m, k, e, h, f, seed=m + h + f, residual=inter_tail == 48).check(env)


@pytest.mark.parametrize("counts", [[400, 150, 50], [256, 257, 87], [1, 64, 65, 128, 129, 600], [0, 900, 0, 31, 32, 33],
                                    [256, 0, 512, 128, 64]])
def test_experts_tiles_of_every_height(env, counts):
    """Shares that leave a 256-row launch tiles of each of its forms, and experts that no
    row meets."""
    rng = np.random.default_rng(len(counts))
    ids = rng.permutation(np.repeat(np.arange(len(counts)), counts))[:, None]
    m, e = len(ids), len(counts)
    if m // e <= 128:
        ids, m = np.repeat(ids, 3, 0), 3 * m
    assert form("experts", m, 1, e, 272, 384)[1] == 256
    Experts(m, 1, e, 272, 384, seed=e, ids=ids).check(env)


@pytest.mark.parametrize("m, k, e", [(70, 12, 20), (66, 9, 9), (80, 24, 64), (65, 64, 64)])
def test_experts_more_than_eight_slots_in_tiles(env, m, k, e):
    """The weighted sum takes its slots eight at a time."""
    assert form("experts", m, k, e, 144, 128)[0] == TILES
    rng = np.random.default_rng(m)
    ids = np.stack([rng.permutation(e)[:k] for _ in range(m)])
    ids[rng.random((m, k)) < 0.2] = -1
    ids[3, 8:] = -1
    ids[4, :8] = -1
    Experts(m, k, e, 144, 128, seed=m, ids=ids, residual=True).check(env, F32)


@pytest.mark.parametrize("m, k, e, h, f, want", [
    (100, 4, 24, 256, 128, 32), (90, 4, 9, 256, 144, 64), (400, 2, 10, 144, 128, 128), (700, 1, 4, 256, 256, 256),
    (2100, 2, 200, 128, 128, 32)])
def test_experts_in_tiles_replayed(env, m, k, e, h, f, want):
    """A captured call in tiles follows new ids, weights and rows at every replay,
    skewed shares and empty slots among them, and equals the eager call each time."""
    mod, s, _ = env
    assert form("experts", m, k, e, h, f)[:2] == [TILES, want]
    rng = np.random.default_rng(m)
    cs = [Experts(m, k, e, h, f, seed=3 + i) for i in range(3)]
    cs[1].ids = np.where(rng.random((m, k)) < 0.3, -1, rng.integers(0, max(1, e // 3), (m, k))).astype(np.int32)
    cs[2].ids = np.full((m, k), e - 1, np.int32)
    c = cs[0]
    mod.reserve_workspace(mod.experts_mlp_workspace_bytes(m, k, e, h, f), s)
    bufs = [DeviceBuffer.from_host(s, a) for a in (c.q, c.asc, c.ids, c.weights)]
    mats = [DeviceBuffer.from_host(s, a) for a in (c.wg, c.sg, c.wu, c.su, c.wd, c.sd)]
    out = DeviceBuffer(m * h, np.uint16)
    graph = Graph(s)
    with graph:
        mod.experts_mlp(s, bufs[0], bufs[1], h, bufs[2], bufs[3], *mats, e, out)
    for n in cs + cs:
        for buf, a in zip(bufs, (n.q, n.asc, n.ids, n.weights)):
            buf.copy_from_host(s, a)
        graph.launch(s)
        s.synchronize()
        n.wg, n.sg, n.wu, n.su, n.wd, n.sd = c.wg, c.sg, c.wu, c.su, c.wd, c.sd
        assert np.array_equal(values(out, s).reshape(m, h), n.run(env))


# ------------------------------------------------------------------ adapters
ONE, ROWS, SORTED = 1, 2, 3

# (rows, columns, width, rank, adapters): the first product's values a wave, and whether the
# projection leaves split-K slabs.
ROW_FORMS = [((1, 40, 64, 16, 2), ONE, 1), ((4, 70, 1040, 256, 3), ONE, 1), ((30, 130, 272, 16, 3), ROWS, 1),
             ((200, 160, 256, 24, 4), ROWS, 2), ((90, 264, 144, 128, 5), ROWS, 2), ((300, 96, 128, 64, 9), ROWS, 8),
             ((170, 33, 80, 104, 3), ROWS, 8)]


@pytest.mark.parametrize("shape, which, each", ROW_FORMS)
@pytest.mark.parametrize("x_bf16", [False, True])
def test_adapters_row_forms(env, shape, which, each, x_bf16):
    assert form("adapters", *shape)[:2] == [which, each]
    Adapters(*shape, seed=sum(shape), residual=not x_bf16).check(env, F32 if x_bf16 else np.uint16, x_bf16=x_bf16)


@pytest.mark.parametrize("shape", [(64, 512, 4096, 16, 3), (40, 96, 12288, 8, 2), (70, 1024, 6400, 24, 5)])
def test_adapters_from_slabs(env, shape):
    """The second product's kernel adds the projection's split-K slabs itself."""
    m, n, k, _, _ = shape
    route = (ctypes.c_int32 * 20)()
    need = lib().w8a8_linear_workspace_bytes_path(m, n, k, PATH_AUTO)
    assert lib().w8a8_diag_linear_route(m, n, k, OUT_I32, 0, PATH_AUTO, need, route, 20) == 0
    assert form("adapters", *shape)[0] == ROWS and route[14] > 1
    Adapters(*shape, seed=m, residual=True).check(env)


# (rows, columns, width, adapters), then rows of a tile of the first product, its shares of
# K, tiles of the projection, and a K tail.
SORTED_FORMS = [((1500, 3000, 400, 32), 32, 1, 128, 1), ((1500, 1024, 2000, 10), 128, 4, 128, 1),
                ((1000, 3000, 1024, 21), 32, 2, 128, 0), ((1300, 2999, 384, 7), 128, 1, 128, 0)]


@pytest.mark.parametrize("shape, bt, shares, tile, tail", SORTED_FORMS)
@pytest.mark.parametrize("rank, ranks", [(24, 32), (64, 64), (104, 128), (200, 256)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_adapters_sorted_forms(env, shape, bt, shares, tile, tail, rank, ranks, x_bf16):
    m, n, k, count = shape
    assert form("adapters", m, n, k, rank, count) == [SORTED, bt, ranks, shares, 1, tile, tail, 0]
    Adapters(m, n, k, rank, count, seed=m + rank, residual=rank == 64).check(env, F32 if rank == 104 else np.uint16,
                                                                             x_bf16=x_bf16)


@pytest.mark.parametrize("m, n, k, rank, count, tail", [
    (4096, 3000, 384, 16, 6, 0), (4096, 3001, 272, 64, 3, 1), (4000, 3088, 144, 8, 90, 1), (5000, 2561, 128, 128, 40, 0)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_adapters_in_large_tiles(env, m, n, k, rank, count, tail, x_bf16):
    """256 x 256 tiles of the projection, which a full context takes: runs of one
    adapter, many in a tile, rows without any, ragged rows and columns."""
    assert form("adapters", m, n, k, rank, count)[5:7] == [256, tail]
    rng = np.random.default_rng(m + n)
    ids = rng.integers(-1, count, m)
    ids[m // 3:2 * m // 3] = count - 1
    Adapters(m, n, k, rank, count, seed=n, ids=ids, residual=x_bf16).check(env, F32 if rank == 64 else np.uint16,
                                                                          x_bf16=x_bf16)


def test_adapters_sorted_by_many_workgroups(env):
    """More rows than 64 workgroups of 4096 sort."""
    m, n, k, rank, count = 270_001, 8, 16, 8, 5
    assert form("adapters", m, n, k, rank, count)[:5] == [SORTED, 128, 32, 1, 66]
    Adapters(m, n, k, rank, count, seed=2).check(env, x_bf16=True)


@pytest.mark.parametrize("m, n, k, rank, count", [(900, 512, 512, 256, 3), (1500, 1600, 400, 40, 32),
                                                  (4096, 2824, 128, 32, 4)])
def test_adapters_sorted_replayed(env, m, n, k, rank, count):
    """A captured call with sorted rows follows new ids and rows at every replay."""
    mod, s, _ = env
    assert form("adapters", m, n, k, rank, count)[0] == SORTED
    c = Adapters(m, n, k, rank, count, seed=m)
    mod.reserve_workspace(mod.linear_adapters_workspace_bytes(m, n, k, rank, count), s)
    q, asc, w, ws, x, ids, a, b, sc = (DeviceBuffer.from_host(s, v) for v in (
        c.q, c.asc, c.w, c.ws, bf16_bits(c.x), c.ids, bf16_bits(c.a), bf16_bits(c.b), c.scaling))
    out = DeviceBuffer(m * n, np.uint16)
    graph = Graph(s)
    with graph:
        mod.linear_adapters(s, q, asc, w, ws, k, x, ids, a, b, sc, out)
    orders = [c.ids, np.sort(c.ids), np.full(m, count - 1, np.int32), np.full(m, -1, np.int32), c.ids[::-1].copy()]
    for turn, order in enumerate(orders + orders[:2]):
        c.ids, c.x = order, np.roll(c.x, 1, 0)
        ids.copy_from_host(s, c.ids)
        x.copy_from_host(s, bf16_bits(c.x))
        graph.launch(s)
        s.synchronize()
        assert np.array_equal(values(out, s).reshape(m, n), c.run(env, x_bf16=True)), turn
