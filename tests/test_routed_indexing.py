"""The routed layers' index arithmetic, replayed on the CPU: which workgroup
takes which tile, how many tiles a sort can list, and that the rings of the K
loop never read a stage that has not landed nor overwrite one still read
(inferrous_amd/csrc/experts_tiles.hip, row_sort.hpp, tile_stream.hpp)."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import _lib


@pytest.mark.parametrize("seed", range(8))
def test_every_live_tile_has_one_workgroup(seed):
    """own_tile: workgroups 0 .. grid - 1 (a multiple of 8, for the most tiles there
    can be) take each (tile, part, column) of the live ones once."""
    rng = np.random.default_rng(seed)
    experts, slots = int(rng.integers(1, 200)), int(rng.integers(1, 5000))
    bt, parts, cols = [(32, 1, 6), (64, 1, 9), (128, 1, 16), (256, 2, 4), (256, 1, 5)][seed % 5]
    share = rng.dirichlet(np.full(experts, 0.3))
    counts = np.bincount(rng.choice(experts, slots, p=share), minlength=experts)
    tiles = int(np.sum(-(-counts // bt)))
    most = slots // bt + min(slots, experts)
    assert tiles <= most
    grid = -(-most * parts * cols // 8) * 8
    work = tiles * parts * cols
    per = -(-work // 8)
    taken = []
    for b in range(grid):
        at = b % 8 * per + b // 8
        if b // 8 < per and at < work:
            taken.append((at // cols, at % cols))
    assert sorted(taken) == [(u, c) for u in range(tiles * parts) for c in range(cols)]


@pytest.mark.parametrize("items, classes", [(1, 1), (63, 3), (64, 64), (1000, 7), (4096, 1023), (4097, 5), (9000, 60)])
def test_sort_positions(items, classes):
    """The counting sort's runs, counts and peers give the stable order."""
    rng = np.random.default_rng(items)
    ids = rng.integers(-1, classes + 1, items)
    per = items if items <= 4096 else 1024 if items <= 64 * 4096 else 4096
    blocks = -(-items // per)
    live = (ids >= 0) & (ids < classes)
    totals = np.bincount(ids[live], minlength=classes)
    first = np.concatenate([[0], np.cumsum(totals)[:-1]])
    pos = np.full(items, -1)
    for b in range(blocks):
        b0, b1 = min(b * per, items), min((b + 1) * per, items)
        before = np.bincount(ids[:b0][live[:b0]], minlength=classes)
        run = -(-(b1 - b0) // 1024) * 64
        assert run <= 64 * 4  # a lane's items fit its registers
        nxt = first + before
        for w in range(16):
            begin = min(b0 + w * run, b1)
            for i in range(begin, min(begin + run, b1)):
                if live[i]:
                    pos[i] = nxt[ids[i]]
                    nxt[ids[i]] += 1
    order = np.argsort(np.where(live, ids, classes), kind="stable")[:live.sum()]
    assert np.array_equal(pos[order], np.arange(live.sum()))


@pytest.mark.parametrize("sa, sb", [(2, 2), (2, 3), (3, 3), (4, 4), (2, 4)])
@pytest.mark.parametrize("la, ln", [(1, 4), (4, 4), (3, 2), (5, 4), (1, 8)])
@pytest.mark.parametrize("kt_count", [1, 2, 3, 4, 5, 9, 32])
def test_rings_of_the_k_loop(sa, sb, la, ln, kt_count):
    """One wave's issue order and waits: when stage kt + 1 is read every load of it
    has landed (loads complete in order, a wait leaves the newest n), and a load's
    slot was released by a barrier after its last read."""
    issued, landed, slots = [], 0, {}
    reads_done = -1  # the last stage that a barrier released

    def load(ring, depth, kt):
        old = slots.get((ring, kt % depth))
        assert old is None or old <= reads_done, (ring, kt, old, reads_done)
        slots[(ring, kt % depth)] = kt
        issued.extend([(ring, kt)] * (la if ring == "t" else ln))

    def wait(n):
        nonlocal landed
        landed = max(landed, len(issued) - n)

    def check(kt):
        for ring, depth in (("t", sa), ("n", sb)):
            assert slots[(ring, kt % depth)] == kt
            assert max(i for i, l in enumerate(issued) if l == (ring, kt)) < landed, (ring, kt)

    for s in range(sb - 1):
        if s >= kt_count:
            break
        if s < sa - 1:
            load("t", sa, s)
        load("n", sb, s)
    wait((sa - 2) * la + (sb - 2) * ln if kt_count >= sb - 1 else 0)
    if sa - 1 < kt_count:
        load("t", sa, sa - 1)
    check(0)
    for kt in range(kt_count - 1):
        more_n, more_t = kt + sb - 1 < kt_count, kt + sa < kt_count
        if more_n:
            load("n", sb, kt + sb - 1)
        wait((ln if sb > sa else 0) + (sa - 2) * (la + ln) if more_n else 0)
        reads_done = kt  # the barrier: stage kt is read
        check(kt + 1)
        if more_t:
            load("t", sa, kt + sa)


def test_workspaces_grow_with_the_rows_of_one_form():
    """More rows of the same form never need less; every form's need is positive and
    a multiple of 256."""
    L = _lib.lib()
    for k, e, h, i in ((8, 128, 2048, 768), (2, 8, 2048, 1024), (1, 1, 16, 16)):
        sizes = [L.w8a8_experts_mlp_workspace_bytes(m, k, e, h, i) for m in (65, 128, 1000, 4096, 20000)]
        assert all(s > 0 and s % 256 == 0 for s in sizes) and sizes == sorted(sizes)
        assert L.w8a8_experts_mlp_workspace_bytes(0, k, e, h, i) == 0
    assert L.w8a8_experts_mlp_workspace_bytes(4, 2, 8, 72, 16) == 0
    for m in (1, 2, 64, 300, 5000):
        assert L.w8a8_linear_adapters_workspace_bytes(m, 4096, 4096, 16, 4) > 0
    assert L.w8a8_linear_adapters_workspace_bytes(8, 4096, 4096, 12, 4) == 0
