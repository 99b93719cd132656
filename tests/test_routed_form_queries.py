"""The queries of the routed layers' forms (no GPU), and the two-stage ring of the
K loop that sums block by block, replayed (inferrous_amd/csrc/tile_stream.hpp)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from inferrous_amd import _lib


def query(op, *shape, length=8, null=False):
    got = (ctypes.c_int32 * 8)(*[7] * 8)
    status = getattr(_lib.lib(), f"w8a8_diag_{op}_form")(*shape, None if null else got, length)
    return status, list(got)


@pytest.mark.parametrize("op, shape, refused", [
    ("experts", (8, 2, 8, 64, 48), [(8, 2, 8, 72, 48), (8, 0, 8, 64, 48), (8, 2, 1025, 64, 48), (1 << 24, 2, 8, 64, 48)]),
    ("adapters", (8, 33, 64, 16, 4), [(8, 33, 72, 16, 4), (8, 33, 64, 12, 4), (8, 33, 64, 16, 1024),
                                      ((1 << 21) + 1, 33, 64, 16, 4)])])
def test_form_queries(op, shape, refused):
    assert query(op, *shape)[0] == _lib.OK and query(op, *shape)[1][0] in (1, 2, 3)
    assert query(op, *shape, null=True)[0] == _lib.ENULL
    assert query(op, *shape, length=7)[0] == _lib.EWORKSPACE
    assert query(op, 0, *shape[1:]) == (_lib.OK, [0] * 8)
    for r in refused:
        assert query(op, *r)[0] == _lib.ESHAPE


def test_forms_follow_the_rows():
    """One row, a decode batch and a prompt of the benchmark's sizes."""
    assert [query("experts", m, 8, 64, 4096, 1024)[1][:2] for m in (1, 256, 1024, 4096)] == [
        [1, 0], [2, 128], [2, 128], [2, 256]]
    assert [query("adapters", m, 4096, 4096, 16, 4)[1][0] for m in (1, 4, 64, 4096)] == [1, 1, 2, 3]


@pytest.mark.parametrize("la, ln", [(9, 8), (2, 1), (5, 4)])
@pytest.mark.parametrize("kt_count", [1, 2, 3, 8, 33])
def test_ring_of_the_blocked_k_loop(la, ln, kt_count):
    """Before stage kt is read every load of it has landed for every wave, and the next
    stage's loads go where the last stage's reads have returned."""
    issued, slots, landed, reads_done = [], {}, 0, -1

    def loads(kt):
        for ring, n in (("t", la), ("n", ln)):
            old = slots.get((ring, kt % 2))
            assert old is None or old <= reads_done
            slots[(ring, kt % 2)] = kt
            issued.extend([(ring, kt)] * n)

    loads(0)
    for kt in range(kt_count):
        landed = len(issued)          # the wait for all loads, then the barrier
        reads_done = kt - 1           # every wave waited for its reads of the last stage
        if kt + 1 < kt_count:
            loads(kt + 1)
        for ring in ("t", "n"):
            assert slots[(ring, kt % 2)] == kt
            assert max(i for i, l in enumerate(issued) if l == (ring, kt)) < landed
    assert np.unique([kt for _, kt in issued]).size == kt_count
