"""The page table's width (no GPU): a buffer for more sequences than the batch has
is read by the width that the caller names, never by a guess."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import KvCache, _lib, module
from inferrous_amd.module import LoadedModule
from test_routed_refusals import A, Buf

F, B, I, U = np.float32, np.uint16, np.int32, np.uint8
M, HEADS, KV, DIM = 3, 4, 2, 64


class Recorder:
    """In the library's place: the arguments of the last call."""

    def __getattr__(self, name):
        def call(*args):
            self.args = args
            return _lib.OK
        return call


@pytest.fixture
def calls(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(module, "lib", lambda: r)
    return r


def cache():
    return KvCache.over(Buf(10 * KV * 128 * DIM, U), Buf(10 * KV * 2, F), 1, 10, KV, DIM)


def decode(calls, table, lengths=M, **kw):
    mod = LoadedModule(None)
    mod._routed_workspace = lambda stream, size_of, *shape, **kw: (A, shape)
    mod.attention_decode(None, Buf(M * HEADS * DIM, B), cache(), Buf(lengths, I), Buf(table, I), HEADS,
                         Buf(M * HEADS * DIM, B), **kw)
    assert calls.args[-1] == (M, HEADS, KV, DIM, calls.args[11])   # the workspace's shape has the same width
    return calls.args[11]


def prepare(calls, table, past=M, seqs=M, starts=False, **kw):
    if starts:
        kw["starts"] = Buf(seqs + 1, I)
    LoadedModule(None).prepare_qk(None, Buf(M * (HEADS + 2 * KV) * DIM, B), HEADS, KV, DIM, Buf(10 * DIM, F),
                                  Buf(M * HEADS * DIM, B), past=Buf(past, I), cache=cache(), table=Buf(table, I), **kw)
    return calls.args[-1]


CALLS = [decode, prepare, lambda *a, **kw: prepare(*a, starts=True, **kw)]


@pytest.mark.parametrize("call", CALLS)
def test_a_table_of_the_batch(calls, call):
    assert call(calls, M * 5) == 5
    assert call(calls, M * 5, table_width=5) == 5


@pytest.mark.parametrize("call", CALLS)
def test_a_table_for_more_sequences(calls, call):
    """64 rows of 6 pages are three rows of 6, not of 128."""
    assert call(calls, 64 * 6, 64, table_width=6) == 6
    assert call(calls, 64 * 6, table_width=6) == 6
    assert call(calls, M * 6 + 1, table_width=6) == 6


@pytest.mark.parametrize("call", CALLS)
def test_a_width_that_could_be_two_is_refused(calls, call):
    """Every sequence's buffers are for 6 of them: the table's 36 are 6 rows of 6 or 3 of 12."""
    with pytest.raises(ValueError, match="table_width"):
        call(calls, 6 * 6, 6)
    assert call(calls, 3 * 7, 6) == 7     # six rows it cannot be


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("table, width", [(M * 5, 6), (M * 5, 0), (M * 5, -5), (M * 5 - 1, 5)])
def test_a_width_that_the_table_does_not_have(calls, call, table, width):
    with pytest.raises(ValueError):
        call(calls, table, table_width=width)
