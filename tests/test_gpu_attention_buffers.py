"""Attention on buffers that a program keeps for its largest batch: tables, lengths
and rows for more sequences than the call has.  (Inputs, 64-bit forms and
tolerances: test_gpu_attention.py.)"""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, DeviceBuffer, load
from test_gpu_attention import Decode, Prepare, bf16_bits, close, dev, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


def test_decode_of_fewer_rows_than_the_buffers(env):
    mod, s, _ = env
    c = Decode(1, [130, 5, 64, 200, 77, 1, 0, 191], 8, 2, 128)   # 8 rows of 4 pages
    q, cache, lengths = dev(s, bf16_bits(c.q)), c.cache.put(s), dev(s, np.array(c.lengths, np.int32))
    table = dev(s, c.table)
    want, err = c.want()
    for m in (1, 2, 4, 8):
        out = dev(s, np.full(8 * 8 * 128, 7, np.uint16))
        mod.attention_decode(s, q, cache, lengths, table, 8, DeviceBuffer.view_of(out, 0, m * 8 * 128),
                             table_width=c.width)
        got = values(out, s).reshape(8, 8, 128)
        close(got[:m], want[:m], err[:m])
        assert np.all(out.to_host_vec(s).reshape(8, -1)[m:] == 7)


@pytest.mark.parametrize("packed", [False, True])
def test_prepare_of_fewer_sequences_than_the_buffers(env, packed):
    """The pages of the sequences behind the batch are left as they were."""
    mod, s, _ = env
    c = Prepare(2, [1, 1, 1, 1], [130, 5, 64, 200], 8, 2, 128)
    behind = c.table[2:][c.table[2:] >= 0]
    table = dev(s, c.table)
    c.rows, c.past, c.m, c.starts = c.rows[:2], c.past[:2], 2, c.starts[:3]
    past = dev(s, np.array([130, 5, 64, 200], np.int32))
    c.held, kv = c.cache.put(s), c.kv
    c.q_out, c.k_out, c.v_out = (dev(s, np.full(2 * n * 128, 0x4242, np.uint16)) for n in (8, kv, kv))
    mod.prepare_qk(s, dev(s, bf16_bits(c.x)), 8, kv, 128, dev(s, c.rope), c.q_out, q_gain=dev(s, c.gains[0]),
                   k_gain=dev(s, c.gains[1]), starts=dev(s, c.starts) if packed else None, past=past, k_out=c.k_out,
                   v_out=c.v_out, cache=c.held, table=table, table_width=c.width)
    codes = c.held.codes.to_host_vec(s).reshape(c.cache.pages, -1)[behind]
    assert np.array_equal(codes, c.cache.codes().reshape(c.cache.pages, -1)[behind])
    c.x = c.x[:2]
    c.check(s)
