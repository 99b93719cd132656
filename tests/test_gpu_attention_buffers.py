"""Attention on buffers as programs keep them: tables, lengths and rows for more
sequences than the call has, layers of one cache, rows of any stride.  (Inputs, 64-bit forms and
tolerances: test_gpu_attention.py.)"""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, DeviceBuffer, KvCache, OUT_BF16, OUT_F32, _lib, load
from test_gpu_attention import Decode, Prefill, Prepare, bf16_bits, close, dev, values

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


@pytest.mark.parametrize("layer", [0, 1, 2])
def test_layers_of_a_cache(env, layer):
    """A layer's call gives what a cache of that layer alone does; the others stay as they were."""
    mod, s, _ = env
    c = Decode(3, [300, 70, 4000], 8, 2, 128)
    want = c.run(env)
    rng = np.random.default_rng(layer)
    codes = rng.integers(0, 256, (3, c.cache.pages, 2 * 2 * 64 * 128), dtype=np.uint8)
    scales = np.exp2(rng.integers(-9, 9, (3, c.cache.pages, 4))).astype(np.float32)
    codes[layer], scales[layer] = c.cache.codes().reshape(c.cache.pages, -1), c.cache.s.reshape(c.cache.pages, -1)
    cache = KvCache.over(dev(s, codes), dev(s, scales), 3, c.cache.pages, 2, 128)
    out = DeviceBuffer(c.m * 8 * 128, np.uint16)
    mod.attention_decode(s, dev(s, bf16_bits(c.q)), cache, dev(s, np.array(c.lengths, np.int32)), dev(s, c.table), 8, out,
                         layer=layer)
    assert np.array_equal(values(out, s).reshape(want.shape), want)

    p = Prepare(4, [70, 3], [10, 64], 8, 2, 128)
    p.run(env)
    alone = [b.to_host_vec(s) for b in (p.held.codes, p.held.scales, p.q_out)]
    n = p.cache.pages
    codes = rng.integers(0, 256, (3, n, 2 * 2 * 64 * 128), dtype=np.uint8)
    scales = np.exp2(rng.integers(-9, 9, (3, n, 4))).astype(np.float32)
    codes[layer], scales[layer] = p.cache.codes().reshape(n, -1), p.cache.s.reshape(n, -1)
    cache = KvCache.over(dev(s, codes), dev(s, scales), 3, n, 2, 128)
    q = DeviceBuffer(p.m * 8 * 128, np.uint16)
    mod.prepare_qk(s, dev(s, bf16_bits(p.x)), 8, 2, 128, dev(s, p.rope), q, q_gain=dev(s, p.gains[0]),
                   k_gain=dev(s, p.gains[1]), starts=dev(s, p.starts), past=dev(s, np.array(p.past, np.int32)),
                   cache=cache, table=dev(s, p.table), layer=layer)
    codes[layer], scales[layer] = alone[0].reshape(n, -1), alone[1].reshape(n, -1)
    assert np.array_equal(cache.codes.to_host_vec(s), codes.reshape(-1))
    assert np.array_equal(cache.scales.to_host_vec(s), scales.reshape(-1))
    assert np.array_equal(q.to_host_vec(s), alone[2])


def apart(a, stride, first, fill):
    """Rows of a [m, ...] with `stride` values from one to the next, `first` values before the first."""
    m = len(a)
    out = np.full(first + m * stride, fill, a.dtype)
    out[first:].reshape(m, stride)[:, :a.reshape(m, -1).shape[1]] = a.reshape(m, -1)
    return out


@pytest.mark.parametrize("heads, kv, dim", [(8, 2, 128), (3, 3, 64), (14, 2, 64)])
@pytest.mark.parametrize("dtype", [OUT_BF16, OUT_F32])
def test_prompts_with_a_stride_each(env, heads, kv, dim, dtype):
    """The C entry's three strides, NaN between the rows."""
    mod, s, _ = env
    c = Prefill(5, [150, 1, 65], heads, kv, dim)
    want = c.run(env)
    strides = heads * dim + 8, kv * dim + 136, (heads + 2 * kv) * dim
    held = [dev(s, apart(bf16_bits(a), n, 8 * i, 0x7FC0)) for i, (a, n) in enumerate(zip((c.q, c.k, c.v), strides))]
    at = [x for i, (b, n) in enumerate(zip(held, strides)) for x in (b.ptr + 16 * i, n)]
    out = DeviceBuffer(c.m * heads * dim, np.uint16 if dtype == OUT_BF16 else np.float32)
    starts = dev(s, c.starts)
    assert _lib.lib().w8a8_attention_prefill(s.handle, *at, c.m, heads, kv, dim, starts.ptr, 3, dim ** -0.5, out.ptr,
                                             dtype) == _lib.OK
    assert np.array_equal(values(out, s).reshape(want.shape), want)


@pytest.mark.parametrize("heads, kv, dim", [(8, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("bf16_rows", [True, False])
@pytest.mark.parametrize("packed", [True, False])
def test_prepare_with_a_stride_each(env, heads, kv, dim, bf16_rows, packed):
    mod, s, _ = env
    rows, past = ([70, 3], [10, 64]) if packed else ([1, 1, 1], [63, 0, 200])
    p = Prepare(6, rows, past, heads, kv, dim)
    p.run(env, one_row=not packed)
    want = [b.to_host_vec(s) for b in (p.q_out, p.k_out, p.v_out, p.held.codes, p.held.scales)]
    strides = heads * dim + 8, kv * dim + 136, (heads + 2 * kv) * dim
    parts = p.x[:, :heads], p.x[:, heads:heads + kv], p.x[:, heads + kv:]
    rows_of = (lambda a: bf16_bits(a)) if bf16_rows else (lambda a: np.ascontiguousarray(a, np.float32))
    fill, size = (0x7FC0, 2) if bf16_rows else (np.nan, 4)
    held = [dev(s, apart(rows_of(a), n, 8 * i, fill)) for i, (a, n) in enumerate(zip(parts, strides))]
    at = [x for i, (b, n) in enumerate(zip(held, strides)) for x in (b.ptr + 8 * size * i, n)]
    cache, table, gains = p.cache.put(s), dev(s, p.table), [dev(s, g) for g in p.gains]
    rope, starts, tokens = dev(s, p.rope), dev(s, p.starts), dev(s, np.array(past, np.int32))
    out = [DeviceBuffer(p.m * n * dim, np.uint16) for n in (heads, kv, kv)]
    assert _lib.lib().w8a8_prepare_qk(
        s.handle, *at, OUT_BF16 if bf16_rows else OUT_F32, p.m, heads, kv, dim, gains[0].ptr, gains[1].ptr, 1e-6, rope.ptr,
        len(p.rope), starts.ptr if packed else None, tokens.ptr, len(rows), out[0].ptr, out[1].ptr, out[2].ptr,
        cache.codes.ptr, cache.scales.ptr, cache.pages, table.ptr, p.width) == _lib.OK
    for got, was in zip([*out, cache.codes, cache.scales], want):
        assert np.array_equal(got.to_host_vec(s), was)
