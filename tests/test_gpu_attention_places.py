"""Attention where memory and streams are not the usual ones: offsets that pass
32 bits, caches that reach to the end of their buffers, streams and graphs beside
each other, and the same call twice.  (Inputs and 64-bit forms:
test_gpu_attention.py.)"""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, DeviceBuffer, Graph, KvCache, load
from test_gpu_attention import Cache, Decode, Prefill, Prepare, bf16_bits, close, dev, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


def test_a_cache_of_more_than_4_gib(env):
    """The pages of an ordinary case moved to both ends of a large cache."""
    mod, s, _ = env
    c = Decode(1, [300, 70, 129, 0, 64], 16, 8, 128)
    pages, held = 40000, c.cache.pages
    block = 8 * 2 * 64 * 128
    big = KvCache(1, pages, 8, 128)
    to = np.where(np.arange(held) % 2 == 0, np.arange(held), pages - 1 - np.arange(held)).astype(np.int32)
    codes = c.cache.codes().reshape(held, -1)
    for i, p in enumerate(to):
        DeviceBuffer.view_of(big.codes, int(p) * block, block).copy_from_host(s, codes[i])
        DeviceBuffer.view_of(big.scales, int(p) * 16, 16).copy_from_host(s, c.cache.s[i].reshape(-1))
    table = np.where(c.table >= 0, to[c.table], -1).astype(np.int32)
    out = DeviceBuffer(c.m * 16 * 128, np.uint16)
    lengths = dev(s, np.array(c.lengths, np.int32))
    mod.attention_decode(s, dev(s, bf16_bits(c.q)), big, lengths, dev(s, table), 16, out)
    close(values(out, s).reshape(c.m, 16, 128), *c.want())

    # the same from copies of those pages, and rows that prepare_qk puts beside them
    again = (20000 + np.arange(held)).astype(np.int32)
    again[1::2] = pages - 1 - held - np.arange(held)[1::2]
    mod.copy_pages(s, big, dev(s, to), dev(s, again))
    table2 = np.where(c.table >= 0, again[c.table], -1).astype(np.int32)
    out2 = DeviceBuffer(c.m * 16 * 128, np.uint16)
    mod.attention_decode(s, dev(s, bf16_bits(c.q)), big, lengths, dev(s, table2), 16, out2)
    assert np.array_equal(out.to_host_vec(s), out2.to_host_vec(s))

    p = Prepare(2, [70, 64], [0, 0], 16, 8, 128)
    ends = (pages - 1 - 2 * held - np.arange(p.cache.pages)).astype(np.int32)
    where = np.where(p.table >= 0, ends[p.table], -1).astype(np.int32)
    q_out = DeviceBuffer(p.m * 16 * 128, np.uint16)
    kw = dict(q_gain=dev(s, p.gains[0]), k_gain=dev(s, p.gains[1]), starts=dev(s, p.starts))
    mod.prepare_qk(s, dev(s, bf16_bits(p.x)), 16, 8, 128, dev(s, p.rope), q_out, cache=big, table=dev(s, where), **kw)
    small = KvCache(1, p.cache.pages, 8, 128)
    mod.prepare_qk(s, dev(s, bf16_bits(p.x)), 16, 8, 128, dev(s, p.rope), q_out, cache=small, table=dev(s, p.table), **kw)
    codes, scales = small.codes.to_host_vec(s).reshape(-1, block), small.scales.to_host_vec(s).reshape(-1, 16)
    for page in p.table[p.table >= 0]:
        at = int(ends[page])
        assert np.array_equal(DeviceBuffer.view_of(big.codes, at * block, block).to_host_vec(s), codes[page])
        assert np.array_equal(DeviceBuffer.view_of(big.scales, at * 16, 16).to_host_vec(s), scales[page])


def test_rows_further_apart_than_4_gib(env):
    mod, s, _ = env
    c = Prefill(3, [2100], 2, 1, 64)
    stride = 1 << 20
    wide = DeviceBuffer(2099 * stride + 64, np.uint16)
    v = bf16_bits(c.v).reshape(-1, 64)
    for r in range(2100):
        DeviceBuffer.view_of(wide, r * stride, 64).copy_from_host(s, v[r])
    q, k = dev(s, bf16_bits(c.q)), dev(s, bf16_bits(c.k))
    outs = [DeviceBuffer(2100 * 128, np.uint16) for _ in range(2)]
    mod.attention_prefill(s, q, k, dev(s, v), 2, 1, 64, outs[0])
    mod.attention_prefill(s, q, k, wide, 2, 1, 64, outs[1], v_stride=stride)
    first, second = (o.to_host_vec(s) for o in outs)
    assert np.array_equal(first, second)
    close(values(outs[0], s).reshape(2100, 2, 64), *c.want())


@pytest.mark.parametrize("heads, kv, dim", [(8, 2, 128), (3, 1, 64)])
def test_the_end_of_a_buffer(env, heads, kv, dim):
    """Rows of which the last is a view's, with NaN behind it: never read into a result."""
    mod, s, _ = env
    c = Prefill(4, [1, 65, 100], heads, kv, dim)
    want = c.run(env)
    whole = {}
    for name, a in (("q", c.q), ("k", c.k), ("v", c.v)):
        bits = bf16_bits(a).reshape(-1)
        whole[name] = dev(s, np.concatenate([bits, np.full(64 * 1024, 0x7FC0, np.uint16)]))
        whole[name + "v"] = DeviceBuffer.view_of(whole[name], 0, len(bits))
    out = DeviceBuffer(c.m * heads * dim, np.uint16)
    mod.attention_prefill(s, whole["qv"], whole["kv"], whole["vv"], heads, kv, dim, out, starts=dev(s, c.starts))
    assert np.array_equal(values(out, s).reshape(want.shape), want)


def test_the_same_call_twice_gives_the_same_bits(env):
    for c in (Prefill(5, [700, 3], 8, 2, 128), Decode(6, [5000, 40, 900], 8, 2, 128), Decode(7, [2000], 7, 1, 64)):
        first = c.run(env)
        for _ in range(3):
            assert np.array_equal(c.run(env), first)


def test_two_streams_at_once(env):
    """Each stream's calls use its own workspace."""
    mod, _, ctx = env
    streams = [ctx.new_stream() for _ in range(2)]
    cases = [Decode(8, [4000, 500], 8, 2, 128), Decode(9, [700, 3900, 20], 8, 2, 128)]
    held = []
    for s, c in zip(streams, cases):
        held.append(dict(q=dev(s, bf16_bits(c.q)), cache=c.cache.put(s), lengths=dev(s, np.array(c.lengths, np.int32)),
                         table=dev(s, c.table), heads=8, out=DeviceBuffer(c.m * 8 * 128, np.uint16)))
        mod.attention_decode(s, **held[-1])
        s.synchronize()
    want = [h["out"].to_host_vec(s) for h, s in zip(held, streams)]
    for h, s in zip(held, streams):
        h["out"].fill_zero(s)
    for _ in range(50):
        for h, s in zip(held, streams):
            mod.attention_decode(s, **h)
    for h, s, w, c in zip(held, streams, want, cases):
        assert np.array_equal(h["out"].to_host_vec(s), w)
        close(values(h["out"], s).reshape(c.m, 8, 128), *c.want())


def test_prompts_replayed(env):
    """A captured append, attention and copy: new rows, lengths and pairs in the same buffers."""
    mod, _, ctx = env
    s = ctx.new_stream()
    a, b = Prepare(10, [40, 100, 7], [0, 0, 0], 8, 2, 128), Prepare(11, [100, 7, 40], [0, 0, 0], 8, 2, 128)
    width = max(a.width, b.width)
    cache = [KvCache(1, 24, 2, 128) for _ in range(2)]
    rope, m = dev(s, max(a.rope, b.rope, key=len)), a.m
    x, starts, table = DeviceBuffer(a.x.size, np.uint16), DeviceBuffer(4, np.int32), DeviceBuffer(3 * width, np.int32)
    src, dst = DeviceBuffer(2, np.int32), DeviceBuffer(2, np.int32)
    q, out = ([DeviceBuffer(m * 8 * 128, np.uint16) for _ in range(2)] for _ in range(2))
    k, v = ([DeviceBuffer(m * 2 * 128, np.uint16) for _ in range(2)] for _ in range(2))

    def step(i):
        mod.prepare_qk(s, x, 8, 2, 128, rope, q[i], starts=starts, k_out=k[i], v_out=v[i], cache=cache[i], table=table)
        mod.attention_prefill(s, q[i], k[i], v[i], 8, 2, 128, out[i], starts=starts)
        mod.copy_pages(s, cache[i], src, dst)

    graph = Graph(s)
    with graph:
        step(1)
    for n in range(4):
        c = (a, b)[n % 2]
        x.copy_from_host(s, bf16_bits(c.x).reshape(-1))
        starts.copy_from_host(s, c.starts)
        t = np.full((3, width), -1, np.int32)
        t[:, :c.width] = np.where(c.table >= 0, c.table + n, -1)
        table.copy_from_host(s, t.reshape(-1))
        src.copy_from_host(s, np.array([n, n + 1], np.int32))
        dst.copy_from_host(s, np.array([20 + n % 2, 22 + n % 2], np.int32))
        step(0)
        s.synchronize()
        graph.launch(s)
        for pair in (q, out, k, v):
            assert np.array_equal(pair[0].to_host_vec(s), pair[1].to_host_vec(s))
        for name in ("codes", "scales"):
            one, two = (getattr(i, name).to_host_vec(s) for i in cache)
            assert np.array_equal(one, two)


def test_an_empty_batch_and_one_row(env):
    mod, s, _ = env
    Prefill(12, [0, 1, 0], 4, 2, 64).check(env)
    Decode(13, [1], 1, 1, 64).check(env)
    rng = np.random.default_rng(0)
    cache = Cache(rng, 2, 2, 64).put(s)
    none = DeviceBuffer.view_of(DeviceBuffer(8, np.uint16), 0, 0)
    mod.attention_prefill(s, none, none, none, 4, 2, 64, none)
    mod.attention_decode(s, none, cache, DeviceBuffer.view_of(DeviceBuffer(1, np.int32), 0, 0), dev(s, np.zeros(1, np.int32)),
                         4, none)
