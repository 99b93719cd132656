"""Attention's host-side checks (no GPU): malformed arguments are refused with
the documented status before any HIP call, the Python methods refuse wrong
lengths and types, and the page bookkeeping keeps its promises."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import KvCache, PagePool, _lib
from inferrous_amd.module import LoadedModule
from test_routed_refusals import A, Buf, no_device

WELL = _lib.EINIT  # a well-formed call stops at the init check
without_gpu = pytest.mark.skipif(not no_device(), reason="well-formed calls on fake addresses: without a GPU only")


def prepare(**kw):
    a = dict(q=A, qs=48 * 128, k=A, ks=48 * 128, v=A, vs=48 * 128, dt=_lib.OUT_BF16, m=3, h=32, kv=8, d=128, qg=A, kg=A,
             eps=1e-6, rope=A, rr=100, starts=A, past=A, s=2, qo=A, ko=A, vo=A, c=A, sc=A, pages=10, t=A, w=4)
    a.update(kw)
    return _lib.lib().w8a8_prepare_qk(None, *a.values())


@without_gpu
@pytest.mark.parametrize("kw, status", [
    (dict(), WELL), (dict(dt=_lib.OUT_F32), WELL), (dict(qg=None, kg=None, past=None, ko=None, vo=None), WELL),
    (dict(c=None, sc=None, t=None, pages=0, w=0), WELL), (dict(starts=None, s=3), WELL), (dict(m=0, q=None), _lib.OK),
    (dict(dt=_lib.OUT_I32), _lib.EARG), (dict(eps=-1.0), _lib.EARG), (dict(eps=float("nan")), _lib.EARG),
    (dict(d=96), _lib.ESHAPE), (dict(h=0), _lib.ESHAPE), (dict(kv=0), _lib.ESHAPE), (dict(kv=7), _lib.ESHAPE),
    (dict(h=1032), _lib.ESHAPE), (dict(qs=4088), _lib.ESHAPE), (dict(qs=4100), _lib.ESHAPE), (dict(ks=1016), _lib.ESHAPE),
    (dict(vs=1028), _lib.ESHAPE), (dict(starts=None), _lib.ESHAPE), (dict(s=0), _lib.ESHAPE), (dict(rr=0), _lib.ESHAPE),
    (dict(pages=0), _lib.ESHAPE), (dict(pages=1 << 31), _lib.ESHAPE), (dict(w=0), _lib.ESHAPE),
    (dict(m=1 << 25), _lib.ESHAPE), (dict(m=1 << 22, starts=None, s=1 << 22), _lib.ESHAPE),
    *[({n: None}, _lib.ENULL) for n in ("q", "k", "v", "rope", "qo", "sc", "t")],
    *[({n: A + 8}, _lib.EALIGN) for n in ("q", "k", "v", "qg", "kg", "rope", "qo", "ko", "vo", "c")],
    *[({n: A + 2}, _lib.EALIGN) for n in ("starts", "past", "sc", "t")]])
def test_prepare_qk(kw, status):
    assert prepare(**kw) == status


def prefill(**kw):
    a = dict(q=A, qs=4096, k=A, ks=1024, v=A, vs=6144, m=3, h=32, kv=8, d=128, starts=A, s=2, scale=0.1, out=A,
             dt=_lib.OUT_BF16)
    a.update(kw)
    return _lib.lib().w8a8_attention_prefill(None, *a.values())


@without_gpu
@pytest.mark.parametrize("kw, status", [
    (dict(), WELL), (dict(dt=_lib.OUT_F32), WELL), (dict(starts=None, s=1), WELL), (dict(m=0, q=None), _lib.OK),
    (dict(dt=_lib.OUT_I32), _lib.EARG), (dict(scale=0.0), _lib.EARG), (dict(scale=-1.0), _lib.EARG),
    (dict(scale=float("nan")), _lib.EARG), (dict(scale=float("inf")), _lib.EARG), (dict(d=32), _lib.ESHAPE),
    (dict(kv=5), _lib.ESHAPE), (dict(qs=4104 - 16), _lib.ESHAPE), (dict(ks=1028), _lib.ESHAPE), (dict(s=0), _lib.ESHAPE),
    (dict(starts=None), _lib.ESHAPE), (dict(m=(1 << 24) + 1), _lib.ESHAPE), (dict(m=1 << 24, h=1024, kv=1024, qs=1 << 17,
                                                                              ks=1 << 17, vs=1 << 17), _lib.ESHAPE),
    *[({n: None}, _lib.ENULL) for n in ("q", "k", "v", "out")],
    *[({n: A + 8}, _lib.EALIGN) for n in ("q", "k", "v", "out")], (dict(starts=A + 2), _lib.EALIGN)])
def test_attention_prefill(kw, status):
    assert prefill(**kw) == status


@without_gpu
@pytest.mark.parametrize("stride", ["qs", "ks", "vs"])
def test_strides_keep_offsets_in_32_bits(stride):
    for call in (prepare, prefill):
        assert call(**{stride: 1 << 24}) == WELL and call(**{stride: (1 << 24) + 8}) == _lib.ESHAPE


def decode(short=0, **kw):
    a = dict(q=A, m=3, h=32, kv=8, d=128, c=A, sc=A, pages=10, n=A, t=A, w=64, scale=0.1, out=A, dt=_lib.OUT_BF16, ws=A)
    a.update(kw)
    need = _lib.lib().w8a8_attention_decode_workspace_bytes(a["m"], a["h"], a["kv"], a["d"], a["w"])
    return _lib.lib().w8a8_attention_decode(None, *a.values(), max(0, need - short))


@without_gpu
@pytest.mark.parametrize("kw, status", [
    (dict(), WELL), (dict(dt=_lib.OUT_F32), WELL), (dict(m=0, q=None), _lib.OK), (dict(w=1, ws=None), WELL),
    (dict(dt=_lib.OUT_I32), _lib.EARG), (dict(scale=0.0), _lib.EARG), (dict(scale=float("nan")), _lib.EARG),
    (dict(d=80), _lib.ESHAPE), (dict(kv=3), _lib.ESHAPE), (dict(pages=0), _lib.ESHAPE), (dict(w=0), _lib.ESHAPE),
    (dict(w=(1 << 24) + 1), _lib.ESHAPE), (dict(m=1 << 24), _lib.ESHAPE),
    *[({n: None}, _lib.ENULL) for n in ("q", "c", "sc", "n", "t", "out")],
    *[({n: A + 8}, _lib.EALIGN) for n in ("q", "c", "out", "ws")],
    *[({n: A + 2}, _lib.EALIGN) for n in ("sc", "n", "t")],
    (dict(ws=None), _lib.EWORKSPACE), (dict(m=1, short=1), _lib.EWORKSPACE)])
def test_attention_decode(kw, status):
    assert decode(**kw) == status


@pytest.mark.parametrize("heads, kv", [(32, 8), (14, 2), (40, 1), (8, 8)])
@pytest.mark.parametrize("width", [1, 16, 64, 1024])
def test_a_workspace_for_the_largest_batch_serves_every_smaller_one(heads, kv, width):
    need = [_lib.lib().w8a8_attention_decode_workspace_bytes(m, heads, kv, 128, width) for m in range(1, 600)]
    assert need == sorted(need)


@without_gpu
def test_scale_times_log2_e_is_finite():
    for call in (prefill, decode):
        assert call(scale=2e38) == WELL and call(scale=2.4e38) == _lib.EARG


def copy(**kw):
    a = dict(c=A, sc=A, layers=2, pages=10, kv=8, d=128, src=A, dst=A, n=3)
    a.update(kw)
    return _lib.lib().w8a8_copy_pages(None, *a.values())


@without_gpu
@pytest.mark.parametrize("kw, status", [
    (dict(), WELL), (dict(n=0, c=None), _lib.OK), (dict(d=96), _lib.ESHAPE), (dict(kv=0), _lib.ESHAPE),
    (dict(layers=0), _lib.ESHAPE), (dict(pages=0), _lib.ESHAPE), (dict(pages=1 << 31), _lib.ESHAPE),
    (dict(n=1 << 21, layers=36), _lib.ESHAPE), (dict(layers=0xffffffff, n=0xffffffff), _lib.ESHAPE),
    *[({n: None}, _lib.ENULL) for n in ("c", "sc", "src", "dst")], (dict(c=A + 8), _lib.EALIGN),
    *[({n: A + 2}, _lib.EALIGN) for n in ("sc", "src", "dst")]])
def test_copy_pages(kw, status):
    assert copy(**kw) == status


F, B, I, U = np.float32, np.uint16, np.int32, np.uint8


def cache(pages=10, kv=2, dim=64, layers=2):
    return KvCache.over(Buf(layers * pages * kv * 128 * dim, U), Buf(layers * pages * kv * 2, F), layers, pages, kv, dim)


def test_cache_refuses():
    for kw in (dict(layers=0), dict(pages=0), dict(kv=0), dict(dim=96)):
        with pytest.raises(ValueError):
            cache(**kw)
    with pytest.raises(ValueError):
        KvCache.over(Buf(2 * 128 * 64 - 1, U), Buf(4, F), 1, 1, 2, 64)
    with pytest.raises(ValueError):
        KvCache.over(Buf(2 * 128 * 64, U), Buf(3, F), 1, 1, 2, 64)
    with pytest.raises(TypeError):
        KvCache.over(Buf(2 * 128 * 64, B), Buf(4, F), 1, 1, 2, 64)
    for i in (-1, 2):
        with pytest.raises(ValueError):
            cache().layer(i)
    assert cache().layer(1) == (A + 10 * 2 * 128 * 64, A + 10 * 2 * 8)


@pytest.mark.parametrize("kw", [
    dict(q=Buf(3 * 8 * 64 - 1, B)), dict(q=Buf(3 * 8 * 64, I)), dict(q_out=Buf(3 * 4 * 64 + 1, B)),
    dict(q_out=Buf(3 * 4 * 64, F)), dict(k=Buf(3 * 2 * 64, B)), dict(k=Buf(3 * 2 * 64, F), v=Buf(3 * 2 * 64, F)),
    dict(k=Buf(3 * 2 * 64 - 1, B), v=Buf(3 * 2 * 64, B)), dict(rope=Buf(63, F)), dict(rope=Buf(640, B)),
    dict(q_gain=Buf(63, F)), dict(k_gain=Buf(64, B)), dict(starts=Buf(3, F)), dict(starts=Buf(0, I)),
    dict(past=Buf(1, I)), dict(past=Buf(2, F)), dict(k_out=Buf(3 * 2 * 64 - 1, B)), dict(v_out=Buf(3 * 2 * 64, F)),
    dict(table=None), dict(table=Buf(7, I)), dict(table=Buf(8, F)), dict(cache=None), dict(cache=cache(kv=4)),
    dict(cache=cache(dim=128)), dict(layer=2), dict(heads=0), dict(kv_heads=0)])
def test_prepare_method_refuses(kw):
    a = dict(q=Buf(3 * 8 * 64, B), heads=4, kv_heads=2, head_dim=64, rope=Buf(640, F), q_out=Buf(3 * 4 * 64, B),
             starts=Buf(3, I), past=Buf(2, I), cache=cache(), table=Buf(8, I))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        LoadedModule(None).prepare_qk(None, **a)


@pytest.mark.parametrize("kw", [
    dict(q=Buf(3 * 256 - 1, B)), dict(q=Buf(3 * 256, F)), dict(k=Buf(3 * 128 - 1, B)), dict(v=Buf(3 * 128 - 1, B)),
    dict(v=Buf(3 * 128, B), v_stride=136), dict(out=Buf(3 * 256 + 1, B)), dict(out=Buf(3 * 256, I)),
    dict(starts=Buf(3, F)), dict(starts=Buf(0, I)), dict(heads=0), dict(kv_heads=0)])
def test_prefill_method_refuses(kw):
    a = dict(q=Buf(3 * 256, B), k=Buf(3 * 128, B), v=Buf(3 * 128, B), heads=4, kv_heads=2, head_dim=64,
             out=Buf(3 * 256, B))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        LoadedModule(None).attention_prefill(None, **a)


@pytest.mark.parametrize("kw", [
    dict(q=Buf(3 * 256 - 1, B)), dict(q=Buf(3 * 256, F)), dict(lengths=Buf(2, I)), dict(lengths=Buf(3, F)),
    dict(table=Buf(8, I)), dict(table=Buf(2, I)), dict(table=Buf(9, F)), dict(table=None), dict(out=Buf(3 * 256 + 1, B)),
    dict(out=Buf(3 * 256, U)), dict(heads=3, q=Buf(3 * 192, B), out=Buf(3 * 192, B)), dict(heads=0), dict(layer=2)])
def test_decode_method_refuses(kw):
    a = dict(q=Buf(3 * 256, B), cache=cache(), lengths=Buf(3, I), table=Buf(9, I), heads=4, out=Buf(3 * 256, B))
    a.update(kw)
    mod = LoadedModule(None)
    mod._routed_workspace = lambda stream, size_of, *shape, **kw: (A, 1 << 40)
    with pytest.raises((ValueError, TypeError)):
        mod.attention_decode(None, **a)


def test_copy_method_refuses():
    for src, dst in ((Buf(3, F), Buf(3, I)), (Buf(3, I), Buf(3, F)), (Buf(3, I), Buf(2, I))):
        with pytest.raises((ValueError, TypeError)):
            LoadedModule(None).copy_pages(None, cache(), src, dst)


# ------------------------------------------------------------------ the pool
def test_pool_extends_forks_and_frees():
    p = PagePool(6)
    a = p.add()
    assert p.extend(a, 0) == [] and p.extend(a, 64) == [] and p.table([a]).tolist() == [[0]]
    assert p.extend(a, 1) == [] and p.length(a) == 65 and p.table([a], 4).tolist() == [[0, 1, -1, -1]]
    b = p.fork(a)
    assert p.length(b) == 65 and p.table([b]).tolist() == [[0, 1]] and p.free_pages == 4
    assert p.extend(b, 1) == [(1, 2)]             # the last page is shared and not full
    assert p.table([a, b]).tolist() == [[0, 1], [0, 2]]
    assert p.extend(a, 1) == []                   # now its own
    p.free(a)
    assert p.free_pages == 4 and len(p) == 1      # page 0 still serves b
    p.free(b)
    assert p.free_pages == 6
    with pytest.raises(KeyError):
        p.extend(a, 1)


def test_pool_shares_full_pages_without_a_copy():
    p = PagePool(4)
    a = p.add()
    p.extend(a, 128)
    b = p.fork(a)
    assert p.extend(b, 5) == [] and p.table([a, b]).tolist() == [[0, 1, -1], [0, 1, 2]]


def test_pool_refuses_and_stays_as_it_was():
    p = PagePool(2)
    a = p.add()
    p.extend(a, 100)
    b = p.fork(a)
    for seq, n, error in ((a, 60, MemoryError), (b, 1, MemoryError), (a, -1, ValueError)):
        with pytest.raises(error):
            p.extend(seq, n)
        assert p.free_pages == 0 and p.length(a) == p.length(b) == 100 and p.table([a, b]).tolist() == [[0, 1]] * 2
    with pytest.raises(ValueError):
        p.table([a], 1)
    with pytest.raises(ValueError):
        PagePool(0)


@pytest.mark.parametrize("seed", range(8))
def test_pool_against_a_plain_model(seed):
    """Random calls: every token of every sequence stays where its table says,
    no page in use is handed out, and compacting packs."""
    rng = np.random.default_rng(seed)
    p, memory, want, count = PagePool(40), np.full((40, 64), -1, np.int64), {}, 0
    for _ in range(400):
        act = rng.integers(0, 10)
        if act < 2 or not want:
            want[p.add()] = []
        elif act < 7:
            seq, n = int(rng.choice(list(want))), int(rng.integers(0, 150))
            try:
                pairs = p.extend(seq, n)
            except MemoryError:
                continue
            assert {a for a, _ in pairs}.isdisjoint(b for _, b in pairs)
            for a, b in pairs:
                memory[b] = memory[a]
            table = p.table([seq])[0]
            for i in range(n):
                t = len(want[seq])
                memory[table[t // 64], t % 64] = count
                want[seq].append(count)
                count += 1
        elif act == 7:
            seq = int(rng.choice(list(want)))
            want[p.fork(seq)] = list(want[seq])
        elif act == 8:
            seq = int(rng.choice(list(want)))
            p.free(seq)
            del want[seq]
        else:
            pairs = p.compact()
            assert {a for a, _ in pairs}.isdisjoint(b for _, b in pairs)
            for a, b in pairs:
                memory[b] = memory[a]
                memory[a] = -1
            used = {int(x) for s in want for x in p.table([s])[0] if x >= 0}
            assert used == set(range(len(used))) and p.free_pages == 40 - len(used)
        for seq, tokens in want.items():
            table = p.table([seq])[0]
            assert p.length(seq) == len(tokens)
            assert [memory[table[t // 64], t % 64] for t in range(len(tokens))] == tokens
