"""The routed layers' host-side checks (no GPU): malformed arguments are
refused with the documented status before any HIP call, and the Python
methods refuse wrong lengths and types."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from inferrous_amd import _lib
from inferrous_amd.module import LoadedModule

A = 0x10000  # aligned fake addresses: validation never dereferences them


def no_device():
    c = ctypes.c_int()
    _lib.lib().w8a8_device_count(ctypes.byref(c))
    return c.value == 0


WELL = _lib.EINIT  # a well-formed call stops at the init check
pytestmark = pytest.mark.skipif(not no_device(), reason="well-formed calls on fake addresses: without a GPU only")


def route(**kw):
    a = dict(logits=A, dt=_lib.OUT_F32, m=3, e=64, score=0, bias=None, groups=1, top_groups=1, group_top=1, k=8,
             renorm=1, scale=1.0, ids=A, w=A)
    a.update(kw)
    return _lib.lib().w8a8_route_experts(None, a["logits"], a["dt"], a["m"], a["e"], a["score"], a["bias"],
                                         a["groups"], a["top_groups"], a["group_top"], a["k"], a["renorm"],
                                         a["scale"], a["ids"], a["w"])


@pytest.mark.parametrize("kw, status", [
    (dict(), WELL), (dict(dt=_lib.OUT_BF16), WELL), (dict(m=0, logits=None), _lib.OK),
    (dict(dt=_lib.OUT_I32), _lib.EARG), (dict(score=2), _lib.EARG), (dict(group_top=0), _lib.EARG),
    (dict(group_top=3), _lib.EARG), (dict(e=0), _lib.ESHAPE), (dict(e=1025), _lib.ESHAPE),
    (dict(groups=0), _lib.ESHAPE), (dict(groups=3), _lib.ESHAPE), (dict(groups=8, top_groups=9), _lib.ESHAPE),
    (dict(groups=8, top_groups=0), _lib.ESHAPE), (dict(groups=16, top_groups=1, k=5), _lib.ESHAPE),
    (dict(e=1024, groups=128, top_groups=64), _lib.ESHAPE), (dict(k=0), _lib.ESHAPE), (dict(k=65), _lib.ESHAPE),
    (dict(m=1 << 40), _lib.ESHAPE), (dict(logits=None), _lib.ENULL), (dict(ids=None), _lib.ENULL),
    (dict(w=None), _lib.ENULL), (dict(logits=A + 2), _lib.EALIGN), (dict(logits=A + 2, dt=_lib.OUT_BF16), WELL),
    (dict(bias=A + 1), _lib.EALIGN), (dict(ids=A + 2), _lib.EALIGN)])
def test_route_experts(kw, status):
    assert route(**kw) == status


def experts(**kw):
    a = dict(q=A, asc=A, m=3, h=64, ids=A, w=A, k=2, e=8, wg=A, sg=A, wu=A, su=A, wd=A, sd=A, i=48, res=None, out=A,
             dt=_lib.OUT_BF16, ws=A, short=0)
    a.update(kw)
    need = _lib.lib().w8a8_experts_mlp_workspace_bytes(a["m"], a["k"], a["e"], a["h"], a["i"])
    return _lib.lib().w8a8_experts_mlp(None, a["q"], a["asc"], a["m"], a["h"], a["ids"], a["w"], a["k"], a["e"],
                                       a["wg"], a["sg"], a["wu"], a["su"], a["wd"], a["sd"], a["i"], a["res"],
                                       a["out"], a["dt"], a["ws"], need - a["short"])


@pytest.mark.parametrize("kw, status", [
    (dict(), WELL), (dict(dt=_lib.OUT_F32, res=A), WELL), (dict(m=0, q=None), _lib.OK),
    (dict(dt=_lib.OUT_I32), _lib.EARG), (dict(h=72), _lib.ESHAPE), (dict(i=8), _lib.ESHAPE), (dict(h=0), _lib.ESHAPE),
    (dict(i=0), _lib.ESHAPE), (dict(e=0), _lib.ESHAPE), (dict(e=1025), _lib.ESHAPE), (dict(k=0), _lib.ESHAPE),
    (dict(k=65), _lib.ESHAPE), (dict(m=1 << 24), _lib.ESHAPE), (dict(h=65552), _lib.ESHAPE),
    *[({n: None}, _lib.ENULL) for n in ("q", "asc", "ids", "w", "wg", "sg", "wu", "su", "wd", "sd", "out")],
    *[({n: A + 8}, _lib.EALIGN) for n in ("q", "wg", "wu", "wd", "ws", "res", "out")],
    *[({n: A + 2}, _lib.EALIGN) for n in ("asc", "ids", "w", "sg", "su", "sd")],
    (dict(ws=None), _lib.EWORKSPACE), (dict(short=1), _lib.EWORKSPACE)])
def test_experts_mlp(kw, status):
    assert experts(**kw) == status


def adapters(**kw):
    a = dict(q=A, asc=A, m=3, w=A, ws=A, n=33, k=64, x=A, xt=_lib.OUT_F32, ids=A, a=A, b=A, s=A, r=16, c=4, res=None,
             out=A, dt=_lib.OUT_BF16, wsp=A, short=0)
    a.update(kw)
    need = _lib.lib().w8a8_linear_adapters_workspace_bytes(a["m"], a["n"], a["k"], a["r"], a["c"])
    return _lib.lib().w8a8_linear_adapters(None, a["q"], a["asc"], a["m"], a["w"], a["ws"], a["n"], a["k"], a["x"],
                                           a["xt"], a["ids"], a["a"], a["b"], a["s"], a["r"], a["c"], a["res"],
                                           a["out"], a["dt"], a["wsp"], need - a["short"])


@pytest.mark.parametrize("kw, status", [
    (dict(), WELL), (dict(xt=_lib.OUT_BF16, res=A, dt=_lib.OUT_F32), WELL), (dict(m=0, q=None), _lib.OK),
    (dict(n=0, w=None), _lib.OK), (dict(dt=_lib.OUT_I32), _lib.EARG), (dict(xt=_lib.OUT_I32), _lib.EARG),
    (dict(k=72), _lib.ESHAPE), (dict(k=0), _lib.ESHAPE), (dict(r=0), _lib.ESHAPE), (dict(r=12), _lib.ESHAPE),
    (dict(r=264), _lib.ESHAPE), (dict(m=(1 << 21) + 1), _lib.ESHAPE), (dict(n=(1 << 22) + 1), _lib.ESHAPE),
    (dict(c=1023), WELL), (dict(c=1024), _lib.ESHAPE), (dict(c=0), _lib.ESHAPE), (dict(c=65537), _lib.ESHAPE),
    *[({n: None}, _lib.ENULL) for n in ("q", "asc", "w", "ws", "x", "ids", "a", "b", "s", "out")],
    *[({n: A + 8}, _lib.EALIGN) for n in ("q", "w", "x", "a", "b", "wsp")],
    *[({n: A + 2}, _lib.EALIGN) for n in ("asc", "ws", "ids", "s", "res")],
    (dict(wsp=None), _lib.EWORKSPACE), (dict(short=1), _lib.EWORKSPACE)])
def test_linear_adapters(kw, status):
    assert adapters(**kw) == status


class Buf:
    def __init__(self, n, dtype):
        self.n, self.dtype, self.ptr = n, np.dtype(dtype), A
        self.nbytes = n * self.dtype.itemsize

    def __len__(self):
        return self.n


F, B, I, C = np.float32, np.uint16, np.int32, np.int8


@pytest.mark.parametrize("kw", [
    dict(logits=Buf(65, F)), dict(n_experts=0), dict(ids=Buf(7, I)), dict(ids=Buf(6, F)), dict(weights=Buf(6, I)),
    dict(weights=Buf(4, F)), dict(logits=Buf(64, C)), dict(score="relu"), dict(bias=Buf(31, F)), dict(bias=Buf(32, I)),
    dict(ids=Buf(0, I), weights=Buf(0, F))])
def test_route_method_refuses(kw):
    a = dict(logits=Buf(64, F), n_experts=32, ids=Buf(6, I), weights=Buf(6, F))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        LoadedModule(None).route_experts(None, **a)


@pytest.mark.parametrize("kw", [
    dict(q=Buf(191, C)), dict(q=Buf(192, F)), dict(asc=Buf(4, F)), dict(ids=Buf(5, I)), dict(ids=Buf(6, F)),
    dict(s0=Buf(385, F)), dict(s1=Buf(383, F)), dict(w0=Buf(8 * 48 * 64 - 1, C)), dict(wd=Buf(8, C)),
    dict(sd=Buf(511, F)), dict(out=Buf(191, B)), dict(out=Buf(192, C)), dict(residual=Buf(192, B)),
    dict(residual=Buf(1, F)), dict(n_experts=0)])
def test_experts_method_refuses(kw):
    a = dict(q=Buf(192, C), asc=Buf(3, F), width=64, ids=Buf(6, I), weights=Buf(6, F), w0=Buf(8 * 48 * 64, C),
             s0=Buf(8 * 48, F), w1=Buf(8 * 48 * 64, C), s1=Buf(8 * 48, F), wd=Buf(8 * 48 * 64, C), sd=Buf(512, F),
             n_experts=8, out=Buf(192, B))
    a.update(kw)
    mod = LoadedModule(None)
    mod._routed_workspace = lambda stream, size_of, *shape: (A, 1 << 40)
    with pytest.raises((ValueError, TypeError)):
        mod.experts_mlp(None, **a)


@pytest.mark.parametrize("kw", [
    dict(a=Buf(4 * 16 * 64 - 1, B)), dict(a=Buf(4 * 16 * 64, F)), dict(b=Buf(4 * 33 * 16 - 1, B)),
    dict(ids=Buf(2, I)), dict(ids=Buf(3, F)), dict(x=Buf(191, F)), dict(x=Buf(192, C)), dict(scaling=Buf(0, F)),
    dict(scaling=Buf(4, B)), dict(out=Buf(98, B)), dict(residual=Buf(98, F)), dict(residual=Buf(99, B)),
    dict(w=Buf(33 * 64 - 1, C)), dict(q=Buf(191, C))])
def test_adapters_method_refuses(kw):
    a = dict(q=Buf(192, C), asc=Buf(3, F), w=Buf(33 * 64, C), ws=Buf(33, F), width=64, x=Buf(192, F), ids=Buf(3, I),
             a=Buf(4 * 16 * 64, B), b=Buf(4 * 33 * 16, B), scaling=Buf(4, F), out=Buf(99, B))
    a.update(kw)
    mod = LoadedModule(None)
    mod._routed_workspace = lambda stream, size_of, *shape: (A, 1 << 40)
    with pytest.raises((ValueError, TypeError)):
        mod.linear_adapters(None, **a)
