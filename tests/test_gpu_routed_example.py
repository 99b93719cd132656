"""The example layer (examples/routed_layer.py): every step's output against its
64-bit form on the step's own inputs, from one row to a prompt."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import numpy as np
import pytest

from inferrous_amd import CudaContext, load
from test_gpu_routed import Adapters, Experts, close_bf16, dev, from_bits, route_oracle

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "routed_layer", Path(__file__).resolve().parent.parent / "examples" / "routed_layer.py")
routed_layer = importlib.util.module_from_spec(spec)
spec.loader.exec_module(routed_layer)


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    mod, s = load(ctx), ctx.new_stream()
    return mod, s, routed_layer.Weights(s, experts=12, inter=208, adapters=3, rank=16)


@pytest.mark.parametrize("rows", [1, 6, 70])
def test_layer(env, rows):
    mod, s, w = env
    h, k = routed_layer.HIDDEN, 3
    rng = np.random.default_rng(rows)
    attn = (rng.standard_normal((rows, h)).astype(np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32)
    res = rng.standard_normal((rows, h)).astype(np.float32)
    ids = rng.integers(-1, 3, rows).astype(np.int32)
    b = routed_layer.Rows(rows, k, w.experts)
    routed_layer.layer(mod, s, w, b, dev(s, attn.reshape(-1)), dev(s, res.reshape(-1)), dev(s, ids))
    host = lambda name, *shape: getattr(b, name).to_host_vec(s).reshape(shape)  # noqa: E731

    c = Adapters.__new__(Adapters)
    c.m, c.n, c.k, c.rank, c.count = rows, h, h, w.rank, w.adapters
    c.x, c.q, c.asc, c.ids, c.residual = attn, host("q_attn", rows, h), host("s_attn", rows), ids, res
    c.w, c.ws = w.host["o"][0].reshape(h, h), w.host["o"][1]
    c.a = from_bits(w.host["a"]).reshape(w.adapters, w.rank, h)
    c.b = from_bits(w.host["b"]).reshape(w.adapters, h, w.rank)
    c.scaling = w.host["scaling"]
    close_bf16(host("x2", rows, h), *c.want())

    want, weights, near = route_oracle(host("logits", rows, w.experts), k, "softmax", None, 1, 1, 1, True, 1.0)
    assert np.array_equal(host("ids", rows, k)[~near], want[~near])
    assert np.all(np.abs(host("weights", rows, k) - weights)[~near] <= 2.0 ** -19)

    e = Experts.__new__(Experts)
    e.m, e.k, e.e, e.h, e.f = rows, k, w.experts, h, w.inter
    e.q, e.asc, e.ids, e.weights = host("q", rows, h), host("s", rows), host("ids", rows, k), host("weights", rows, k)
    e.wg, e.wu = (w.host[n][0].reshape(e.e, e.f, h) for n in ("gate", "up"))
    e.sg, e.su = (w.host[n][1].reshape(e.e, e.f) for n in ("gate", "up"))
    e.wd, e.sd = w.host["down"][0].reshape(e.e, h, e.f), w.host["down"][1].reshape(e.e, h)
    e.residual = host("x2", rows, h)
    close_bf16(host("x3", rows, h), *e.want())
