"""One decoder layer's second half with routed weights, on an MI355X:

  x2 = residual + o(attn) + the request's adapter beside o   linear_adapters
  n  = RMSNorm(x2), quantized                                norm_quantize
  experts of each row from the router's logits               linear, route_experts
  x3 = x2 + the weighted sum of the experts' SwiGLU          experts_mlp

Rows may belong to different requests: each names its adapter (or none), and
each finds its own experts.  Run it for a small layer with random weights:

  python examples/routed_layer.py [rows]
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from inferrous_amd import CudaContext, DeviceBuffer, Event, load  # noqa: E402

HIDDEN = 4096  # norm_quantize's width


class Weights:
    """Random weights of one layer: o, its adapters, the router and the experts."""

    def __init__(self, stream, experts: int, inter: int, adapters: int, rank: int, seed: int = 0):
        rng = np.random.default_rng(seed)
        self.experts, self.inter, self.adapters, self.rank = experts, inter, adapters, rank

        def matrix(n, k, size=1.0):
            w = rng.integers(-127, 128, n * k, dtype=np.int8)
            return w, ((0.5 + rng.random(n)) * (size / (73.0 * k ** 0.5))).astype(np.float32)

        def bf16(a):
            return (np.ascontiguousarray(a, np.float32).view(np.uint32) >> 16).astype(np.uint16)

        self.host = {
            "o": matrix(HIDDEN, HIDDEN, 0.3), "router": matrix(experts, HIDDEN, 1.5),
            "gate": matrix(experts * inter, HIDDEN), "up": matrix(experts * inter, HIDDEN),
            "down": matrix(experts * HIDDEN, inter, 0.5),
            "a": bf16(rng.standard_normal((adapters, rank, HIDDEN)) * HIDDEN ** -0.5).reshape(-1),
            "b": bf16(rng.standard_normal((adapters, HIDDEN, rank)) * 0.1).reshape(-1),
            "scaling": (1.0 + rng.random(adapters)).astype(np.float32),
            "gain": (1.0 + 0.1 * rng.standard_normal(HIDDEN)).astype(np.float32),
        }
        for name, a in self.host.items():
            setattr(self, name, tuple(DeviceBuffer.from_host(stream, t) for t in a) if isinstance(a, tuple)
                    else DeviceBuffer.from_host(stream, a))


class Rows:
    """Buffers of one batch of rows."""

    def __init__(self, rows: int, top_k: int, experts: int):
        f32 = lambda n: DeviceBuffer(n, np.float32)  # noqa: E731
        n = rows * HIDDEN
        self.rows = rows
        self.q_attn, self.s_attn, self.x2 = DeviceBuffer(n, np.int8), f32(rows), f32(n)
        self.normed, self.q, self.s, self.maxima = f32(n), DeviceBuffer(n, np.int8), f32(rows), \
            DeviceBuffer(rows, np.uint32)
        self.logits = f32(rows * experts)
        self.ids, self.weights = DeviceBuffer(rows * top_k, np.int32), f32(rows * top_k)
        self.x3 = f32(n)


def layer(mod, stream, w: Weights, b: Rows, attn, residual, adapter_ids) -> DeviceBuffer:
    """attn and residual: float32 [rows * HIDDEN]; adapter_ids: int32 [rows], -1 for none."""
    mod.quantize(stream, None, attn, HIDDEN, b.q_attn, b.s_attn)
    mod.linear_adapters(stream, b.q_attn, b.s_attn, *w.o, HIDDEN, attn, adapter_ids, w.a, w.b, w.scaling, b.x2,
                        residual=residual)
    mod.norm_quantize(stream, None, b.x2, w.gain, b.normed, b.q, b.s, b.maxima)
    mod.linear(stream, None, b.q, b.s, *w.router, HIDDEN, b.logits)
    mod.route_experts(stream, b.logits, w.experts, b.ids, b.weights)
    mod.experts_mlp(stream, b.q, b.s, HIDDEN, b.ids, b.weights, *w.gate, *w.up, *w.down, w.experts, b.x3,
                    residual=b.x2)
    return b.x3


def main(rows: int) -> None:
    ctx = CudaContext(0)
    mod, stream = load(ctx), ctx.new_stream()
    w = Weights(stream, experts=32, inter=512, adapters=4, rank=16)
    b = Rows(rows, top_k=4, experts=w.experts)
    rng = np.random.default_rng(1)
    attn, residual = (DeviceBuffer.from_host(stream, rng.standard_normal(rows * HIDDEN).astype(np.float32))
                      for _ in range(2))
    ids = DeviceBuffer.from_host(stream, rng.integers(-1, 4, rows).astype(np.int32))
    x3 = layer(mod, stream, w, b, attn, residual, ids)
    first, last = Event(), Event()
    first.record(stream)
    for _ in range(20):
        layer(mod, stream, w, b, attn, residual, ids)
    last.record(stream)
    last.synchronize()
    out = x3.to_host_vec(stream)
    print(f"{rows} rows: {1e3 * first.elapsed_ms(last) / 20:.1f} us a pass, |x3| {np.abs(out).mean():.4f}, "
          f"experts of row 0: {b.ids.to_host_vec(stream)[:4].tolist()}")


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 8)
