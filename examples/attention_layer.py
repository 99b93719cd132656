"""One decoder layer's first half over a paged 8-bit cache, on an MI355X:

  qkv  = the projection of RMSNorm(x), quantized             norm_quantize, linear
  q, k = head norms and rotations; k and v into the cache    prepare_qk
  attn = attention of whole prompts, or of one row of each   attention_prefill,
         sequence over the cache                             attention_decode
  x2   = x + o(attn)                                         quantize, linear_residual

Sequences come and go: a pool hands out the cache's pages, forked sequences
share their full ones, and copies (of a page that a fork still writes to, or
to close the gaps that ended sequences left) run on the device.  Run it for a
few prompts and some steps with random weights:

  python examples/attention_layer.py [sequences] [steps]
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from inferrous_amd import CudaContext, DeviceBuffer, Event, KvCache, PagePool, load  # noqa: E402

HIDDEN = 4096  # norm_quantize's width
HEADS, KV_HEADS, HEAD_DIM = 32, 8, 128
WIDTH, KV_WIDTH = HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM


def rotations(positions: int, theta: float = 1e6) -> np.ndarray:
    """float32 [positions, HEAD_DIM]: cosines, then sines."""
    a = np.arange(positions)[:, None] * theta ** (-np.arange(HEAD_DIM // 2) * 2.0 / HEAD_DIM)
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


class Weights:
    """Random weights of one layer: the projections and the norms' gains."""

    def __init__(self, stream, seed: int = 0):
        rng = np.random.default_rng(seed)

        def matrix(n, k):
            w = rng.integers(-127, 128, n * k, dtype=np.int8)
            return w, ((0.5 + rng.random(n)) / (73.0 * k ** 0.5)).astype(np.float32)

        def gain(n):
            return (1.0 + 0.1 * rng.standard_normal(n)).astype(np.float32)

        self.host = {"qkv": matrix(WIDTH + 2 * KV_WIDTH, HIDDEN), "o": matrix(HIDDEN, WIDTH), "gain": gain(HIDDEN),
                     "q_gain": gain(HEAD_DIM), "k_gain": gain(HEAD_DIM)}
        for name, a in self.host.items():
            setattr(self, name, tuple(DeviceBuffer.from_host(stream, t) for t in a) if isinstance(a, tuple)
                    else DeviceBuffer.from_host(stream, a))


class Rows:
    """Buffers of one batch of rows."""

    def __init__(self, rows: int):
        f32, i8, bf16 = (lambda n, t=t: DeviceBuffer(rows * n, t) for t in (np.float32, np.int8, np.uint16))
        self.rows = rows
        self.normed, self.n8, self.n_scales, self.maxima = f32(HIDDEN), i8(HIDDEN), f32(1), DeviceBuffer(rows, np.uint32)
        self.qkv = bf16(WIDTH + 2 * KV_WIDTH)
        self.q, self.k, self.v, self.attn = bf16(WIDTH), bf16(KV_WIDTH), bf16(KV_WIDTH), bf16(WIDTH)
        self.a8, self.a_scales = i8(WIDTH), f32(1)
        self.out, self.x2 = f32(HIDDEN), f32(HIDDEN)


class Layer:
    """The layer, its cache and the sequences in it."""

    def __init__(self, ctx, pages: int, positions: int):
        self.mod, self.stream = load(ctx), ctx.new_stream()
        self.weights = Weights(self.stream)
        self.cache, self.pool = KvCache(1, pages, KV_HEADS, HEAD_DIM), PagePool(pages)
        self.rope = self.put(rotations(positions), np.float32)

    def put(self, a, dtype=np.int32) -> DeviceBuffer:
        return DeviceBuffer.from_host(self.stream, np.asarray(a, dtype).reshape(-1))

    def copy(self, pairs) -> None:
        if pairs:
            src, dst = zip(*pairs)
            self.mod.copy_pages(self.stream, self.cache, self.put(src), self.put(dst))

    def run(self, b: Rows, x: DeviceBuffer, seqs, rows=None) -> DeviceBuffer:
        """x: float32 [rows * HIDDEN].  rows: how many each of ``seqs`` brings (new
        sequences' whole prompts); None for one more row of each."""
        mod, s, w = self.mod, self.stream, self.weights
        past = [self.pool.length(i) for i in seqs]
        for i, n in zip(seqs, rows or [1] * len(seqs)):
            self.copy(self.pool.extend(i, n))
        table = self.put(self.pool.table(seqs))
        starts = None if rows is None else self.put(np.concatenate([[0], np.cumsum(rows)]))
        mod.norm_quantize(s, None, x, w.gain, b.normed, b.n8, b.n_scales, b.maxima)
        mod.linear(s, None, b.n8, b.n_scales, *w.qkv, HIDDEN, b.qkv)
        mod.prepare_qk(s, b.qkv, HEADS, KV_HEADS, HEAD_DIM, self.rope, b.q, q_gain=w.q_gain, k_gain=w.k_gain,
                       starts=starts, past=self.put(past), k_out=b.k, v_out=b.v, cache=self.cache, table=table)
        if rows is None:
            mod.attention_decode(s, b.q, self.cache, self.put([n + 1 for n in past]), table, HEADS, b.attn)
        else:
            mod.attention_prefill(s, b.q, b.k, b.v, HEADS, KV_HEADS, HEAD_DIM, b.attn, starts=starts)
        mod.quantize(s, None, b.attn, WIDTH, b.a8, b.a_scales)
        mod.linear_residual(s, None, b.a8, b.a_scales, *w.o, WIDTH, x, b.out, b.x2)
        return b.x2


def main(sequences: int, steps: int) -> None:
    rng = np.random.default_rng(1)
    prompts = rng.integers(1, 600, sequences).tolist()
    layer = Layer(CudaContext(0), pages=sequences * ((600 + steps) // 64 + 2), positions=1024 + steps)
    rows = lambda n: layer.put(rng.standard_normal((n, HIDDEN)), np.float32)  # noqa: E731
    seqs = [layer.pool.add() for _ in prompts]
    layer.run(Rows(sum(prompts)), rows(sum(prompts)), seqs, prompts)
    b, x = Rows(sequences), rows(sequences)
    layer.run(b, x, seqs)
    first, last = Event(), Event()
    first.record(layer.stream)
    for _ in range(steps):
        layer.run(b, x, seqs)
    last.record(layer.stream)
    last.synchronize()
    out = b.x2.to_host_vec(layer.stream)
    print(f"{sequences} sequences of {min(prompts)} to {max(prompts)} tokens: "
          f"{1e3 * first.elapsed_ms(last) / max(1, steps):.1f} us a step with the host's part, "
          f"|x2| {np.abs(out).mean():.4f}, {layer.pool.pages - layer.pool.free_pages} pages in use")


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 4, int(sys.argv[2]) if len(sys.argv) > 2 else 20)
