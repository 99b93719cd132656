"""The example layer (examples/attention_layer.py): prompts, forks, steps, ended
sequences and compaction, every operator's output against its 64-bit form on the
operator's own inputs (tolerances: test_gpu_attention.py)."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import numpy as np
import pytest

from inferrous_amd import CudaContext
from test_gpu_attention import E4M3, PAGE, close, from_bits, softmax_sums

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "attention_layer", Path(__file__).resolve().parent.parent / "examples" / "attention_layer.py")
al = importlib.util.module_from_spec(spec)
spec.loader.exec_module(al)
GROUP = al.HEADS // al.KV_HEADS


class Checked:
    """The layer beside what its operators should have left."""

    def __init__(self, pages, positions):
        self.layer = al.Layer(CudaContext(0), pages, positions)
        self.rope = al.rotations(positions).astype(np.float64)
        self.tokens = {}   # of each sequence, its keys and values as prepare_qk took them
        self.rng = np.random.default_rng(0)

    def rotate(self, x, gain, positions):
        x = x / np.sqrt((x ** 2).mean(2, keepdims=True) + 1e-6) * gain.astype(np.float64)
        h = al.HEAD_DIM // 2
        c, s, a, b = self.rope[positions, None, :h], self.rope[positions, None, h:], x[..., :h], x[..., h:]
        return (np.concatenate([a * c - b * s, b * c + a * s], 2),
                np.concatenate([abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)], 2))

    def run(self, seqs, rows=None):
        layer = self.layer
        past = [layer.pool.length(i) for i in seqs]
        counts = rows or [1] * len(seqs)
        m = sum(counts)
        b, x = al.Rows(m), self.rng.standard_normal((m, al.HIDDEN)).astype(np.float32)
        layer.run(b, layer.put(x, np.float32), seqs, rows)
        host = lambda name: getattr(b, name).to_host_vec(layer.stream)  # noqa: E731
        heads = lambda name: from_bits(host(name)).reshape(m, -1, al.HEAD_DIM)  # noqa: E731

        w = layer.weights.host
        qkv = heads("qkv").astype(np.float64)
        positions = np.concatenate([p + np.arange(n) for p, n in zip(past, counts)])
        want, size = self.rotate(qkv[:, :al.HEADS], w["q_gain"], positions)
        close(heads("q"), want, 2.0 ** -19 * size)
        key, size = self.rotate(qkv[:, al.HEADS:al.HEADS + al.KV_HEADS], w["k_gain"], positions)
        close(heads("k"), key, 2.0 ** -19 * size)
        assert np.array_equal(heads("v"), qkv[:, al.HEADS + al.KV_HEADS:])

        q, attn = heads("q").astype(np.float64), heads("attn")
        starts = np.concatenate([[0], np.cumsum(counts)])
        for i, lo, hi in zip(seqs, starts, starts[1:]):
            for which, z in enumerate((key, qkv[:, al.HEADS + al.KV_HEADS:])):
                old = self.tokens.get(i, [None, None])[which]
                new = z[lo:hi] if old is None else np.concatenate([old, z[lo:hi]])
                self.tokens[i] = [new, *self.tokens.get(i, [None, None])[1:]] if which == 0 else [self.tokens[i][0], new]
        cached = self.check_cache(seqs)
        for i, lo, hi in zip(seqs, starts, starts[1:]):
            if rows is None:
                k, v = cached[i]
            else:
                k, v = heads("k")[lo:hi].astype(np.float64), heads("v")[lo:hi].astype(np.float64)
            for h in range(al.HEADS):
                s = q[lo:hi, h] @ k[:, h // GROUP].T * al.HEAD_DIM ** -0.5
                if rows is not None:
                    s[np.triu(np.ones(s.shape, bool), 1)] = -np.inf
                o, size = softmax_sums(s, v[:, h // GROUP])
                close(attn[lo:hi, h], o, (2.0 ** -7 + 2.0 ** -9) * size)

        # o's exact integer sums; out is rounded once, and so is the sum with x
        sums = (host("a8").reshape(m, -1).astype(np.float64) @ w["o"][0].reshape(al.HIDDEN, -1).astype(np.float64).T)
        out = sums * host("a_scales")[:, None].astype(np.float64) * w["o"][1].astype(np.float64)
        close(host("x2").reshape(m, -1), x + out, (2.0 ** -8 + 2.0 ** -20) * abs(out))

    def check_cache(self, seqs):
        """Every token of every sequence, where the pool says it is: within half
        a step of e4m3, and another half for each time that its page's scale grew."""
        layer = self.layer
        c = layer.cache.codes.to_host_vec(layer.stream).reshape(layer.cache.pages, al.KV_HEADS, 2, -1)
        scales = layer.cache.scales.to_host_vec(layer.stream).reshape(layer.cache.pages, al.KV_HEADS, 2)
        both = (c[:, :, 0].reshape(-1, al.KV_HEADS, PAGE, al.HEAD_DIM),
                c[:, :, 1].reshape(-1, al.KV_HEADS, al.HEAD_DIM, PAGE).transpose(0, 1, 3, 2))
        found = {}
        for i, want in self.tokens.items():
            n = layer.pool.length(i)
            assert len(want[0]) == n
            t = np.arange(n)
            page = layer.pool.table([i])[0][t // PAGE]
            found[i] = []
            for which in (0, 1):
                step = scales[page, :, which].astype(np.float64)[:, :, None]
                got = E4M3[both[which][page, :, t % PAGE]] * step
                # a code in e4m3's normal range stays exact when the scale grows; one that
                # falls below is off by half a step of the subnormals each time, 2 in all
                bound = np.maximum(2.0 ** -4 * abs(want[which]), 2.0 ** -10 * step) + 2.0 ** -9 * step
                assert np.all(abs(got - want[which]) <= bound)
                found[i].append(got)
        return found


def test_sequences_come_and_go():
    c = Checked(pages=24, positions=400)
    pool = c.layer.pool
    seqs = [pool.add() for _ in range(3)]
    c.run(seqs, [5, 130, 200])
    fork = pool.fork(seqs[1])                 # two full pages shared, the third copied at the next step
    c.tokens[fork] = list(c.tokens[seqs[1]])
    for _ in range(2):
        c.run([seqs[2], fork, seqs[0], seqs[1]])
    pool.free(seqs[1])
    del c.tokens[seqs[1]]
    late = pool.add()
    c.run([late], [64])
    pool.free(seqs[0])
    del c.tokens[seqs[0]]
    c.layer.copy(pool.compact())
    c.check_cache([])
    for _ in range(2):
        c.run([fork, late, seqs[2]])


def test_one_sequence_step_by_step():
    """Across the end of a page."""
    c = Checked(pages=4, positions=100)
    seq = c.layer.pool.add()
    c.run([seq], [62])
    for _ in range(4):
        c.run([seq])
