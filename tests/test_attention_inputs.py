"""The inputs that attention is tested with show mistakes (no GPU): the
64-bit form with a mistake planted in it is outside the tolerance of the one without."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_attention import PAGE, close
from test_gpu_attention_peaked import CASES, PROMPTS, Peaked, Spread

MISTAKES = {
    "one key scale": lambda c: dict(key_scale=c.cache.s[c.table[0, 0], 0, 0]),
    "one value scale": lambda c: dict(value_scale=c.cache.s[c.table[0, 0], 0, 1]),
    "key scales for values": lambda c: dict(value_scale=c.cache.s[c.table[0, 0], 0, 0]),
    "half of the columns": lambda c: dict(columns=c.dim // 2),
    "all but four columns": lambda c: dict(columns=c.dim - 4),
    "a wave's pages": lambda c: dict(without=lambda page: page % 4 == 3),
    "the last page": lambda c: dict(without=lambda page: page == (max(c.lengths) - 1) // PAGE),
    "one page within": lambda c: dict(without=lambda page: page == 5),
}


@pytest.mark.parametrize("heads, kv, dim, lengths", CASES)
def test_mistakes_show(heads, kv, dim, lengths):
    c = Peaked(heads, kv, dim, lengths)
    want, err = c.want()
    rounded = want.astype(np.float32)
    close(rounded, want, err)
    assert np.abs(err).max() < 2.0 ** -9 * np.abs(want).max()
    missed = []
    for name, plant in MISTAKES.items():
        wrong = c.want(**plant(c))[0]
        # outside the tolerance in all rows of more than a few pages, not in one place by chance
        for row, n in enumerate(lengths):
            if n > 6 * PAGE and (name != "the last page" or n == max(lengths)):
                try:
                    close(wrong[row].astype(np.float32), want[row], err[row])
                    missed.append((name, n))
                except AssertionError:
                    pass
    assert not missed


WRONG = {
    "half of the columns": lambda c: dict(columns=c.dim // 2),
    "all but 16 columns": lambda c: dict(columns=c.dim - 16),
    "every other 32 keys": lambda c: dict(without=lambda key: key // 32 % 2 == 1),
    "the first 32 keys": lambda c: dict(without=lambda key: key < 32),
    "another head's keys": lambda c: dict(heads_on=1),
    "other columns' values": lambda c: dict(values_on=32),
}


@pytest.mark.parametrize("heads, kv, dim, rows", PROMPTS)
def test_mistakes_in_prompts_show(heads, kv, dim, rows):
    c = Spread(heads, kv, dim, rows)
    want, err = c.want()
    close(want.astype(np.float32), want, err)
    missed = []
    for name, plant in WRONG.items():
        if name == "another head's keys" and kv == 1:
            continue
        wrong = c.want(**plant(c))[0]
        for lo, hi in zip(c.starts, c.starts[1:]):
            for part in (slice(lo + 256, lo + 512), slice(hi - 200, hi)):   # rows that are done without a mask, mostly
                if hi - lo > 500:
                    try:
                        close(wrong[part].astype(np.float32), want[part], err[part])
                        missed.append((name, hi - lo))
                    except AssertionError:
                        pass
    assert not missed
