"""The page pool where sequences get shorter (draft tokens that were not taken), and
what copies may be made together (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import PagePool


def test_pool_shortens():
    p = PagePool(5)
    a = p.add()
    p.extend(a, 200)
    p.shorten(a, 200)
    assert p.length(a) == 200 and p.free_pages == 1
    p.shorten(a, 193)
    assert p.length(a) == 193 and p.table([a]).tolist() == [[0, 1, 2, 3]]
    p.shorten(a, 192)
    assert p.free_pages == 2 and p.table([a]).tolist() == [[0, 1, 2]]
    assert p.extend(a, 1) == [] and p.length(a) == 193
    p.shorten(a, 0)
    assert p.free_pages == 5 and p.length(a) == 0 and p.table([a]).tolist() == [[-1]] and len(p) == 1
    assert p.extend(a, 65) == [] and p.length(a) == 65


def test_a_full_page_that_a_shortened_sequence_writes_to_again_is_copied():
    p = PagePool(6)
    a = p.add()
    p.extend(a, 128)
    b = p.fork(a)
    p.shorten(b, 100)                     # within the second page, which a still has in full
    assert p.extend(b, 3) == [(1, 2)] and p.table([a, b]).tolist() == [[0, 1], [0, 2]]
    c = p.fork(a)
    p.shorten(c, 64)
    assert p.extend(c, 1) == [] and p.table([c]).tolist() == [[0, 3]]
    p.shorten(a, 70)
    assert p.extend(a, 1) == []           # c does not have the page any more, b has its own


def test_pool_refuses_to_shorten_and_stays_as_it_was():
    p = PagePool(3)
    a = p.add()
    p.extend(a, 100)
    for n in (-1, 101):
        with pytest.raises(ValueError):
            p.shorten(a, n)
    with pytest.raises(KeyError):
        p.shorten(a + 1, 0)
    assert p.length(a) == 100 and p.free_pages == 1


@pytest.mark.parametrize("seed", range(8))
def test_pool_against_a_plain_model(seed):
    """Random calls, the copies of a few calls of extend made together: every token of
    every sequence stays where its table says."""
    rng = np.random.default_rng(seed)
    p, memory, want, count, pending = PagePool(40), np.full((40, 64), -1, np.int64), {}, 0, []

    def write():
        """The gathered copies at once, then the rows that their calls made room for."""
        pairs, rows = [x for pairs, _, _ in pending for x in pairs], [(s, n) for _, s, n in pending]
        pending.clear()
        to = [b for _, b in pairs]
        assert len(set(to)) == len(to) and {a for a, _ in pairs}.isdisjoint(to)
        held = memory.copy()
        for a, b in pairs:
            memory[b] = held[a]
        nonlocal count
        for seq, n in rows:
            table = p.table([seq])[0]
            for i in range(n):
                t = len(want[seq])
                memory[table[t // 64], t % 64] = count
                want[seq].append(count)
                count += 1

    for _ in range(600):
        act = rng.integers(0, 12)
        if act >= 7:
            write()
        if act < 7 and want:
            seq, n = int(rng.choice(list(want))), int(rng.integers(0, 100))
            try:
                pending.append((p.extend(seq, n), seq, n))
            except MemoryError:
                pass
            continue
        if act == 7 or not want:
            want[p.add()] = []
        elif act == 8:
            seq = int(rng.choice(list(want)))
            want[p.fork(seq)] = list(want[seq])
        elif act == 9:
            seq = int(rng.choice(list(want)))
            p.free(seq)
            del want[seq]
        elif act == 10:
            seq = int(rng.choice(list(want)))
            n = int(rng.integers(0, len(want[seq]) + 1))
            p.shorten(seq, n)
            del want[seq][n:]
        else:
            pairs = p.compact()
            for a, b in pairs:
                memory[b] = memory[a]
                memory[a] = -1
        used = {int(x) for s in want for x in p.table([s])[0] if x >= 0}
        assert p.free_pages == 40 - len(used)
        for seq, tokens in want.items():
            table = p.table([seq])[0]
            assert p.length(seq) == len(tokens) and len(table) >= -(-len(tokens) // 64)
            assert [memory[table[t // 64], t % 64] for t in range(len(tokens))] == tokens
