"""The pages of a decoder's slots (``PagedSlots``) without a GPU: which slot holds which page.  A cache without layers keeps its tables
and lengths on the CPU."""
import random

import pytest
import torch

from metaseq_amd import PagedSlots


def _slots(slots, capacity, pages, page=16, window=0, sinks=0):
    return PagedSlots(0, slots, capacity, 1, 64, pages, page, torch.float16, window, sinks, "cpu")


def _grow(c, wanted):
    c.reserve(wanted)
    for s, pos, n in wanted:
        c.holds(s, pos + n)
        c.lens[s] = pos + n


def _reserve_a_step(c, growing):
    def those(takes_part):
        return [(s, n, 1) for s, n in enumerate(c.host_lens) if 0 <= n < c.capacity and s in takes_part]

    for s, n, _ in c.reserve(those(range(c.batch)), lambda: those(growing)):
        c.host_lens[s] = n + 1
        c.stale.add(s)


def _step(c, growing):
    """What a decode step does that ``growing`` slots take part in: the host counts all, the device those."""
    _reserve_a_step(c, growing)
    for s in growing:
        page = int(c.table[s, int(c.lens[s]) // c.page])
        assert page >= 0 and c.refs[page] == 1 and page in c.host_table[s]
        c.lens[s] += 1


def _sound(c):
    held = [int(p) for p in c.host_table.view(-1) if p >= 0]
    for p, refs in enumerate(c.refs):
        assert held.count(p) == refs and (p in c.free) == (refs == 0)
    assert len(set(c.free)) == len(c.free)


def test_a_paused_slot_takes_no_pages():
    """Three slots in a pool for what they hold: one sits out while the others fill theirs."""
    c = _slots(3, 160, 1 + 2 * 10)
    _grow(c, [(0, 0, 10), (1, 0, 20), (2, 0, 20)])
    for _ in range(140):
        _step(c, [1, 2])
        _sound(c)
    c.exact_lens([0])
    assert c.host_lens == [10, 160, 160]
    with pytest.raises(ValueError, match="pages are needed"):
        c.reserve([(0, 10, 7)])
    _sound(c)


def test_steps_give_back_what_a_window_has_passed():
    c = _slots(2, 2000, 2 * 5, window=40, sinks=5)
    _grow(c, [(0, 0, 30), (1, 0, 1)])
    for i in range(900):
        _step(c, [0, 1])
        _sound(c)
        for s in (0, 1):
            n = int(c.lens[s])
            assert all(int(c.host_table[s, j // 16]) >= 0 for j in range(n) if j > n - 40 or j < 5), (i, s)
    assert c.lens.tolist() == [930, 901]


def test_pages_of_a_call_that_failed_come_back():
    c = _slots(2, 100, 7)
    c.reserve([(0, 0, 64)])                 # (and the pass behind it did not run)
    _grow(c, [(1, 0, 90)])
    _sound(c)
    assert c.host_lens == [-1, 90] and c.free and int((c.host_table[0] >= 0).sum()) == 0


def test_steps_past_the_capacity_leave_the_tables_alone():
    c = _slots(1, 32, 2, window=5)
    _grow(c, [(0, 0, 32)])
    c.lens[0] = 500
    c.stale.add(0)
    c.reclaim()
    _sound(c)


def test_copies_of_what_a_slot_does_not_hold_are_refused():
    """More positions than it has; fewer, whose window reaches back to pages that are given back."""
    c = _slots(3, 200, 30, window=40, sinks=5)
    _grow(c, [(0, 0, 50)])
    with pytest.raises(ValueError, match="holds no 51"):
        c.copy_row(0, 1, 51)
    with pytest.raises(ValueError, match="holds no 1"):
        c.copy_row(2, 1, 1)
    c.copy_row(0, 1, 20)
    c.lens[1] = 20
    for at in range(50, 150, 10):
        _grow(c, [(0, at, 10)])
    # 150: the next position sees 111 .. 149, blocks 1 .. 5 are gone; 135 would see 96, 134 95
    assert [b for b in range(10) if int(c.host_table[0, b]) < 0] == [1, 2, 3, 4, 5]
    for n in (134, 100, 60, 20):
        with pytest.raises(ValueError, match="given back"):
            c.copy_row(0, 2, n)
    assert c.host_lens == [150, 20, -1]
    for n in (150, 149, 135, 16, 3):
        c.copy_row(0, 2, n)
        assert c.host_lens[2] == n
        _sound(c)


def test_a_short_copy_gives_back_its_own_pages():
    """A copy of fewer positions than the source's window has passed: what it grows by comes back like any slot's."""
    c = _slots(2, 200, 12, window=40, sinks=5)
    for at in range(0, 150, 10):
        _grow(c, [(0, at, 10)])
    c.copy_row(0, 1, 16)
    c.lens[1] = 16
    c.release_row(0)
    for at in range(16, 196, 10):
        _grow(c, [(1, at, 10)])
        _sound(c)
        assert int((c.host_table[1] >= 0).sum()) <= 1 + 4, at


@pytest.mark.parametrize("window", [0, 24])
@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_calls(seed, window):
    """Prompts, portions, steps with pauses, copies and releases in a pool that is short: whatever a slot sees is its own or
    shared, what it writes to is its own, and nothing is lost."""
    rng = random.Random(seed)
    c = _slots(5, 120, 14, page=16, window=window, sinks=3)
    content = [dict() for _ in range(14)]       # of the pages: what each place holds
    seen = [[] for _ in range(5)]               # of the slots: what their positions are

    def copy(src, dst):
        content[dst] = dict(content[src])

    c._copy_page = copy

    def write(s, pos, n):
        for j in range(pos, pos + n):
            at = int(c.table[s, j // 16])
            assert at >= 0 and c.refs[at] == 1
            seen[s].append(object())
            content[at][j % 16] = seen[s][j]

    for _ in range(400):
        s, what = rng.randrange(5), rng.choice(["extend", "extend", "step", "step", "step", "copy", "release"])
        if what == "release" and rng.random() < 0.5:
            c.release_row(s)
            c.lens[s] = -1
            seen[s] = []
        elif what == "extend":
            c.exact_lens([s])
            pos, n = max(0, c.host_lens[s]), rng.choice([1, 5, 16, 40])
            try:
                c.reserve([(s, pos, n)])
            except ValueError:
                continue
            write(s, pos, n)
            c.holds(s, pos + n)
            c.lens[s] = pos + n
        elif what == "step":
            growing = [t for t in range(5) if 0 <= int(c.lens[t]) < c.capacity and rng.random() < 0.6]
            try:
                _reserve_a_step(c, growing)
            except ValueError:
                continue
            for t in growing:
                write(t, int(c.lens[t]), 1)
                c.lens[t] += 1
        elif what == "copy":
            d = rng.randrange(5)
            if d != s and int(c.lens[s]) > 0:
                c.copy_row(s, d, int(c.lens[s]))
                c.lens[d] = c.lens[s]
                seen[d] = list(seen[s])
        _sound(c)
        for t in range(5):
            n = int(c.lens[t])
            for j in range(max(n, 0)):
                if not window or j > n - window or j < 3:   # (what a row at position n will see)
                    assert content[int(c.host_table[t, j // 16])][j % 16] is seen[t][j], (what, t, j)
