"""Sequences that go on from one another: pages held together, copies before writing, what rows share.  On the host, with the pools in host
memory: every cell holds the token that was written there, so what a sequence reads can be compared with what it wrote."""
import random

import numpy as np
import pytest
import torch

from quicknn_b200.cache import PAGE, CacheFull, KVCache, PagePool
from quicknn_b200.parts import CacheNeed, StateNeed


def make(max_tokens=2048, max_slots=6, max_seq=1024, window=None, states=False):
    needs = [CacheNeed(1, 4, window), CacheNeed(1, 4, None), CacheNeed(1, 4, window, values=False)]
    st = [StateNeed((3,), "float32"), None, None] if states else [None] * 3
    return KVCache(needs, st, max_tokens, max_slots, max_seq, torch.float32, "cpu", [None, StateNeed((2, 2), "bfloat16"), None] if states else ())


def test_pages_with_several_holders():
    p = PagePool(6)
    a = p.take(2)
    p.share(a)
    p.share(a[:1])
    assert p.holders(1) == 3 and p.holders(2) == 2 and p.n_free == 3 and p.n_held == 2
    p.give_back(a)
    p.audit()
    assert p.n_free == 3
    p.give_back(a)
    assert p.n_free == 4 and p.holders(1) == 1
    p.give_back([1])
    with pytest.raises(RuntimeError):
        p.give_back([1])
    with pytest.raises(RuntimeError):
        p.share([1])
    with pytest.raises(RuntimeError):
        p.share([0])
    p.audit()


class Tape:
    """A cache whose sequences are written cell by cell, as the engine does, and read back."""

    def __init__(self, cache):
        self.c, self.said, self.mark = cache, {}, 0

    def new(self):
        s = self.c.allocate()
        self.said[s] = []
        return s

    def say(self, *slots_n):
        self.c.extend([(s, len(self.said[s]) + n) for s, n in slots_n])
        for s, n in slots_n:
            for _ in range(n):
                self.mark += 1
                pos = len(self.said[s])
                self.said[s].append(self.mark)
                for g in self.c.groups:
                    at = pos % g.ring if g.ring else pos
                    page = g.table_host[s, at // PAGE]
                    assert page > 0 and g.pool.holders(page) == 1
                    g.k[:, page, :, at % PAGE] = self.mark
                    if g.need.values:
                        g.v[:, page, :, at % PAGE] = -self.mark

    def fork(self, sources):
        out = self.c.fork(sources)
        for s, d in zip(sources, out):
            self.said[d] = list(self.said[s])
        return out

    def drop(self, s):
        self.c.free(s)
        del self.said[s]

    def check(self):
        self.c.audit()
        for s, said in self.said.items():
            assert self.c.length(s) == len(said)
            for g in self.c.groups:
                w = g.need.window if g.ring else len(said)
                for pos in range(max(0, len(said) - w), len(said)):
                    at = pos % g.ring if g.ring else pos
                    page = g.table_host[s, at // PAGE]
                    assert (g.k[:, page, :, at % PAGE] == said[pos]).all(), (s, pos)


@pytest.mark.parametrize("window", [None, 100, 128])
def test_forks_write_beside_one_another(window):
    t = Tape(make(window=window))
    a = t.new()
    t.say((a, 150))
    full = next(g for g in t.c.groups if not g.ring)
    before = full.pool.n_held
    b, c = t.fork([a, a])
    assert full.pool.n_held == before and full.held[b] == full.held[a]          # nothing copied yet
    t.check()
    t.say((a, 1), (b, 1), (c, 1))
    assert full.held[b][:2] == full.held[a][:2] and len({full.held[s][2] for s in (a, b, c)}) == 3
    t.check()
    for _ in range(5):
        t.say((a, 31), (b, 33), (c, 70))
        t.check()
    t.drop(a)
    t.check()
    d, = t.fork([c])
    t.say((c, 1))
    t.say((b, 40), (d, 2))
    t.check()
    for s in list(t.said):
        t.drop(s)
    assert all(g.pool.n_held == 0 for g in t.c.groups) and t.c.sharing == 0


def test_a_whole_last_page_is_not_copied():
    t = Tape(make())
    a = t.new()
    t.say((a, 128))
    b, = t.fork([a])
    t.say((a, 1), (b, 1))
    g = t.c.groups[0]
    assert g.held[a][:2] == g.held[b][:2] and g.held[a][2] != g.held[b][2]
    t.check()


def test_the_last_holder_writes_into_the_page_itself():
    t = Tape(make())
    a = t.new()
    t.say((a, 10))
    page = t.c.groups[0].held[a][0]
    b, = t.fork([a])
    t.drop(a)
    t.say((b, 1))
    assert t.c.groups[0].held[b] == [page]
    t.check()


def test_states_are_copied():
    c = make(states=True)
    a = c.allocate()
    for t in c._all_states():
        t[a] = 7
    b, d = c.fork([a, a])
    for t in c._all_states():
        t[a] = 1
        assert (t[b] == 7).all() and (t[d] == 7).all()
    e = c.allocate()
    assert not any(t[e].any() for t in c._all_states())


def test_all_or_nothing():
    c = make(max_tokens=256, max_slots=3)
    a = c.allocate()
    c.extend([(a, 70)])
    with pytest.raises(CacheFull):
        c.fork([a, a, a])
    c.audit()
    b, d = c.fork([a, a])
    with pytest.raises(CacheFull):                       # a copy for two of the three, a page more for the third's 129 tokens: 3 of 2 left
        c.extend([(a, 71), (b, 71), (d, 129)])
    assert [c.length(s) for s in (a, b, d)] == [70] * 3
    c.audit()
    c.extend([(a, 71), (b, 71), (d, 71)])
    assert c.groups[0].pool.n_free == 0
    c.audit()
    with pytest.raises(RuntimeError):
        c.fork([5])
    c.free(a)
    with pytest.raises(RuntimeError):
        c.fork([a])
    assert c.fork([]) == []


def test_cut_back_into_common_pages():
    t = Tape(make())
    a = t.new()
    t.say((a, 200))
    b, = t.fork([a])
    t.say((b, 3))
    t.c.truncate([(b, 90)])
    t.said[b] = t.said[b][:90]
    t.check()
    t.say((b, 5))                                        # into a page that `a` holds too
    t.check()
    t.say((a, 1))
    t.check()


@pytest.mark.parametrize("window", [None, 70, 192])
@pytest.mark.parametrize("seed", range(4))
def test_random_walk(window, seed):
    rnd = random.Random(seed)
    t = Tape(make(max_tokens=4096, max_slots=7, window=window))
    for _ in range(150):
        r = rnd.random()
        live = list(t.said)
        try:
            if r < 0.15 or not live:
                t.new()
            elif r < 0.4:
                t.fork([rnd.choice(live) for _ in range(rnd.choice([1, 1, 2, 3]))])
            elif r < 0.55:
                t.drop(rnd.choice(live))
            else:
                some = rnd.sample(live, rnd.randint(1, len(live)))
                t.say(*[(s, rnd.choice([1, 1, 2, 17, 64, 90])) for s in some if len(t.said[s]) < 800])
        except CacheFull:
            pass
        t.c.audit()
        live = list(t.said)
        rnd.shuffle(live)
        live.sort(key=lambda s: t.c._family[s])
        live = [s for s in live if t.said[s]]
        runs = t.c.families(live)
        for g, found in zip(t.c.groups, t.c.shared_positions(live, runs)):
            for run, (begin, end) in zip(runs, found):
                assert rows_hold(t.c, live, run, g, begin, end) and (end == 0 or longest_common(t.c, live, run, g) <= (end - begin) // PAGE)
    t.check()


def longest_common(c, slots, run, g):
    """Pages that all rows of a run hold together and that no row's ring has lost."""
    rows = slots[run[0]:run[0] + run[1]]
    n = g.pages_per_seq
    first = max(0, (max(c.length(s) for s in rows) - 1) // PAGE - n + 1) if g.ring else 0
    last = (min(c.length(s) for s in rows) - 1) // PAGE
    return sum(len({int(g.table_host[s, p % n]) for s in rows}) == 1 for p in range(first, last + 1))


def rows_hold(c, slots, run, g, begin, end):
    """By the definition: a position's page is the same in all rows, where the row still holds the position."""
    for p in range(begin, end):
        ids = set()
        for s in slots[run[0]:run[0] + run[1]]:
            n = c.length(s)
            if p < n and (not g.ring or p >= n - g.ring):
                ids.add(int(g.table_host[s, (p % g.ring if g.ring else p) // PAGE]))
        if len(ids) > 1:
            return False
    return True


@pytest.mark.parametrize("window", [None, 100, 192])
def test_what_rows_share(window):
    t = Tape(make(max_tokens=8192, max_slots=9, window=window))
    a, z = t.new(), t.new()
    t.say((a, 300), (z, 20))
    assert t.c.families([a, z]) == [] and t.c.sharing == 0
    b, c = t.fork([a, a])
    y, = t.fork([z])
    assert t.c.families([a, b, c, z, y]) == [(0, 3), (3, 2)] and t.c.families([a, z, b, y]) == [] and t.c.families([z, b, c]) == [(1, 2)]
    for round_ in range(8):
        t.say((a, 1), (b, 1 + 9 * round_), (c, 1), (z, 1), (y, 1))
        slots = [a, b, c, z, y]
        runs = t.c.families(slots)
        got = t.c.shared_positions(slots, runs)
        for g, ab in zip(t.c.groups, got):
            for run, (begin, end) in zip(runs, ab):
                assert begin % PAGE == 0 and end % PAGE == 0 and 0 <= begin <= end
                assert rows_hold(t.c, slots, run, g, begin, end)
            if not g.ring:
                assert ab == [(0, 256), (0, 0)]                # the whole pages of what was common
            elif round_ == 0 and window == 192:
                assert ab[0] == (128, 256)                     # the ring's newest page is everyone's own
    t.drop(b)
    t.drop(c)
    assert t.c.families([a, z, y]) == [(1, 2)]
    t.drop(y)
    assert t.c.sharing == 0 and t.c.families([a, z]) == []


def test_tables_of_rows_that_just_forked():
    c = make()
    a = c.allocate()
    c.extend([(a, 130)])
    b, = c.fork([a])
    assert c.shared_positions([a, b], [(0, 2)]) == [[(0, 192)]] * len(c.groups)      # the partly filled page too, as yet
    assert np.array_equal(c.groups[0].table_host[a], c.groups[0].table_host[b])


@pytest.mark.parametrize("order", [0, 1])
def test_a_ring_that_was_extended_and_cut_back_shares_only_what_it_still_holds_in_the_same_pages(order):
    """What undoes a step that could not be launched: the cells that its tokens would have gone into are copies of one sequence's own, at
    the end and, where they have wrapped, in front of what is still common."""
    t = Tape(make(window=192))
    a = t.new()
    t.say((a, 500))                                      # pages 5, 6 and 7 of a ring of three
    b, = t.fork([a])
    t.c.extend([(a, 520)])                               # a place in page 7, and page 8 in that of page 5
    t.c.truncate([(a, 500)])
    rows = [a, b][::1 - 2 * order]
    for g, found in zip(t.c.groups, t.c.shared_positions(rows, [(0, 2)])):
        assert found == ([(6 * PAGE, 7 * PAGE)] if g.ring else [(0, 7 * PAGE)])
        assert rows_hold(t.c, rows, (0, 2), g, *found[0])
    t.say((b, 13))
    t.c.audit()
    for g, found in zip(t.c.groups, t.c.shared_positions(rows, [(0, 2)])):
        assert rows_hold(t.c, rows, (0, 2), g, *found[0])


@pytest.mark.parametrize("window", [70, 192])
@pytest.mark.parametrize("seed", range(4))
def test_random_walk_with_steps_that_are_undone(window, seed):
    rnd = random.Random(1000 + seed)
    c = make(max_tokens=4096, max_slots=7, window=window)
    live = []
    for _ in range(200):
        r = rnd.random()
        try:
            if r < 0.1 or not live:
                live.append(c.allocate())
            elif r < 0.3:
                live += c.fork([rnd.choice(live) for _ in range(rnd.choice([1, 1, 2]))])
            elif r < 0.4:
                c.free(live.pop(rnd.randrange(len(live))))
            else:
                some = [(s, c.length(s)) for s in rnd.sample(live, rnd.randint(1, len(live))) if c.length(s) < 800]
                c.extend([(s, n + rnd.choice([1, 1, 17, 64, 90, 200])) for s, n in some])
                if r > 0.8:
                    c.truncate(some)
        except CacheFull:
            pass
        c.audit()
        rows = sorted((s for s in live if c.length(s)), key=lambda s: (c._family[s], rnd.random()))
        runs = c.families(rows)
        for g, found in zip(c.groups, c.shared_positions(rows, runs)):
            assert all(rows_hold(c, rows, run, g, *f) for run, f in zip(runs, found))
