"""phx_pages_*: the page bookkeeping against a model that keeps every
sequence's tokens in words, and its refusals.  Host only."""
import random

import numpy as np
import pytest

import phobos_amd as px


class Model:
    """Pages hold words; a copy, launched later, carries them over."""

    def __init__(self, pages, P):
        self.pool, self.P = px.Pages(pages, P), P
        self.data = np.zeros((pages, P), np.int64)
        self.words = {}  # sequence -> its tokens
        self.count = 0

    def flush(self):
        src, dst = self.pool.pending(clear=True)
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        order = list(range(len(src)))
        random.Random(len(src)).shuffle(order)  # any order is right
        for i in order:
            self.data[dst[i]] = self.data[src[i]]

    def write(self, seq, start):
        t = self.pool.table(seq)
        for i in range(start, len(self.words[seq])):
            self.data[t[i // self.P], i % self.P] = self.words[seq][i]

    def check(self):
        owners = {}
        for seq, words in self.words.items():
            t = self.pool.table(seq)
            assert len(t) == -(-len(words) // self.P)
            assert len(set(t)) == len(t)
            got = self.data[t].reshape(-1)[:len(words)]
            assert np.array_equal(got, words), seq
            for p in t:
                owners.setdefault(int(p), set()).add(seq)
        used, top, pending = self.pool.stats()
        return owners, used, top, pending


def test_fork_copies_only_the_page_it_writes():
    pool = px.Pages(16, 4)
    a = pool.new()
    pool.resize(a, 10)
    b = pool.fork(a)
    assert list(pool.table(b)) == list(pool.table(a)) == [0, 1, 2]
    pool.resize(b, 11)
    assert list(pool.table(b)) == [0, 1, 3]
    assert [list(x) for x in pool.pending()] == [[2], [3]]
    pool.resize(a, 11)  # a is the page's only owner now
    assert list(pool.table(a)) == [0, 1, 2]
    assert pool.stats() == (4, 4, 1)


def test_a_full_last_page_is_shared_on():
    pool = px.Pages(4, 4)
    a = pool.new()
    pool.resize(a, 8)
    b = pool.fork(a)
    pool.resize(b, 9)
    assert list(pool.table(b)) == [0, 1, 2] and pool.stats()[2] == 0


def test_a_copy_of_a_pending_copy_reads_its_source():
    pool = px.Pages(8, 4)
    a = pool.new()
    pool.resize(a, 2)
    b = pool.fork(a)
    pool.resize(b, 3)  # 0 -> 1
    c = pool.fork(b)
    pool.resize(c, 4)  # from 1, whose words are still in 0
    assert [list(x) for x in pool.pending()] == [[0, 0], [1, 2]]
    with pytest.raises(px.PhxError):
        px.check(px.lib().phx_pages_pending(pool.handle, None, None, 0, None, 1))
    # sources and destinations stay held, whoever is freed
    for s in (a, b, c):
        pool.free(s)
    assert pool.stats() == (3, 3, 2)
    d = pool.new()
    pool.resize(d, 20)
    assert list(pool.table(d)) == [3, 4, 5, 6, 7]
    with pytest.raises(px.PhxError):
        pool.resize(d, 21)
    assert list(pool.table(d)) == [3, 4, 5, 6, 7]


def test_exhausted_changes_nothing():
    pool = px.Pages(3, 4)
    a = pool.new()
    pool.resize(a, 10)
    b = pool.fork(a)
    with pytest.raises(px.PhxError) as e:
        pool.resize(b, 11)  # its own last page would be a fourth
    assert e.value.code == px.PHX_E_EXHAUSTED
    assert pool.stats() == (3, 3, 0) and list(pool.table(b)) == [0, 1, 2]
    pool.resize(b, 8)
    pool.free(a)
    pool.resize(b, 12)
    assert list(pool.table(b)) == [0, 1, 2]


def test_compaction_moves_to_the_lowest_pages():
    pool = px.Pages(10, 1)
    seqs = []
    for _ in range(8):
        seqs.append(pool.new())
        pool.resize(seqs[-1], 1)
    for i in (0, 2, 3, 5):
        pool.free(seqs[i])
    twin = pool.fork(seqs[7])
    pool.compact()
    assert [int(pool.table(seqs[i])[0]) for i in (1, 4, 6, 7)] == [1, 0, 2, 3]
    assert list(pool.table(twin)) == [3]
    assert sorted(zip(*(list(x) for x in pool.pending()))) == [(4, 0), (6, 2), (7, 3)]
    with pytest.raises(px.PhxError):
        pool.compact()
    # what moves are from is not given out before they ran
    n = pool.new()
    pool.resize(n, 3)
    assert list(pool.table(n)) == [5, 8, 9]


@pytest.mark.parametrize("seed", range(8))
def test_random_operations_keep_every_word(seed):
    rng = random.Random(seed)
    P = rng.choice([1, 3, 4])
    m = Model(24, P)
    unwritten = []  # (sequence, first new token): its copies have not run yet
    for step in range(600):
        op = rng.random()
        seqs = sorted(m.words)
        busy = {s for s, _ in unwritten}
        if op < 0.15 or not seqs:
            m.words[m.pool.new()] = np.zeros(0, np.int64)
        elif op < 0.6:
            s = rng.choice(seqs)
            n = rng.randrange(0, 6 * P) if op < 0.25 else len(m.words[s]) + rng.randrange(0, 2 * P)
            before, stats, table = len(m.words[s]), m.pool.stats(), list(m.pool.table(s))
            if s in busy:
                continue
            try:
                m.pool.resize(s, n)
            except px.PhxError as e:
                assert e.code == px.PHX_E_EXHAUSTED
                assert m.pool.stats() == stats and list(m.pool.table(s)) == table
            else:
                if n > before:
                    new = np.arange(m.count, m.count + n - before)
                    m.count += n - before
                    m.words[s] = np.concatenate([m.words[s], new])
                    unwritten.append((s, before))
                else:
                    m.words[s] = m.words[s][:n]
        elif op < 0.75:
            s = rng.choice(seqs)
            if s not in busy:
                m.words[m.pool.fork(s)] = m.words[s].copy()
        elif op < 0.85:
            s = rng.choice(seqs)
            m.pool.free(s)
            del m.words[s]
            unwritten = [u for u in unwritten if u[0] != s]
        elif op < 0.9 and m.pool.stats()[2] == 0 and not unwritten:
            m.pool.compact()
            m.flush()
            owners, used, top, pending = m.check()
            assert (used, top, pending) == (len(owners), len(owners), 0)
        else:  # run the copies, then write the new tokens
            m.flush()
            for u in unwritten:
                m.write(*u)
            unwritten = []
            owners, used, top, pending = m.check()
            assert used == len(owners) and pending == 0 and top == max(owners, default=-1) + 1


def test_refusals():
    L = px.lib()
    for pages, P in [(0, 4), (-1, 4), (4, 0), (4, -3)]:
        with pytest.raises(px.PhxError):
            px.Pages(pages, P)
    pool = px.Pages(4, 4)
    a = pool.new()
    for call in (lambda: pool.resize(a, -1), lambda: pool.resize(a + 1, 1), lambda: pool.fork(7),
                 lambda: pool.free(7), lambda: pool.table(7), lambda: pool.resize(a, 1 << 62)):
        with pytest.raises(px.PhxError):
            call()
    pool.free(a)
    with pytest.raises(px.PhxError):
        pool.free(a)
    assert L.phx_pages_new(None, None) == px.PHX_E_INVALID
    assert L.phx_pages_table(pool.handle, pool.new(), None, 3, None) == px.PHX_E_INVALID
    assert L.phx_pages_destroy(None) == 0


def test_lists_that_change_between_their_size_and_their_contents(monkeypatch):
    # calls on one pool may come from several threads
    pool = px.Pages(16, 4)
    a = pool.new()
    pool.resize(a, 10)
    pool.resize(pool.fork(a), 11)
    L = px.lib()

    def between(name, act):
        """The first call of `name` that asks for a size, then act()."""
        real, left = getattr(L, name), [1]

        def call(*args):
            rc = real(*args)
            if left and left.pop():
                act()
            return rc
        monkeypatch.setattr(L, name, call)

    between("phx_pages_table", lambda: pool.resize(a, 3))
    assert list(pool.table(a)) == [0]
    monkeypatch.undo()
    between("phx_pages_table", lambda: pool.resize(a, 30))
    t = list(pool.table(a))
    assert len(t) == 8 and len(set(t)) == 8
    monkeypatch.undo()
    n = pool.stats()[2]
    assert n >= 1
    between("phx_pages_stats", lambda: pool.pending(clear=True))
    src, dst = pool.pending(clear=True)
    assert len(src) == len(dst) == 0
    monkeypatch.undo()

    def more():
        pool.resize(pool.fork(a), 31)

    between("phx_pages_stats", more)
    src, dst = pool.pending(clear=True)
    assert len(src) == len(dst) == 1 and pool.stats()[2] == 0
