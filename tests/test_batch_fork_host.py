"""What a BatchDecoder does on the host when sequences fork, pages are compacted
and rules hold: who holds which page, what is copied, what is given back."""
import numpy as np
import pytest

from runit_mac_amd import dispatch as d
from runit_mac_amd.batch import PagePool, Rules
from test_batch_host import CFG, Failing, Recorder, decoder


class Copying(Failing):
    """Keeps the copies; they fail when `copies_left` others have been made."""
    copies, copies_left = (), 1 << 30

    def _copy_pages(self, src, dst):
        if self.copies_left == 0:
            raise d.Dispatch("kernel dispatch error: none")
        self.copies_left -= 1
        self.copies = [*self.copies, (list(src), list(dst))]


def pages(b, s):
    return list(b._seqs[s].pages)


def test_pool_counts_holders():
    p = PagePool(4)
    a = p.take(2)
    p.share(a[:1])
    assert [p.holders(x) for x in a] == [2, 1] and p.free == 2
    p.give(a)
    assert p.free == 3 and p.holders(a[0]) == 1 and p.holders(a[1]) == 0
    p.give(a[:1])
    assert p.free == 4
    with pytest.raises(KeyError):
        p.give(a[:1])


def test_fork_shares_until_a_write():
    """A begun page is copied by the first of its two writers; the second keeps
    it.  Whole pages stay shared."""
    b = decoder(Copying)
    s = b.open()
    b.step({s: np.arange(20)})
    before = pages(b, s)
    t = b.fork(s)
    assert pages(b, t) == before and b.length(t) == 20 and b.pool.free == 10 and not b.copies
    b.step({s: [1], t: [2]})
    assert len(b.copies) == 1 and b.copies[0][0] == [before[1]] and b.pool.free == 9
    assert pages(b, s)[0] == pages(b, t)[0] == before[0] and pages(b, t)[1] == before[1]
    assert pages(b, s)[1] == b.copies[0][1][0]
    tables = b.passes[-1]["table"]
    assert list(tables[0, :2]) == pages(b, s) and list(tables[1, :2]) == pages(b, t)
    b.step({s: [3], t: [4]})
    assert len(b.copies) == 1
    b.close(s)
    assert b.pool.free == 10
    b.close(t)
    assert b.pool.free == 12


def test_fork_at_a_page_boundary_copies_nothing():
    b = decoder(Copying)
    s = b.open()
    b.step({s: np.arange(16)})
    t = b.fork(s)
    b.step({s: [1], t: [2]})
    assert not b.copies and pages(b, s)[0] == pages(b, t)[0] and b.pool.free == 9


def test_only_one_of_the_forks_writes():
    b = decoder(Copying)
    s = b.open()
    b.step({s: [1, 2, 3]})
    t, u = b.fork(s), b.fork(s)
    b.step({t: [4]})
    assert len(b.copies) == 1 and pages(b, s) == pages(b, u) != pages(b, t)
    b.step({u: [5]})
    assert len(b.copies) == 2
    b.step({s: [6]})
    assert len(b.copies) == 2 and b.pool.free == 9


def test_trim_into_a_shared_page_then_write():
    b = decoder(Copying)
    s = b.open()
    b.step({s: np.arange(32)})
    t = b.fork(s)
    b.trim(t, 18)
    assert pages(b, t) == pages(b, s)
    b.step({t: [1]})
    assert len(b.copies) == 1 and pages(b, t)[1] != pages(b, s)[1] and b._seqs[t].tokens == [*range(18), 1]
    b.trim(s, 16)
    assert b.pool.holders(pages(b, s)[0]) == 2 and len(pages(b, s)) == 1


def test_fork_behind_a_shared_prompt():
    b = decoder(Copying)
    b.share_prefix(np.arange(21))
    s = b.open()
    t = b.fork(s)
    assert b.length(t) == 21 and pages(b, t) == []
    b.step({s: [1], t: [2]})
    u = b.fork(t)
    b.step({u: [3]})
    assert [len(c[0]) for c in b.copies] == [1] and b._seqs[u].tokens == [*range(21), 2, 3]


def test_pages_for_the_copies_are_asked_for():
    """Three holders that all write need two pages; one too few is refused
    before anything runs."""
    b = decoder(Copying, num_pages=3)
    s = b.open()
    b.step({s: [1, 2]})
    t, u = b.fork(s), b.fork(s)
    b.step({s: [1], t: [2], u: [3]})
    assert [len(c[0]) for c in b.copies] == [2] and b.pool.free == 0
    b = decoder(Copying, num_pages=2)
    s = b.open()
    b.step({s: [1, 2]})
    t, u = b.fork(s), b.fork(s)
    n = len(b.passes)
    with pytest.raises(d.BufferSize):
        b.step({s: [1], t: [2], u: [3]})
    assert b.pool.free == 1 and not b.copies and len(b.passes) == n
    with pytest.raises(d.BufferSize):
        b.fork(s)  # (no room for a fourth sequence)


@pytest.mark.parametrize("left,copies_left", [(0, 9), (1, 9), (9, 0)])
def test_a_call_that_fails_undoes_its_copies(left, copies_left):
    b = decoder(Copying)
    s = b.open()
    b.step({s: np.arange(20)})
    t = b.fork(s)
    was = pages(b, s), pages(b, t), b.pool.free, [b.pool.holders(p) for p in pages(b, s)]
    b.left, b.copies_left = left, copies_left
    with pytest.raises(d.Dispatch):
        b.step({s: np.arange(6), t: np.arange(7)})
    assert (pages(b, s), pages(b, t), b.pool.free, [b.pool.holders(p) for p in pages(b, s)]) == was
    assert b.length(s) == b.length(t) == 20 and b._seqs[s].tokens == b._seqs[t].tokens == [*range(20)]
    b.left = b.copies_left = 1 << 30
    b.step({s: [1], t: [2]})
    assert pages(b, s)[1] != pages(b, t)[1]


def test_compact():
    """Pages in use behind the first ones go to free places before them."""
    b = decoder(Copying)
    b.share_prefix(np.arange(16))
    s, t = b.open(), b.open()
    b.step({s: np.arange(40), t: np.arange(20)})
    u = b.fork(t)
    b.close(s)
    old = pages(b, t)
    assert b.compact() == 3
    src, dst = b.copies[-1]
    held = pages(b, t) + b._prefix_pages
    assert sorted(held) == [0, 1, 2] and pages(b, u) == pages(b, t) and not set(src) & set(dst)
    assert all((dst[src.index(o)] if o in src else o) == n for o, n in zip(old, pages(b, t)))
    n = len(b.copies)
    assert b.compact() == 3 and len(b.copies) == n
    b.step({t: [1], u: [2]})
    b.close(t), b.close(u)
    b.share_prefix([])
    assert b.pool.free == 12 and sorted(b.pool.take(12)) == list(range(12))


def test_tokens_follow_the_positions():
    b = decoder()
    s = b.open()
    b.step({s: np.arange(10)})
    b.verify({s: (10, [11, 12, 40])})
    assert b._seqs[s].tokens == [*range(10), 10, 11, 12] and b.length(s) == 13
    b.score({s: [5, 6]})
    b.trim(s, 3)
    assert b._seqs[s].tokens == [0, 1, 2]


class Ruled(Recorder):
    seen = ()

    def _launch(self, *args):
        self.seen = [*self.seen, self._pick_rules]
        return super()._launch(*args)


def test_rules_reach_their_rows():
    """With the sequence's tokens up to the row, in the pass that keeps it."""
    b = decoder(Ruled)
    s, t, u = b.open(), b.open(), b.open()
    r = Rules(frequency=0.5, prompt_len=3)
    b.step({s: np.arange(5), t: [7, 8], u: np.arange(20, 31)}, rules={t: r, u: r})
    assert b.seen == [[None, (r, [7, 8])], None, [(r, [*range(20, 31)])]]
    b.step({s: [9], t: [9], u: [9]}, rules={u: r})
    assert b.seen[-1] == [None, None, (r, [*range(20, 31), 9])]
    b.step({s: [9]})
    assert b.seen[-1] is None


def test_rules_are_checked():
    n = CFG.vocab
    assert np.array_equal(np.unpackbits(Rules(allowed=np.arange(n) % 3 == 0).mask(n).view(np.uint8), bitorder="little")[:n],
                          np.arange(n) % 3 == 0)
    words = np.arange(16, dtype=np.uint32)
    assert Rules(allowed=words).mask(n) is words
    b = decoder(Ruled)
    s, t = b.open(), b.open()
    for bad in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=np.inf), dict(repetition=np.nan),
                dict(frequency=np.nan), dict(presence=np.inf), dict(prompt_len=-1), dict(bias={n: 1.0}), dict(bias={-1: 1.0}),
                dict(allowed=np.ones(n - 1, bool)), dict(allowed=np.ones(n, np.int32)), dict(allowed=np.ones(17, np.uint32))):
        with pytest.raises(ValueError):
            b.step({s: [1]}, rules={s: Rules(**bad)})
    with pytest.raises(ValueError):
        b.step({s: [1]}, rules={t: Rules()})
    assert not b.passes and b.length(s) == 0


def test_rules_that_leave_no_choice():
    n = CFG.vocab
    b = decoder(Ruled)
    s = b.open()
    for bad in (dict(allowed=np.zeros(n, bool)), dict(allowed=np.zeros(-(-n // 32), np.uint32)), dict(bias={3: np.nan})):
        with pytest.raises(ValueError):
            b.step({s: [1]}, rules={s: Rules(**bad)})
    assert not b.passes and b.length(s) == 0
    b.step({s: [1]}, rules={s: Rules(allowed=np.arange(2 * n)[::2] == 2, bias={3: -np.inf})})
