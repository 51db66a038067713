"""What a BatchDecoder's pages hold when calls fail halfway: each sequence's own
tokens at its positions, over a pool that is kept on the host."""
import numpy as np
import pytest

from runit_mac_amd import dispatch as d
from runit_mac_amd.batch import NO_PAGE
from test_batch_host import Recorder, decoder


class Memory(Recorder):
    """A pool whose positions hold their rows' tokens; the launches of a pass fail
    when `left` others have run, before or (`late`) behind their stores, copies
    when `copies_left` have."""
    left, copies_left, late = 1 << 30, 1 << 30, False

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.mem = np.full((self.pool.num_pages, self.page_size), -1, np.int64)

    def _copy_pages(self, src, dst):
        if self.copies_left == 0:
            raise d.Dispatch("kernel dispatch error: none")
        self.copies_left -= 1
        assert not set(src) & set(dst)
        self.mem[list(dst)] = self.mem[list(src)]

    def _launch(self, batch, rows, picks, targets, top):
        fails, self.left = self.left == 0, max(self.left - 1, 0)
        if fails and not self.late:
            raise d.Dispatch("kernel dispatch error: none")
        h, m = self._host, self._meta
        written = set()
        for i in range(len(batch)):
            r0, r1 = h[m["start"] + i], h[m["start"] + i + 1]
            for r in range(r0, r1):
                pos = int(h[m["kv_len"] + i]) - int(r1 - r)
                page = int(h[m["table"] + i * self.stride + pos // self.page_size])
                assert page != NO_PAGE and (page, pos % self.page_size) not in written
                written.add((page, pos % self.page_size))
                self.mem[page, pos % self.page_size] = h[m["tok"] + r]
        if fails:
            raise d.Dispatch("kernel dispatch error: none")
        return super()._launch(batch, rows, picks, targets, top)

    def held(self, s):
        q, ps, first = self._seqs[s], self.page_size, self.prefix_len // self.page_size
        at = lambda p: self._prefix_pages[p // ps] if p < self.prefix_len else q.pages[p // ps - first]
        return [self.mem[at(p), p % ps] for p in range(q.len)]

    def check(self):
        for s, q in self._seqs.items():
            assert q.len == len(q.tokens) and q.tokens == self.held(s), s
        held = sum({p: 1 for q in self._seqs.values() for p in q.pages}.values()) + len(self._prefix_pages)
        assert held == self.pool.num_pages - self.pool.free


@pytest.mark.parametrize("prefix", [0, 19])
@pytest.mark.parametrize("last,late", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("rows", [2, 5, 10, 64])
def test_forks_of_unequal_length(rows, turned, last, late, prefix):
    """A sequence of 28 positions and its fork of 20, in the same page; both
    write, in one pass or in several, in either order, and the first or last fails."""
    b = decoder(Memory, max_rows=rows)
    b.share_prefix(np.arange(300, 300 + prefix))
    s = b.open()
    b.step({s: np.arange(prefix, 28)})
    t = b.fork(s)
    b.trim(t, 20)
    work = {s: np.arange(100, 103), t: np.arange(200, 210)}
    work = dict(reversed(work.items())) if turned else work
    was = [b.held(x) for x in (s, t)], b.pool.free
    b.left, b.late = -(-13 // rows) - 1 if last else 0, late
    with pytest.raises(d.Dispatch):
        b.step(work)
    assert ([b.held(x) for x in (s, t)], b.pool.free) == was
    b.check()
    b.left = 1 << 30
    b.step(work)
    b.check()


def test_three_holders():
    """The longest of those that all write keeps the page, the last of equals."""
    b = decoder(Memory)
    s = b.open()
    b.step({s: np.arange(12)})
    t, u = b.fork(s), b.fork(s)
    b.trim(s, 9)
    page = b._seqs[s].pages[0]
    b.step({s: [1], t: [2], u: [3]})
    assert b._seqs[u].pages[0] == page and page not in b._seqs[s].pages + b._seqs[t].pages
    b.check()
    b = decoder(Memory)
    s = b.open()
    b.step({s: np.arange(12)})
    t, u = b.fork(s), b.fork(s)
    b.trim(u, 5), b.trim(t, 6)
    page = b._seqs[s].pages[0]
    b.step({s: [1], t: [2], u: [3]})
    assert b._seqs[s].pages[0] == page
    b.check()


@pytest.mark.parametrize("seed", range(40))
def test_any_calls(seed):
    """Forks, trims, steps, drafts and compactions in any order, one in three calls
    failing somewhere: every sequence's positions hold its tokens throughout."""
    rng = np.random.default_rng(seed)
    b = decoder(Memory, max_seqs=5, num_pages=int(rng.integers(8, 30)), max_rows=int(rng.integers(2, 20)))
    b.share_prefix(rng.integers(500, size=rng.integers(0, 40)) if seed % 2 else [])
    failed = 0
    for _ in range(120):
        seqs = list(b._seqs)
        what = rng.choice(["open", "fork", "trim", "close", "compact", *["run"] * 6])
        b.left = int(rng.integers(0, 4)) if rng.random() < 0.3 else 1 << 30
        b.copies_left = int(rng.integers(0, 2)) if rng.random() < 0.1 else 1 << 30
        b.late = bool(rng.random() < 0.5)
        before = {s: (list(q.tokens.ids), q.len) for s, q in b._seqs.items()}, b.pool.free
        try:
            if what == "open":
                b.open()
            elif what == "compact":
                b.compact()
            elif not seqs:
                continue
            elif what == "fork":
                b.fork(rng.choice(seqs))
            elif what == "trim":
                s = rng.choice(seqs)
                b.trim(s, int(rng.integers(b.prefix_len, b.length(s) + 1)))
            elif what == "close":
                b.close(rng.choice(seqs))
            else:
                some = rng.permutation(seqs)[:rng.integers(1, len(seqs) + 1)]
                toks = {int(s): rng.integers(500, size=rng.integers(1, 24)) for s in some}
                call = rng.choice(["step", "score", "verify"])
                if call == "verify":
                    b.verify({s: (int(t[0]), t[1:5]) for s, t in toks.items()})
                else:
                    getattr(b, call)(toks)
        except (d.Dispatch, d.BufferSize, ValueError):
            failed += 1
            assert ({s: (list(q.tokens.ids), q.len) for s, q in b._seqs.items()}, b.pool.free) == before
        b.check()
    assert failed
