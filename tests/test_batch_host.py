"""What a BatchDecoder does on the host: pages, tables, lengths, refusals."""
from types import SimpleNamespace

import numpy as np
import pytest

from runit_mac_amd import dispatch as d
from runit_mac_amd.batch import NO_PAGE, BatchDecoder, PagePool
from runit_mac_amd.decode import DecodeConfig

CFG = DecodeConfig(layers=2, hidden=128, heads=4, kv_heads=2, head_dim=64, ff=256, vocab=500, max_seq=200)


def model(cfg=CFG, lm_fmt="q8_0", **F):
    fmts = [dict(dict.fromkeys(("q", "k", "v", "o", "gate", "up", "down"), "q8_0"), **F)] * cfg.layers
    ctx = SimpleNamespace(new_buffer=lambda n: SimpleNamespace(ptr=1 << 20, nbytes=n, free=lambda: None))
    return SimpleNamespace(cfg=cfg, ctx=ctx, lm_fmt=lm_fmt, fmts=fmts, layers=[{}] * cfg.layers)


class Recorder(BatchDecoder):
    """Launches nothing; keeps each pass's arrays, and predicts the token
    after a row's own."""
    passes = ()

    def _launch(self, batch, rows, picks, targets, top):
        h, m, n = self._host, self._meta, len(batch)
        get = lambda k, size: h[m[k]:m[k] + size].copy()
        self.passes = [*self.passes, dict(tok=get("tok", rows), keep=get("keep", len(picks)), start=get("start", n + 1),
                                          target=get("target", len(picks)), kv_len=get("kv_len", n),
                                          table=get("table", n * self.stride).reshape(n, -1),
                                          shared=get("shared", len(self._prefix_pages)))]
        tok = targets if targets is not None else [(h[m["tok"] + p] + 1) % self.model.cfg.vocab for p in picks]
        k = len(picks)
        return (np.array(tok, np.uint32), *(np.zeros(k) for _ in range(3)),
                *(np.zeros((k, top or 0)) for _ in range(2))) if picks else ()


def decoder(cls=Recorder, **kw):
    kw = dict(dict(max_seqs=3, num_pages=12, page_size=16, max_rows=8, max_top=4), **kw)
    return cls(model(), **kw)


def test_page_pool_gives_each_page_once():
    p = PagePool(5)
    a, b = p.take(2), p.take(3)
    assert sorted(a + b) == [0, 1, 2, 3, 4] and p.free == 0
    with pytest.raises(d.BufferSize):
        p.take(1)
    p.give(a)
    assert p.free == 2 and sorted(p.take(2)) == sorted(a)


def test_step_in_passes():
    """Prompts of 11, 1 and 6 tokens in passes of 8 rows: in order, lengths
    counting the pass's rows, a page for each begun 16 positions."""
    b = decoder()
    s = [b.open() for _ in range(3)]
    prompts = [np.arange(11), [77], np.arange(200, 206)]
    got = b.step(dict(zip(s, prompts)))
    assert got == {s[0]: 11, s[1]: 78, s[2]: 206}
    p = b.passes
    assert [list(x["start"]) for x in p] == [[0, 8], [0, 3, 4, 8], [0, 2]]
    assert [list(x["kv_len"]) for x in p] == [[8], [11, 1, 4], [6]]
    assert [list(x["keep"]) for x in p] == [[], [2, 3], [1]]
    assert np.array_equal(np.concatenate([x["tok"] for x in p]), np.concatenate(prompts))
    assert [b.length(x) for x in s] == [11, 1, 6]
    assert b.pool.free == 9
    assert np.all(p[1]["table"][:, 1:] == NO_PAGE) and len(set(p[1]["table"][:, 0])) == 3
    b.step({s[0]: np.arange(5)})
    assert b.pool.free == 9  # (16 positions)
    b.step({s[0]: [1]})
    assert b.pool.free == 8 and b.passes[-1]["kv_len"][0] == 17
    b.trim(s[0], 16)
    assert b.pool.free == 9 and b.length(s[0]) == 16
    for x in s:
        b.close(x)
    assert b.pool.free == 12


def test_passes_stay_within_what_their_calls_take():
    """65,535 rows of the embedding, 14,336 of the argmax."""
    b = decoder(max_rows=100_000, max_logits=100_000)
    assert b.max_rows == 65535 and b.max_logits == 14336


def test_score_keeps_all_but_the_last():
    b = decoder()
    s, t = b.open(), b.open()
    got = b.score({s: np.arange(100, 110), t: [5]}, top=2)
    assert np.array_equal(got[s].tokens, np.arange(101, 110)) and got[s].top_ids.shape == (9, 2)
    assert got[t].tokens.size == 0 and got[t].top_ids.shape == (0, 2)
    assert [list(x["keep"]) for x in b.passes] == [list(range(8)), [0]]
    assert list(b.passes[1]["target"]) == [109]


@pytest.mark.parametrize("n", [16, 21])
def test_shared_prefix(n):
    """Its pages are the shared table's; sequences begin behind it, on a page
    of their own where it ends inside one."""
    b = decoder()
    b.share_prefix(np.arange(n))
    used = -(-n // 16)
    assert b.prefix_len == n and b.pool.free == 12 - used
    s, t = b.open(), b.open()
    assert b.length(s) == n
    b.step({s: [1, 2], t: [3]})
    p = b.passes[-1]
    assert list(p["kv_len"]) == [n + 2, n + 1] and len(p["shared"]) == used
    own = p["table"][:, n // 16]
    assert len(set(own) | set(p["shared"])) == 2 + used and NO_PAGE not in own
    assert np.all(p["table"][:, :n // 16] == NO_PAGE) and np.all(p["table"][:, n // 16 + 1:] == NO_PAGE)
    b.trim(s, n)
    assert b.pool.free == 12 - used - 1
    with pytest.raises(ValueError):
        b.trim(s, n - 1)
    with pytest.raises(ValueError):
        b.share_prefix([1])
    b.close(s), b.close(t)
    b.share_prefix([])
    assert b.pool.free == 12 and b.prefix_len == 0


def test_verify_keeps_the_accepted():
    b = decoder()
    s, t = b.open(), b.open()
    got = b.verify({s: (10, [11, 12, 40, 41]), t: (20, [])})
    assert got == {s: (2, 13), t: (0, 21)}
    assert b.length(s) == 3 and b.length(t) == 1


class Failing(Recorder):
    """The launches of a pass fail when `left` others have run."""
    left = 1 << 30

    def _launch(self, *args):
        if self.left == 0:
            raise d.Dispatch("kernel dispatch error: none")
        self.left -= 1
        return super()._launch(*args)


@pytest.mark.parametrize("left", [0, 1, 2])
@pytest.mark.parametrize("prefix", [0, 21])
def test_a_call_that_fails_changes_no_sequence(left, prefix):
    """Lengths and pages as before it, in whichever pass it fails; the next
    call begins there."""
    b = decoder(Failing, num_pages=16)
    b.share_prefix(np.arange(prefix))
    s, t = b.open(), b.open()
    b.step({s: np.arange(10), t: [1]})
    free, lens = b.pool.free, [b.length(s), b.length(t)]
    for call in (lambda: b.step({s: np.arange(15), t: np.arange(9)}), lambda: b.score({t: np.arange(20), s: [1]}),
                 lambda: b.verify({s: (1, np.arange(18)), t: (2, [3])})):
        b.left = left
        with pytest.raises(d.Dispatch):
            call()
        assert b.pool.free == free and [b.length(s), b.length(t)] == lens
    b.left = 1 << 30
    b.step({s: [7]})
    assert b.passes[-1]["kv_len"][0] == lens[0] + 1 and b.length(s) == lens[0] + 1
    b.close(s), b.close(t)
    b.share_prefix([])
    assert b.pool.free == 16


def test_a_prompt_that_does_not_fit_leaves_the_shared_one():
    """Refused before anything of it has run; one whose passes fail is gone,
    as is the old one, whose pages it may have taken."""
    b = decoder(Failing, num_pages=4)
    b.share_prefix(np.arange(20))
    n = len(b.passes)
    with pytest.raises(d.BufferSize):
        b.share_prefix(np.arange(65))
    assert b.prefix_len == 20 and b.pool.free == 2 and len(b.passes) == n
    b.share_prefix(np.arange(64))  # (with the old one's pages)
    assert b.prefix_len == 64 and b.pool.free == 0
    b.left = 1
    with pytest.raises(d.Dispatch):
        b.share_prefix(np.arange(20))
    assert b.prefix_len == 0 and b.pool.free == 4
    with pytest.raises(ValueError):
        b.length(b._next)


def test_refusals():
    for kw in (dict(max_seqs=0), dict(num_pages=0), dict(page_size=8), dict(page_size=48), dict(kv="bf16"),
               dict(max_rows=0), dict(max_logits=0), dict(max_top=-1), dict(max_len=0)):
        with pytest.raises(ValueError):
            decoder(**kw)
    for bad in (model(lm_fmt="f16"), model(gate="q4_0"), model(DecodeConfig(layers=1, head_dim=96))):
        with pytest.raises(ValueError):
            BatchDecoder(bad, 1, 1)
    b = decoder(max_len=40)
    s = b.open()
    for work in ({s + 1: [1]}, {s: [500]}, {s: [-1]}, {s: []}, {s: np.arange(41)}):
        for call in (b.step, b.score):
            with pytest.raises(ValueError):
                call(work)
    with pytest.raises(TypeError):
        b.step({s: [1.5]})
    with pytest.raises(ValueError):
        b.step({s: [1]}, top=5)
    with pytest.raises(ValueError):
        b.share_prefix([1])
    with pytest.raises(ValueError):
        b.length(99)
    assert b.length(s) == 0 and b.pool.free == 12 and not b.passes
    b.open(), b.open()
    with pytest.raises(d.BufferSize):
        b.open()
    b = decoder(num_pages=2)
    s, t = b.open(), b.open()
    with pytest.raises(d.BufferSize):
        b.step({s: np.arange(20), t: [1]})
    assert b.pool.free == 2 and not b.passes  # (nothing of it has run)
