"""Sequences decoded together over pages of 4 bits, forked, compacted and under
rules: what each pass stores, attends to and chooses, against 64 bits."""
import numpy as np
import pytest

import oracle_lib as ora
from paged_ref import rope64
from q4_ref import decode, encode
from runit_mac_amd import dispatch as d
from runit_mac_amd.batch import BatchDecoder, Rules
from runit_mac_amd.decode import Q4K_M, DecodeConfig, DecodeModel
from test_gpu_batch import SMALL, TINY, check_scores, host_logits

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


def held(b, s, layer):
    """The sequence's keys and values of a layer as its pages hold them, f64."""
    q, c = b._seqs[s], b.model.cfg
    n, first = q.len, b.prefix_len // b.page_size
    table = np.full((1, b.stride), 0xFFFFFFFF, np.uint32)
    table[0, :first] = b._prefix_pages[:first]
    table[0, first:first + len(q.pages)] = q.pages
    u = lambda *v: b.ctx.buffer_from(np.array(v, np.uint32))  # (the batch keeps them)
    p = b._pages[layer]
    batch = d.PagedBatch(p.k_pages, p.v_pages, b.kv, b.pool.num_pages, b.page_size, c.kv_heads, c.head_dim,
                         b.ctx.buffer_from(table), b.stride, 1, u(n), rows=n, row_start=u(0, n))
    outs = [b.ctx.new_buffer(4 * n * c.kv_dim) for _ in range(2)]
    d.paged_gather_f32(b.ctx, batch, *outs)
    b.ctx.flush()
    k, v = (o.read(np.float32).reshape(n, c.kv_heads, c.head_dim).astype(np.float64) for o in outs)
    if b.prefix_len % b.page_size:  # (the positions before its end in the page where the prefix ends are the prefix's)
        pre = np.arange(first * b.page_size, b.prefix_len)
        batch = d.PagedBatch(p.k_pages, p.v_pages, b.kv, b.pool.num_pages, b.page_size, c.kv_heads, c.head_dim,
                             u(*b._prefix_pages), len(b._prefix_pages), 1, u(b.prefix_len), rows=b.prefix_len,
                             row_start=u(0, b.prefix_len))
        d.paged_gather_f32(b.ctx, batch, *outs)
        b.ctx.flush()
        for x, o in zip((k, v), outs):
            x[pre] = o.read(np.float32, b.prefix_len * c.kv_dim).reshape(b.prefix_len, c.kv_heads, c.head_dim)[pre]
    return k, v


def last_layer(b, rows):
    c = b.model.cfg
    read = lambda name, *shape: b._read(name, rows * int(np.prod(shape)), np.float32).reshape(rows, *shape).astype(np.float64)
    return (read("q", c.heads, c.head_dim), read("k", c.kv_heads, c.head_dim), read("v", c.kv_heads, c.head_dim),
            read("att", c.heads, c.head_dim))


def check_pass(b, work):
    """The last pass's rows ({sequence: tokens}, in one pass): keys rotated and stored
    to the nearest code, and the attention over what is stored."""
    c = b.model.cfg
    rows = sum(len(t) for t in work.values())
    q, k, v, att = last_layer(b, rows)
    r, G = 0, c.heads // c.kv_heads
    for s, t in work.items():
        n, L = len(t), b.length(s)
        K, V = held(b, s, c.layers - 1)
        pos = np.arange(L - n, L)
        for got, x in ((K, rope64(k[r:r + n], pos, c.theta)), (V, v[r:r + n])):
            want = decode(*encode(x))
            g = x.reshape(*x.shape[:-1], -1, 32)
            step = np.repeat(((np.maximum(g.max(-1), 0) - np.minimum(g.min(-1), 0)) / 15), 32, -1)
            # (next to the border of two codes either is right: then off by half a step, its 64th more)
            assert np.all(np.abs(got[L - n:] - x) <= step * (0.5 + 1 / 64) + 1e-6)
            assert np.mean(got[L - n:] != want) < 0.01
        for i in range(n):
            for h in range(c.heads):
                kk, vv = K[:pos[i] + 1, h // G], V[:pos[i] + 1, h // G]
                x = kk @ q[r + i, h] / np.sqrt(c.head_dim)
                w = np.exp(x - x.max())
                mag = (np.abs(kk) @ np.abs(q[r + i, h])).max() / np.sqrt(c.head_dim)
                tol = w @ np.abs(vv) / w.sum() * (2 * (c.head_dim + 16) * mag + len(x) + 64) * F32
                tol += len(x) * np.abs(vv).max(0) * w.max() / w.sum() * 2.0 ** -37
                assert np.all(np.abs(att[r + i, h] - w @ vv / w.sum()) <= tol), (s, i, h)
        r += n


@pytest.mark.parametrize("quant,cfg_kw,page", [(None, TINY, 16), (Q4K_M, SMALL, 32)])
@pytest.mark.parametrize("prefix", [0, 37])
def test_passes_over_pages_of_four_bits(ctx, quant, cfg_kw, page, prefix):
    """Prompts, steps, drafts and forks, with and without a shared prompt that
    ends inside a page."""
    cfg = DecodeConfig(**cfg_kw)
    m = DecodeModel(ctx, cfg, seed=31, quant=quant)
    rng = np.random.default_rng(32)
    b = BatchDecoder(m, 4, 40, page, kv="q4", max_rows=128, max_top=4)
    tokens = lambda n: rng.integers(cfg.vocab, size=n)
    if prefix:
        b.share_prefix(tokens(prefix))
    s, t, u = (b.open() for _ in range(3))
    work = {s: tokens(33), t: tokens(2), u: tokens(50)}
    b.step(work)
    check_pass(b, work)
    f = b.fork(u)
    for _ in range(3):
        work = {x: tokens(1) for x in (s, t, u, f)}
        before = {x: held(b, x, 0) for x in work}
        b.step(work, top=4)
        check_pass(b, work)
        for x, (k, v) in before.items():  # what was there is what it was
            k2, v2 = held(b, x, 0)
            assert np.array_equal(k2[:-1], k) and np.array_equal(v2[:-1], v)
    base = b.length(f)
    b.verify({f: (3, [4, 5, 6])})
    assert base < b.length(f) <= base + 4
    before = {x: held(b, x, 1) for x in (t, u, f)}
    b.close(s)
    used = b.compact()
    assert used == b.pool.num_pages - b.pool.free
    assert all(p < used for x in (t, u, f) for p in b._seqs[x].pages)
    for x, kv in before.items():
        assert all(np.array_equal(a, c) for a, c in zip(held(b, x, 1), kv))
    work = {x: tokens(2) for x in (f, t, u)}
    b.step(work)
    check_pass(b, work)
    b.free(), m.free()


@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_forks_are_their_sequences(ctx, kv):
    """Each branch's scores are those of its tokens alone on the CPU reference
    model, whichever of them wrote first, behind a shared prompt too."""
    cfg = DecodeConfig(**SMALL)
    m = DecodeModel(ctx, cfg, seed=41, quant=Q4K_M)
    host = ora.HostStepModel.from_recipe(m)
    rng = np.random.default_rng(42)
    for prefix in (0, 21):
        b = BatchDecoder(m, 4, 30, 16, kv=kv, max_rows=64, max_top=4)
        common = list(rng.integers(cfg.vocab, size=prefix))
        if prefix:
            b.share_prefix(common)
        s = b.open()
        history = {s: common + list(rng.integers(cfg.vocab, size=23))}
        b.step({s: history[s][prefix:]})
        for i in range(3):
            f = b.fork(s)
            history[f] = list(history[s])
            work = {x: rng.integers(cfg.vocab, size=1 + (x + i) % 3) for x in history}
            got = b.step(work, top=4)
            if i == 1:
                b.compact()
            for x, t in work.items():
                history[x] += list(t)
                token, scores = got[x]
                assert token == scores.top_ids[0, 0]
                check_scores(scores, host_logits(host, history[x])[-1:], np.array([token]), kv)
        b.free()
    m.free()


def test_more_pages_than_a_call_copies(ctx):
    """A pool of 140,000 pages, half of them moved at once."""
    m = DecodeModel(ctx, DecodeConfig(**TINY), seed=43)
    b, n = BatchDecoder(m, 1, 140_000, 16, kv="q4", max_rows=16), 70_000
    page, p = b._pages[0].page_bytes("q4", m.cfg.kv_heads, 16, m.cfg.head_dim), b._pages[-1]
    for pool in (p.k_pages, p.v_pages):
        raw = np.random.default_rng(pool % 1000).integers(0, 256, n * page, np.uint8)
        ctx._check(ctx.lib.rt_upload(ctx.handle, pool, raw.ctypes.data, raw.nbytes))
        b._copy_pages(range(n), range(2 * n - 1, n - 1, -1))
        got = np.empty(n * page, np.uint8)
        ctx._check(ctx.lib.rt_download(ctx.handle, got.ctypes.data, pool + n * page, got.nbytes))
        assert np.array_equal(got.reshape(n, page)[::-1], raw.reshape(n, page))
    b.free(), m.free()


def test_rules_choose_the_token(ctx):
    """Penalties, biases and masks of some sequences of a step: the logits they
    leave, the token chosen from them, the scores of the logits as they are."""
    cfg = DecodeConfig(**TINY)
    m = DecodeModel(ctx, cfg, seed=51)
    rng = np.random.default_rng(52)
    b = BatchDecoder(m, 5, 30, 16, kv="q4", max_rows=64, max_logits=2, max_top=4)
    seqs = [b.open() for _ in range(5)]
    prompts = {s: rng.integers(cfg.vocab, size=9) for s in seqs}
    plain = b.step(prompts)
    again = {s: [int(plain[s])] for s in seqs}
    for s in seqs:
        b.trim(s, 8)
    last = {s: prompts[s][8:] for s in seqs}
    allowed = rng.random(cfg.vocab) < 0.01
    rules = {seqs[0]: Rules(bias={again[seqs[0]][0]: -np.inf}),
             seqs[1]: Rules(allowed=allowed, repetition=1.2),
             seqs[3]: Rules(repetition=1.5, frequency=0.7, presence=0.3, prompt_len=5, bias={3: 2.0, 7: -1.0})}
    for top in (None, 4):
        got = b.step(last, top=top, rules=rules)
        chosen = {s: g if top is None else g[0] for s, g in got.items()}
        assert chosen[seqs[0]] != again[seqs[0]][0] and allowed[chosen[seqs[1]]]
        assert chosen[seqs[2]] == again[seqs[2]][0] and chosen[seqs[4]] == again[seqs[4]][0]
        if top:
            # (logits two rows at a time: the last pair's is the fifth sequence alone)
            assert all(g[1].logprob.shape == (1,)
                       for g in got.values())
            assert got[seqs[0]][1].rank[0] >= 1 and got[seqs[0]][1].top_ids[0, 0] == again[seqs[0]][0]
        for s in seqs:
            b.trim(s, 8)
    # one sequence's logits before and after
    s = seqs[3]
    tok, _ = b.step({s: last[s]}, top=2, rules={s: rules[s]})[s]
    raw = b._read("logits", cfg.vocab, np.float32).astype(np.float64)
    after = b._rules_buf["logits"].read(np.float32, cfg.vocab).astype(np.float64)
    want, have = raw.copy(), prompts[s]
    some, count = np.unique(have), np.bincount(have[5:], minlength=cfg.vocab)
    want[some] = np.where(want[some] > 0, want[some] / 1.5, want[some] * 1.5)
    want -= 0.7 * count + 0.3 * (count > 0)
    want[[3, 7]] += [2.0, -1.0]
    named = np.union1d(some, [3, 7])
    rest = np.setdiff1d(np.arange(cfg.vocab), named)
    assert np.array_equal(after[rest], raw[rest])
    assert np.all(np.abs(after - want) <= (np.abs(want) + np.abs(raw) + 10) * 6 * F32)
    assert tok == np.flatnonzero(after == after.max())[0]
    b.free(), m.free()


def test_rules_leave_no_logit(ctx):
    """Penalties that make the one token allowed -inf: an error, and the sequences
    as they were."""
    cfg = DecodeConfig(**TINY)
    m = DecodeModel(ctx, cfg, seed=61)
    b = BatchDecoder(m, 2, 20, 16, kv="q4", max_rows=8, max_logits=1)
    s, t = b.open(), b.open()
    b.step({s: [9, 9, 9], t: [3, 4]})
    before, free = held(b, s, 1), b.pool.free
    only = Rules(allowed=np.arange(cfg.vocab) == 9, frequency=3e38)
    with pytest.raises(ValueError, match="no token"):
        b.step({s: [9, 1], t: [5]}, rules={s: only})
    assert b.length(s) == 3 and b.length(t) == 2 and b.pool.free == free
    assert all(np.array_equal(x, y) for x, y in zip(held(b, s, 1), before))
    only.frequency = 1.0
    assert b.step({s: [9, 1], t: [5]}, rules={s: only})[s] == 9
    b.free(), m.free()


@pytest.mark.parametrize("kv", ["q4", "f16"])
@pytest.mark.parametrize("turned", [False, True])
def test_forks_of_unequal_length_after_a_failure(ctx, kv, turned, monkeypatch):
    """A fork that was trimmed and its origin write to the page that both hold, and the
    call's last pass fails: both hold what they held, and go on."""
    m = DecodeModel(ctx, DecodeConfig(**TINY), seed=71)
    b = BatchDecoder(m, 2, 20, 16, kv=kv, max_rows=8)
    rng = np.random.default_rng(72)
    tokens = lambda n: rng.integers(m.cfg.vocab, size=n)
    s = b.open()
    b.step({s: tokens(28)})
    t = b.fork(s)
    b.trim(t, 20)
    before, free = {(x, i): held(b, x, i) for x in (s, t) for i in range(m.cfg.layers)}, b.pool.free
    same = lambda: all(np.array_equal(y, z[:len(y)]) for (x, i), kv in before.items() for y, z in zip(kv, held(b, x, i)))
    work = {s: tokens(3), t: tokens(10)}
    work = dict(reversed(work.items())) if turned else work
    launch, left = b._launch, [1]

    def failing(*args):
        if left[0] == 0:
            raise d.Dispatch("kernel dispatch error: none")
        left[0] -= 1
        return launch(*args)

    monkeypatch.setattr(b, "_launch", failing)
    with pytest.raises(d.Dispatch):
        b.step(work)
    assert b.length(s) == 28 and b.length(t) == 20 and b.pool.free == free and same()
    left[0] = 9
    b.step(work)
    assert b.length(s) == 31 and b.length(t) == 30 and same()
    b.free(), m.free()
