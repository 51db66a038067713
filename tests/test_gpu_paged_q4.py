"""Batches over pages of 4 bits: append, rows read back, attention, against 64
bits.  What no row may see — places behind a sequence's length, pages that no
table names, later rows' positions — holds NaN; rows behind the last sequence
keep what they held."""
import numpy as np
import pytest

from paged_ref import NONE, Batch, rope64
from q4_ref import Batch4, decode, encode, step, up7
from runit_mac_amd import dispatch as d
from test_gpu_paged import HEADS, MARK, attend, check, shared_batch, spread

pytestmark = pytest.mark.gpu


def shared4(seqs, P, H, KVH, hd, ps, seed, **kw):
    """As shared_batch, over pages of 4 bits: what the first sequence's pages hold
    of the first P positions; the others' page where they end has NaN there."""
    b = Batch4([(P + k, n) for k, n in seqs], H, KVH, hd, ps, seed=seed, **kw)
    K, V = b.get(b.k, 0)[:P], b.get(b.v, 0)[:P]
    table = b.table[0, :-(-P // ps)].copy()
    keys, vals = [b.get(b.k, s) for s in range(len(seqs))], [b.get(b.v, s) for s in range(len(seqs))]
    for s in range(len(seqs)):
        n = min(P, int(b.kv[s]))
        keys[s][:n], vals[s][:n] = K[:n], V[:n]
        b.table[s, :P // ps] = NONE
        if s and P % ps and int(b.kv[s]) > P // ps * ps:
            for name in "kv":
                b.words[name][1][b.table[s, P // ps], :, :P % ps] = 0xFFFF
    return b, table, keys, vals


@pytest.mark.parametrize("H,KVH,hd", HEADS)
def test_decode_rows(ctx, H, KVH, hd):
    """One row a sequence: from a single position to several chunks, lengths at
    and around tiles and pages."""
    seqs = [(n - 1, 1) for n in (1, 2, 15, 16, 17, 63, 64, 65, 130, 700)]
    b = Batch4(seqs, H, KVH, hd, 16, seed=H + hd, one=True, spare_rows=2)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("ps", [16, 64])
def test_ragged_rows(ctx, H, KVH, hd, ps):
    """Sequences with no row, one, drafts and prompt chunks; no length at all."""
    seqs = [(0, 1), (5, 0), (40, 3), (0, 0), (0, 37), (129, 21), (300, 1), (13, 70)]
    b = Batch4(seqs, H, KVH, hd, ps, seed=H + hd + ps, spare_rows=3)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3])
def test_long_sequence(ctx, hd, new):
    """One sequence over many chunks, beside a short one."""
    b = Batch4([(8001 - new, new), (20, 1)], 4, 2, hd, 128, seed=hd, one=new == 1)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("n", [67, 200])
def test_many_sequences_in_chunks(ctx, n, one):
    seqs, _ = spread(n, (lambda i: 1) if one else (lambda i: i % 3), n)
    b = Batch4(seqs, 4, 2, 64, 16, seed=n, one=one, spare_rows=1)
    check(attend(ctx, b), *b.attention())


def test_many_sequences_among_prompt_chunks(ctx):
    seqs, at = spread(130, lambda i: (0, 1, 5, 1)[i % 4] if i not in (1, 63, 64, 128) else 40, 51)
    b = Batch4(seqs, 14, 2, 64, 16, seed=52)
    only = [int(b.start[i]) + j for i in at for j in range(int(b.new[i]))]
    ref, tol = b.attention(only=only)
    got = attend(ctx, b)
    assert np.all(np.isfinite(got))
    check(got[only], ref[only], tol[only])


@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (28, 4, 128), (14, 2, 256)])
def test_a_full_device(ctx, H, KVH, hd, new):
    """Long sequences, so many that every workgroup has tens of turns and memory
    is busy: what is read is what has come.  Against what the pages hold, read
    back row by row."""
    rng, ps, n = np.random.default_rng(hd + new), 64, 24
    kv = rng.integers(5000, 9000, n) + new
    per = -(-kv // ps)
    total, page = int(per.sum()), d.PagedBatch.page_bytes("q4", KVH, ps, hd)
    table = np.full((n, per.max()), NONE, np.uint32)
    at = 0
    for s, k in enumerate(per):
        table[s, :k] = np.arange(at, at + k)
        at += k
    pools = []
    for _ in range(2):
        raw = rng.integers(0, 256, (total * KVH, page // KVH), np.uint8)
        words = raw[:, ps * hd // 2:].view(np.uint16)  # steps of 0.02 .. 0.4, zero points of 6 .. 9
        words[:] = (np.exp(rng.uniform(np.log(0.02), np.log(0.4), words.shape)).astype(np.float16).view(np.uint16) & 0xFFF0) | \
            rng.integers(6, 10, words.shape, np.uint16)
        pools.append(ctx.buffer_from(raw))
    u = lambda a: ctx.buffer_from(np.asarray(a, np.uint32))
    start = np.arange(n + 1) * new
    q = rng.standard_normal((n * new, H, hd)).astype(np.float32)
    batch = d.PagedBatch(*pools, "q4", total, ps, KVH, hd, u(table), table.shape[1], n, u(kv), rows=n * new, row_start=u(start))
    bq, bo = ctx.buffer_from(q), ctx.new_buffer(4 * q.size)
    outs = []
    for _ in range(3):
        d.paged_attention_f32(ctx, batch, bq, bo, H)
        ctx.flush()
        outs.append(bo.read(np.float32).reshape(q.shape))
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])
    for s in (0, 7, n - 1):
        L = int(kv[s])
        one = d.PagedBatch(*pools, "q4", total, ps, KVH, hd, u(table[s]), table.shape[1], 1, u([L]), rows=L, row_start=u([0, L]))
        back = [ctx.new_buffer(4 * L * KVH * hd) for _ in range(2)]
        d.paged_gather_f32(ctx, one, *back)
        ctx.flush()
        K, V = (b.read(np.float32).reshape(L, KVH, hd).astype(np.float64) for b in back)
        for i in {0, new - 1}:
            r, seen = s * new + i, L - new + i + 1
            for h in range(0, H, 5):
                k, v, x = K[:seen, h * KVH // H], V[:seen, h * KVH // H], q[r, h].astype(np.float64)
                sc = k @ x / np.sqrt(hd)
                w = np.exp(sc - sc.max())
                mag = (np.abs(k) @ np.abs(x)).max() / np.sqrt(hd)
                tol = w @ np.abs(v) / w.sum() * (2 * (hd + 16) * mag + seen + 64) * 2.0 ** -24
                tol += seen * np.abs(v).max(0) * w.max() / w.sum() * 2.0 ** -37
                assert np.all(np.abs(outs[0][r, h] - w @ v / w.sum()) <= tol), (s, i, h)


@pytest.mark.parametrize("H,KVH,hd", [(71, 1, 64), (80, 2, 128), (130, 1, 64)])
@pytest.mark.parametrize("P", [0, 70])
def test_many_heads_of_a_group(ctx, H, KVH, hd, P):
    seqs = [(0, 1), (16, 1), (200, 1), (1900, 1)]
    if P:
        b, table, *kv = shared4(seqs, P, H, KVH, hd, 16, seed=H, one=True)
    else:
        b, table, kv = Batch4(seqs, H, KVH, hd, 16, seed=H, one=True), None, []
    check(attend(ctx, b, shared=(table, P) if P else None), *b.attention(*kv))


@pytest.mark.parametrize("new", [1, 40])
def test_page_stride(ctx, new):
    b = Batch4([(100, 1), (30, new)], 14, 2, 64, 32, seed=5, gap=4096 + 16)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("new", [3, 40])
def test_pages_behind_four_billion_bytes(ctx, new):
    """The same bytes as from a small pool, appended, read back and attended."""
    H, KVH, hd, ps, far = 14, 2, 64, 16, 2 ** 32 + 64
    b = Batch4([(50, new)], H, KVH, hd, ps, seed=34)
    rng = np.random.default_rng(35)
    kv = [ctx.buffer_from(rng.standard_normal((new, KVH, hd)).astype(np.float32)) for _ in range(2)]
    raw, outs = {x: b.bytes_of(x) for x in "kv"}, []
    page, end = raw["k"].shape[1], (50 + new - 1) // ps
    first, last = b.table[0, 0], b.table[0, end]
    table = np.full(b.table.size, NONE, np.uint32)
    table[0], table[end] = 0, 1  # the sequence's other pages are none
    for stride in (page, far):
        pools = [ctx.new_buffer(stride + page) for _ in range(2)]
        for pool, x in zip(pools, "kv"):
            pool.write(raw[x][first])
            pool.write(raw[x][last], stride)
        batch = d.PagedBatch(*pools, "q4", 2, ps, KVH, hd, ctx.buffer_from(table), table.size, 1,
                             ctx.buffer_from(b.kv.astype(np.uint32)), rows=new,
                             row_start=ctx.buffer_from(b.start.astype(np.uint32)), page_stride=stride)
        q, o = ctx.buffer_from(b.q[:new]), ctx.new_buffer(4 * new * H * hd)
        back = [ctx.new_buffer(4 * new * KVH * hd) for _ in range(2)]
        d.rope_kv_append_paged_f32(ctx, batch, q, *kv, q, H, 1e6)
        d.paged_attention_f32(ctx, batch, q, o, H)
        d.paged_gather_f32(ctx, batch, *back)
        ctx.flush()
        outs.append(np.concatenate([x.read(np.float32) for x in (o, *back)]))
        for x in pools:
            x.free()
    assert np.all(np.isfinite(outs[0])) and np.array_equal(*outs)


@pytest.mark.parametrize("new", [2, 40])
def test_a_page_of_more_than_four_billion_bytes(ctx, new):
    """Rows behind a prefix that has no pages, at the end of a page of 2^26 positions
    of 256 elements."""
    H, KVH, hd, ps = 2, 1, 256, 2 ** 26
    P, L = ps - 96, ps - 5
    rng = np.random.default_rng(new)
    u = lambda *a: ctx.buffer_from(np.array(a, np.uint32))
    pools = [ctx.new_buffer(d.PagedBatch.page_bytes("q4", KVH, ps, hd)) for _ in range(2)]
    q = rng.standard_normal((L - P, H, hd)).astype(np.float32)
    k, v = (rng.standard_normal((L - P, KVH, hd)).astype(np.float32) for _ in range(2))
    rows = L - P  # (all are stored, the last `new` attend)
    batch = d.PagedBatch(*pools, "q4", 1, ps, KVH, hd, u(0), 1, 1, u(L), rows=rows, row_start=u(0, rows))
    bo, back = ctx.new_buffer(q.nbytes), [ctx.new_buffer(k.nbytes) for _ in range(2)]
    d.rope_kv_append_paged_f32(ctx, batch, ctx.buffer_from(q), ctx.buffer_from(k), ctx.buffer_from(v), bo, H, 1e6)
    d.paged_gather_f32(ctx, batch, *back)
    ctx.flush()
    K, V = (b.read(np.float32).reshape(k.shape) for b in back)
    pos = np.arange(P, L)
    for got, x in ((K, rope64(k, pos, 1e6)), (V, v.astype(np.float64))):
        g = x.reshape(rows, KVH, -1, 32)
        half = up7(((np.maximum(g.max(-1), 0) - np.minimum(g.min(-1), 0)) / 15)) / 2
        # (angles of 2^26 in 64 bits are off by 2^-27 at most)
        assert np.all(np.abs(got - x) <= np.repeat(half, 32, -1) + 1e-6)
    q = q[-new:]
    batch = d.PagedBatch(*pools, "q4", 1, ps, KVH, hd, u(0), 1, 1, u(L), rows=new, row_start=u(0, new))
    out = ctx.new_buffer(q.nbytes)
    d.shared_prefix_attention_f32(ctx, batch, ctx.buffer_from(q), out, H, u(NONE), P)
    ctx.flush()
    got = out.read(np.float32).reshape(q.shape)
    for i in range(new):
        seen = rows - new + i + 1
        for h in range(H):
            x = K[:seen, 0].astype(np.float64) @ q[i, h] / np.sqrt(hd)
            w = np.exp(x - x.max())
            mag = (np.abs(K[:seen, 0]) @ np.abs(q[i, h])).max() / np.sqrt(hd)
            tol = w @ np.abs(V[:seen, 0]) / w.sum() * (2 * (hd + 16) * mag + seen + 64) * 2.0 ** -24
            tol += seen * np.abs(V[:seen, 0]).max(0) * w.max() / w.sum() * 2.0 ** -37
            assert np.all(np.abs(got[i, h] - w @ V[:seen, 0].astype(np.float64) / w.sum()) <= tol), (i, h)
    for x in pools:
        x.free()


@pytest.mark.parametrize("P", [0, 64])
@pytest.mark.parametrize("new", [1, 40])
def test_two_contexts_at_once(ctx, new, P):
    """Calls of two contexts under way together give what each gives alone."""
    other = d.HipContext()

    def together():
        sides, want = [], []
        for c, seed in ((ctx, 1), (other, 2)):
            b, table, *_ = shared4([(900, new), (P + 30, 1), (2000, new)], P, 28, 4, 128, 16, seed=seed)
            want.append(attend(c, b, shared=(table, P) if P else None))
            sides.append((c, b.upload(c), c.buffer_from(b.q), c.new_buffer(b.q.nbytes), c.buffer_from(table.astype(np.uint32)), b))
        for _ in range(20):
            for c, batch, q, out, table, b in sides:
                if P:
                    d.shared_prefix_attention_f32(c, batch, q, out, 28, table, P)
                else:
                    d.paged_attention_f32(c, batch, q, out, 28)
        for (c, _, _, out, _, b), w in zip(sides, want):
            c.flush()
            assert np.array_equal(out.read(np.float32).reshape(b.q.shape)[:b.R], w)

    together()
    other.close()


def test_missing_pages(ctx):
    """Ids that are no page: their positions are not seen; a row that sees
    nothing gives zeros."""
    b = Batch4([(200, 1), (40, 3), (31, 1), (90, 60)], 14, 2, 64, 16, seed=6)
    keys = [b.get(b.k, s) for s in range(4)]
    vals = [b.get(b.v, s) for s in range(4)]
    for s, page, bad in ((0, 0, NONE), (0, 5, b.total), (1, 1, 0x80000000), (2, 0, NONE), (2, 1, NONE), (3, 3, NONE),
                         (3, 6, NONE)):
        b.table[s, page] = bad
        keys[s][page * 16:page * 16 + 16] = np.nan
    ref, tol = b.attention(keys, vals)
    got = attend(ctx, b)
    assert np.all(got[4] == 0.0)
    check(got, ref, tol)


@pytest.mark.parametrize("new", [6, 50])
def test_rows_before_the_first_position(ctx, new):
    """kv_len below a sequence's rows: those at positions below 0 see nothing."""
    b = Batch4([(0, new), (9, 2)], 14, 2, 64, 16, seed=7)
    b.kv[0] = 4
    ref, tol = b.attention()
    got = attend(ctx, b)
    assert np.all(got[:new - 4] == 0.0)
    check(got, ref, tol)


def test_length_beyond_the_table(ctx):
    b = Batch4([(60, 4)], 4, 2, 64, 16, seed=8)
    b.stride = 3  # 48 positions
    b.table = np.ascontiguousarray(b.table[:, :3])
    check(attend(ctx, b), *b.attention([b.get(b.k, 0)], [b.get(b.v, 0)]))


@pytest.mark.parametrize("H,KVH,hd,new", [(4, 2, 64, 12), (14, 2, 64, 60), (14, 2, 128, 60), (10, 1, 256, 60)])
@pytest.mark.parametrize("word", [0x7C00, 0x7E00, 0xFFFF])
def test_later_values_stay_with_the_rows_that_see_them(ctx, H, KVH, hd, new, word):
    """A group of values that is not finite, in a tile that earlier rows see in
    part: the rows that see it have it."""
    G, bad = H // KVH, 20 + new * 2 // 3
    b = Batch4([(20, new), (3, 1)], H, KVH, hd, 16, seed=9)
    b.words["v"][1][b.table[0, bad // 16], KVH - 1, bad % 16, 1] = word
    got = attend(ctx, b)
    ref, tol = b.attention()
    sees = np.zeros(got.shape, bool)
    sees[bad - 20:new, (KVH - 1) * G:, 32:64] = True
    assert not np.any(np.isfinite(got[sees]))
    check(got[~sees], ref[~sees], tol[~sees])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("kept,P", [(50, 0), (3000, 0), (0, 300)])
def test_queries_that_are_not_finite(ctx, bad, new, kept, P):
    seqs, args = [(kept, new), (9, 2)], (14, 2, 64, 16)
    if P:
        b, table, *kv = shared4(seqs, P, *args, seed=33)
    else:
        b, table, kv = Batch4(seqs, *args, seed=33), None, []
    b.q[new - 1, 3, 7] = bad
    got = attend(ctx, b, shared=(table, P) if P else None)
    assert not np.any(np.isfinite(got[new - 1, 3]))
    b.q[new - 1, 3, 7] = 0.0
    ref, tol = b.attention(*kv)
    rest = np.ones(got.shape, bool)
    rest[new - 1, 3] = False
    check(got[rest], ref[rest], tol[rest])


@pytest.mark.parametrize("hd,rows", [(64, 376), (128, 256), (256, 128)])
def test_blocks_of_long_chunks(ctx, hd, rows):
    """As many blocks as fit at once: each takes its whole sequence, of 140
    tiles, in one chunk."""
    b = Batch4([(2240 - rows, rows)], 256, 16, hd, 64, seed=hd)
    b.table[0, 33] = NONE
    keys, vals = [b.get(b.k, 0)], [b.get(b.v, 0)]
    keys[0][33 * 64:34 * 64] = np.nan
    only = [0, 1, rows // 2, rows - 1]
    ref, tol = b.attention(keys, vals, only)
    check(attend(ctx, b)[only], ref[only], tol[only])


def test_values_far_apart(ctx):
    """Large and tiny keys, values and queries: the attention of what is held."""
    b = Batch4([(150, 2), (40, 20)], 14, 2, 64, 32, seed=10)
    for name, pool in (("k", b.k), ("v", b.v)):
        c = b.cells(pool).astype(np.float64)
        c *= 2.0 ** (np.arange(32) % 9 - 4)[:, None] * np.where(np.arange(64) < 32, 2.0 ** -10, 4.0)
        b.words[name] = list(encode(c))
        b.cells(pool)[:] = decode(*b.words[name])
    b.q[::3] *= 2.0 ** 3
    b.q[1::3] *= 2.0 ** -20
    check(attend(ctx, b), *b.attention())


def test_the_largest_steps(ctx):
    """Values of almost 2^15, and steps of 2^-20."""
    for scale in (30000.0, 2.0 ** -18):
        b = Batch4([(120, 1), (9, 44)], 14, 2, 64, 16, seed=58)
        c = b.cells(b.v).astype(np.float64)
        b.words["v"] = list(encode(np.clip(c / 3, -1, 1) * scale))
        b.cells(b.v)[:] = decode(*b.words["v"])
        assert np.nanmax(np.abs(b.cells(b.v).astype(np.float64))) > 0
        check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("new", [2, 44])
@pytest.mark.parametrize("scale", [30000.0, 2.0 ** -18, 2.0 ** -15])
def test_keys_of_the_largest_and_smallest_steps(ctx, scale, new):
    """Keys below the normal numbers of f16, of almost 2^15, and queries as much the other way."""
    b = Batch4([(120, 1), (90, new)], 14, 2, 128, 16, seed=59)
    c = b.cells(b.k).astype(np.float64)
    b.words["k"] = list(encode(np.clip(c / 3, -1, 1) * scale))
    b.cells(b.k)[:] = decode(*b.words["k"])
    b.q = (b.q / np.float32(scale)).astype(np.float32)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("mag", [26, 31, 34])
@pytest.mark.parametrize("new", [1, 60])
def test_large_scores(ctx, mag, new):
    """Scores of about 2^mag log 2, each row's largest far above the others: its
    value is the output (a weight as a pair of f16, sums and the division are off by
    less than 2^-20 together)."""
    H, KVH, hd, ps = 14, 2, 64, 16
    b = Batch4([(300 - new, new)], H, KVH, hd, ps, seed=mag)
    rng = np.random.default_rng(mag)
    sign = rng.choice([-1.0, 1.0], hd)
    up, best, last = 0, [], 0
    rows = np.zeros((300, KVH, hd))
    for i in range(300):
        if i in (0, 5, 77, 150, 251, 280):  # larger than all before them
            up, last = up + 1, i
        best.append(last)
        rows[i] = (32.0 * (8 + up) if last == i else 64.0) * sign
    n, w = encode(rows)
    for i in range(300):
        at = (b.table[0, i // ps], slice(None), i % ps)
        b.words["k"][0][at], b.words["k"][1][at] = n[i], w[i]
    held = decode(n, w)
    a = 2.0 ** (mag - 8) / (1.4427 * np.sqrt(hd))
    b.q[:] = a * sign
    scores = held[:, 0] @ sign * a / np.sqrt(hd)
    assert all(scores[best[i]] - np.delete(scores[:i + 1], best[i]).max(initial=0) > 1e3 for i in range(300))
    got = attend(ctx, b)
    for i in range(new):
        at = best[300 - new + i]
        v = np.repeat(b.cells(b.v)[b.table[0, at // ps], :, at % ps].astype(np.float64), H // KVH, 0)
        check(got[i], v, np.abs(v) * 2.0 ** -20, what=i)


@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("P,ps", [(1, 16), (64, 32), (133, 16), (1000, 64)])
def test_shared_prefix(ctx, H, KVH, hd, P, ps):
    seqs = [(0, 1), (17, 1), (3, 5), (30, 0), (0, 20), (100, 1)]
    b, table, keys, vals = shared4(seqs, P, H, KVH, hd, ps, seed=P + hd, spare_rows=1)
    check(attend(ctx, b, shared=(table, P)), *b.attention(keys, vals))


@pytest.mark.parametrize("one", [False, True])
def test_shared_prefix_of_many(ctx, one):
    """Rows of 70 sequences, or of 140 with none to three, over a long prefix."""
    rng = np.random.default_rng(11)
    P = 2048 if one else 1003
    seqs = [(int(k), 1 if one else i % 4 if i < 131 else 0) for i, k in enumerate(rng.integers(0, 90, 70 if one else 140))]
    b, table, keys, vals = shared4(seqs, P, 14, 2, 64, 64 if one else 16, seed=12, one=one, spare_rows=2)
    check(attend(ctx, b, shared=(table, P)), *b.attention(keys, vals))


def test_shared_prefix_rows_inside_it(ctx):
    b, table, keys, vals = shared4([(0, 4), (5, 2)], 50, 4, 2, 64, 16, seed=13)
    b.kv[0] = 30
    keys[0], vals[0] = keys[0][:30], vals[0][:30]
    check(attend(ctx, b, shared=(table, 50)), *b.attention(keys, vals))


@pytest.mark.parametrize("new,P", [(1, 0), (40, 0), (40, 133), (1, 133)])
def test_replays(ctx, new, P):
    """Equal results call for call; a captured graph follows the lengths, with an
    eager call of another batch over the same workspace between the replays."""
    seqs, args = [(900, new), (10, 1), (333, 1)], (14, 2, 64, 16)
    if P:
        b, table, keys, vals = shared4(seqs, P, *args, seed=36)
        bt = ctx.buffer_from(table.astype(np.uint32))
        call = lambda *x: d.shared_prefix_attention_f32(ctx, *x, 14, bt, P)
    else:
        b = Batch4(seqs, *args, seed=36)
        keys, vals = [b.get(b.k, s) for s in range(3)], [b.get(b.v, s) for s in range(3)]
        call = lambda *x: d.paged_attention_f32(ctx, *x, 14)
    other = Batch4([(300, 30), (5, 9)], *args, seed=37)
    batch, bq, bo = b.upload(ctx), ctx.buffer_from(b.q), ctx.new_buffer(4 * b.q.size)
    call(batch, bq, bo)
    ctx.flush()
    first, most = bo.read(np.float32), int(b.kv[0])
    ctx.capture_begin()
    call(batch, bq, bo)
    graph = ctx.capture_end()
    for n in (most, 300, 190, most):
        b.kv[0] = n
        b.bl.write(b.kv.astype(np.uint32))
        check(attend(ctx, other), *other.attention(), what="eager")
        graph.launch()
        ctx.flush()
        got = bo.read(np.float32)
        if n == most:
            assert np.array_equal(got, first)
        ref = b.attention([keys[0][:n], *keys[1:]], [vals[0][:n], *vals[1:]])
        check(got.reshape(b.q.shape)[:b.R], *ref, what=n)


# ───────────────────────────── append, and back ─────────────────────────────

def near(got_n, got_w, x, rel):
    """Codes and words of x [...][hd], known to rel of the largest of its group:
    the step is the next of seven bits from a fifteenth of the range, the value
    within half a step."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
    s, e = (hi - lo) / 15, rel.reshape(g.shape).max(-1)
    dd = step(got_w)
    assert np.all(up7(np.maximum(s - e, 0)) <= dd) and np.all(dd <= up7(s + e))
    err = np.abs(decode(got_n, got_w) - x)
    assert np.all(err <= np.repeat(dd / 2, 32, -1) * (1 + 2.0 ** -18) + rel)


@pytest.mark.parametrize("H,KVH,hd,ps", [(14, 2, 64, 16), (28, 4, 128, 64), (3, 1, 256, 32), (80, 16, 64, 16)])
@pytest.mark.parametrize("one", [False, True])
def test_append(ctx, H, KVH, hd, ps, one):
    seqs = [(0, 1), (15, 1), (16, 1), (500, 1)] if one else [(0, 1), (9, 0), (14, 40), (0, 0), (300, 3), (31, 1)]
    b = Batch4(seqs, H, KVH, hd, ps, seed=hd + ps, one=one, spare_rows=2, gap=16)
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((b.rows, KVH, hd)).astype(np.float32) for _ in range(2))
    k[1] *= 2.0 ** -15  # steps near 2^-20
    v[0, :, :32] = np.abs(v[0, :, :32])
    v[2, :, 32:] = 0
    v[3 if one else 5, 0] *= 9000
    batch, bq = b.upload(ctx), ctx.buffer_from(b.q)
    bo = ctx.buffer_from(np.full(b.q.shape, MARK, np.float32))
    theta = 10000.0
    d.rope_kv_append_paged_f32(ctx, batch, bq, ctx.buffer_from(k), ctx.buffer_from(v), bo, H, theta)
    ctx.flush()
    got = bo.read(np.float32).reshape(b.q.shape)
    assert np.all(got[b.R:] == MARK)
    seq = np.repeat(np.arange(len(seqs)), b.new)
    pos = b.kv[seq] - b.new[seq] + np.arange(b.R) - b.start[seq]
    # the angle to 2^-24 of half a turn, its sine and cosine, two products and a sum
    bound = lambda x: np.repeat((np.abs(x[..., :hd // 2]) + np.abs(x[..., hd // 2:]))[..., None, :], 2, -2).reshape(
        x.shape) * 2.0 ** -20
    assert np.all(np.abs(got[:b.R] - rope64(b.q[:b.R], pos, theta)) <= bound(b.q[:b.R]))
    for name, x, tol in (("k", rope64(k[:b.R], pos, theta), bound(k[:b.R])),
                         ("v", v[:b.R].astype(np.float64), np.abs(v[:b.R]) * 2.0 ** -22)):
        raw, n, w = b.read(name)
        at = (b.table[seq, pos // ps], slice(None), pos % ps)
        big = np.repeat((np.abs(x.reshape(b.R, KVH, -1, 32)) <= 32768).all(-1), 32, -1)
        rows = decode(n[at], w[at])
        assert np.all(np.isnan(rows[~big])) and not np.any(np.isnan(rows[big]))
        near(n[at], np.where(np.isnan(step(w[at])), 0, w[at]), np.where(big, x, 0), np.where(big, tol, 0))
        # nothing else was written
        b.words[name][0][at], b.words[name][1][at] = n[at], w[at]
        assert np.array_equal(raw, b.bytes_of(name))
        # and back
        for dt, call in ((np.float32, d.paged_gather_f32), (np.float16, d.paged_gather_f16)):
            outs = [ctx.buffer_from(np.full((b.rows, KVH, hd), MARK, dt)) for _ in range(2)]
            call(ctx, batch, *outs)
            ctx.flush()
            back = outs["kv".index(name)].read(dt).reshape(b.rows, KVH, hd)
            assert np.array_equal(back[:b.R].astype(np.float64), rows, equal_nan=True)
            assert np.all(back[b.R:] == MARK)
    # in place
    d.rope_kv_append_paged_f32(ctx, batch, bq, ctx.buffer_from(k), ctx.buffer_from(v), bq, H, theta)
    ctx.flush()
    again = bq.read(np.float32).reshape(b.q.shape)
    assert np.array_equal(again[:b.R], got[:b.R]) and np.array_equal(again[b.R:], b.q[b.R:])


@pytest.mark.parametrize("H,KVH,hd", HEADS)
def test_append_of_many_rows(ctx, H, KVH, hd):
    """Long chunks store and rotate what their rows do a few at a time."""
    ps, seqs = 64, [(0, 900), (77, 0), (130, 1), (1000, 1200)]
    kv, new = np.array([a + n for a, n in seqs]), np.array([n for _, n in seqs])
    rng, R = np.random.default_rng(hd + H), int(new.sum())
    per = -(-kv // ps)
    table = np.full((len(seqs), per.max()), NONE, np.uint32)
    for s, ids in enumerate(np.split(rng.permutation(per.sum()), np.cumsum(per)[:-1])):
        table[s, :len(ids)] = ids
    start = np.concatenate([[0], np.cumsum(new)])
    q, k, v = (rng.standard_normal((R + 3, n, hd)).astype(np.float32) for n in (H, KVH, KVH))
    size, got = int(per.sum()) * d.PagedBatch.page_bytes("q4", KVH, ps, hd), []
    u = lambda a: ctx.buffer_from(np.asarray(a, np.uint32))
    for most in (R, 200):
        pools, out = [ctx.buffer_from(np.full(size, 0x5A, np.uint8)) for _ in range(2)], np.full_like(q, MARK)
        for at in range(0, 1200, most):
            n = np.clip(new - at, 0, most)
            rows = np.concatenate([start[s] + at + np.arange(n[s]) for s in range(len(seqs))] + [np.arange(R, R + 3)]).astype(int)
            bo = ctx.buffer_from(np.full((len(rows), H, hd), MARK, np.float32))
            batch = d.PagedBatch(*pools, "q4", int(per.sum()), ps, KVH, hd, u(table), table.shape[1], len(seqs),
                                 u(kv - new + at + n), rows=len(rows), row_start=u(np.concatenate([[0], np.cumsum(n)])))
            d.rope_kv_append_paged_f32(ctx, batch, *(ctx.buffer_from(x[rows]) for x in (q, k, v)), bo, H, 1e6)
            ctx.flush()
            out[rows] = bo.read(np.float32).reshape(len(rows), H, hd)
        got.append((out, *(p.read(np.uint8) for p in pools)))
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    assert np.all(got[0][0][R:] == MARK)


def test_append_of_what_is_not_finite(ctx):
    """The group has NaN, the others their values."""
    b = Batch4([(0, 3)], 2, 1, 64, 16, seed=3)
    v = np.random.default_rng(4).standard_normal((3, 1, 64)).astype(np.float32)
    v[0, 0, 3], v[1, 0, 40], v[2, 0, 63] = np.inf, np.nan, -40000
    batch, bq = b.upload(ctx), ctx.buffer_from(b.q)
    d.rope_kv_append_paged_f32(ctx, batch, bq, ctx.buffer_from(v), ctx.buffer_from(v), bq, 2, 1e4)
    ctx.flush()
    _, n, w = b.read("v")
    got = decode(n, w)[b.table[0, 0], 0, :3]
    bad = np.array([[1, 0], [0, 1], [0, 1]], bool).repeat(32, -1)
    assert np.all(np.isnan(got[bad])) and np.all(np.isfinite(got[~bad]))


def test_append_without_a_page(ctx):
    b = Batch4([(20, 3), (16, 4)], 4, 2, 64, 16, seed=5)
    b.table[0, 1] = NONE
    b.kv[1] = 2  # two of its four rows are before the first position
    ones = ctx.buffer_from(np.ones((b.R, 2, 64), np.float32))
    batch, bo = b.upload(ctx), ctx.new_buffer(4 * b.q.size)
    d.rope_kv_append_paged_f32(ctx, batch, ctx.buffer_from(b.q), ones, ones, bo, 4, 1e4)
    ctx.flush()
    n, w = encode(np.ones(64))
    b.words["v"][0][b.table[1, 0], :, :2], b.words["v"][1][b.table[1, 0], :, :2] = n, w
    assert np.array_equal(b.read("v")[0], b.bytes_of("v"))
    outs = [ctx.buffer_from(np.full((b.R, 2, 64), MARK, np.float32)) for _ in range(2)]
    d.paged_gather_f32(ctx, batch, *outs)
    ctx.flush()
    back = outs[1].read(np.float32).reshape(b.R, 2, 64)
    assert np.all(back[:5] == 0) and np.allclose(back[5:], decode(n, w), rtol=0, atol=0)


@pytest.mark.parametrize("f16", [False, True])
def test_rows_read_back(ctx, f16):
    """f32 and f16 pages: as they are; f16 outputs of f32 pages are rounded.
    Either output alone; rows without a place are zeros."""
    seqs = [(0, 1), (5, 0), (40, 3), (129, 21), (13, 70)]
    b = Batch(seqs, 6, 3, 128, 16, f16, seed=70, spare_rows=3, gap=8)
    b.table[3, 9] = NONE
    batch = b.upload(ctx)
    for dt, call in ((np.float32, d.paged_gather_f32), (np.float16, d.paged_gather_f16)):
        for which in ((1, 1), (1, 0), (0, 1)):
            outs = [ctx.buffer_from(np.full((b.rows, 3, 128), MARK, dt)) for _ in range(2)]
            call(ctx, batch, *(o if w else None for o, w in zip(outs, which)))
            ctx.flush()
            for o, w, pool in zip(outs, which, (b.k, b.v)):
                got = o.read(dt).reshape(b.rows, 3, 128)
                if not w:
                    assert np.all(got == MARK)
                    continue
                want = np.full(got.shape, MARK, dt)
                for s in range(len(seqs)):
                    n = int(b.new[s])
                    rows = np.nan_to_num(b.get(pool, s)[int(b.kv[s]) - n:])
                    want[b.start[s]:b.start[s + 1]] = rows.astype(b.k.dtype).astype(dt)
                assert np.array_equal(got, want)


def test_append_then_attention(ctx):
    """Decode steps over growing pages, against the same values in 64 bits."""
    H, KVH, hd, ps, theta = 14, 2, 64, 16, 1e6
    b = Batch4([(14, 1), (0, 1), (31, 1)], H, KVH, hd, ps, seed=20, one=True)
    b.table = np.arange(12, dtype=np.uint32).reshape(3, 4)[:, ::-1].copy()
    b.stride, b.total = 4, 12
    rng = np.random.default_rng(21)
    kept = [14, 0, 31]
    for name in "kv":
        c = np.full((12, KVH, ps, hd), np.nan)
        for s, n in enumerate(kept):
            for p in range(n):
                c[b.table[s, p // ps], :, p % ps] = rng.standard_normal((KVH, hd))
        b.words[name] = list(encode(c))
    batch = b.upload(ctx)
    for i in range(20):
        b.kv = np.array(kept) + i + 1
        b.bl.write(b.kv.astype(np.uint32))
        q, k, v = (rng.standard_normal((3, h, hd)).astype(np.float32) for h in (H, KVH, KVH))
        bq, bo = ctx.buffer_from(q), ctx.new_buffer(4 * q.size)
        d.rope_kv_append_paged_f32(ctx, batch, bq, ctx.buffer_from(k), ctx.buffer_from(v), bq, H, theta)
        d.paged_attention_f32(ctx, batch, bq, bo, H)
        ctx.flush()
        b.q = bq.read(np.float32).reshape(q.shape)
        pools = [decode(*b.read(x)[1:]).astype(np.float16).reshape(12, -1) for x in "kv"]
        b.k, b.v = pools
        for s in range(3):
            x = rope64(k[s:s + 1], b.kv[s:s + 1] - 1, theta)[0]
            assert np.max(np.abs(b.get(b.k, s)[-1] - x)) <= np.ptp(x, -1).max() / 15 * 0.51
        check(bo.read(np.float32).reshape(q.shape), *b.attention(), what=i)


def test_refusals(ctx):
    b = Batch4([(20, 1)], 4, 2, 64, 16, seed=30, one=True)
    q, o = ctx.buffer_from(b.q), ctx.new_buffer(4 * b.q.size)

    def refused(what, fn=None, **kw):
        batch = b.upload(ctx)
        for k, v in kw.items():
            setattr(batch, k, v)
        n = d.launch_count(ctx)
        with pytest.raises(d.Dispatch, match=what):
            (fn or (lambda bt: d.paged_attention_f32(ctx, bt, q, o, 4)))(batch)
        assert d.launch_count(ctx) == n

    refused("f16=3", f16=3)
    refused("page_stride=1160", page_stride=1160)
    refused("page_stride=1136", page_stride=1136)
    refused("page_size=8 ", page_size=8)
    refused("16-byte aligned", k_pages=b.bk.ptr + 4)
    gather = lambda *outs: lambda bt: d.paged_gather_f32(ctx, bt, *outs)
    refused("null buffer", fn=gather(None, None))
    refused("16-byte aligned", fn=gather(o.ptr + 4, None))
    refused("num_kv_heads=0", fn=gather(o, None), num_kv_heads=0)
    refused("null buffer", fn=gather(o, None), kv_len=None)
    with pytest.raises(d.Dispatch, match="null batch"):
        ctx._check(ctx.lib.rt_paged_gather_f32(ctx.handle, None, q.ptr, o.ptr))
    n = d.launch_count(ctx)
    batch = b.upload(ctx)
    batch.n_seqs = batch.rows = 0
    d.paged_gather_f16(ctx, batch, None, None)
    assert d.launch_count(ctx) == n
