"""Batches over paged caches (rt_rope_kv_append_paged_f32,
rt_paged_attention_f32, rt_shared_prefix_attention_f32) against 64 bits.
What no row may see — places behind a sequence's length, pages that no table
names, later rows' positions — holds NaN or infinities; rows behind the last
sequence keep what they held."""
import ctypes

import numpy as np
import pytest

from paged_ref import NONE, Batch, rope64
from runit_mac_amd import dispatch as d

pytestmark = pytest.mark.gpu

MARK = 7.0


def attend(ctx, b, batch=None, shared=None):
    bo = ctx.buffer_from(np.full((b.rows, b.H, b.hd), MARK, np.float32))
    bq = ctx.buffer_from(b.q)
    batch = batch or b.upload(ctx)
    if shared is None:
        d.paged_attention_f32(ctx, batch, bq, bo, b.H)
    else:
        table, n = shared
        d.shared_prefix_attention_f32(ctx, batch, bq, bo, b.H, ctx.buffer_from(table.astype(np.uint32)), n)
    ctx.flush()
    got = bo.read(np.float32).reshape(b.rows, b.H, b.hd)
    assert np.all(got[b.R:] == MARK), "rows behind the last sequence"
    return got[:b.R]


def check(got, ref, tol, what=""):
    err = np.abs(got - ref)
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.nanmax(err)),
                           float(tol.min()))


HEADS = [(14, 2, 64), (28, 4, 128), (3, 3, 64), (10, 1, 256), (40, 2, 64)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,KVH,hd", HEADS)
def test_decode_rows(ctx, H, KVH, hd, f16):
    """One row a sequence: from a single position to several chunks, lengths at
    and around tiles and pages."""
    seqs = [(n - 1, 1) for n in (1, 2, 15, 16, 17, 63, 64, 65, 130, 700)]
    b = Batch(seqs, H, KVH, hd, 16, f16, seed=H + hd, one=True, spare_rows=2)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("ps", [16, 64])
def test_ragged_rows(ctx, H, KVH, hd, ps, f16):
    """Sequences with no row, one, drafts and prompt chunks; no length at all."""
    seqs = [(0, 1), (5, 0), (40, 3), (0, 0), (0, 37), (129, 21), (300, 1), (13, 70)]
    b = Batch(seqs, H, KVH, hd, ps, f16, seed=H + hd + ps, spare_rows=3)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_long_sequence(ctx, hd, f16):
    """One sequence over many chunks, beside a short one."""
    b = Batch([(8000, 1), (20, 1)], 4, 2, hd, 128, f16, seed=hd, one=True)
    check(attend(ctx, b), *b.attention())


def test_many_sequences(ctx):
    """More sequences than a wave has lanes, and than there are workgroups."""
    rng = np.random.default_rng(3)
    seqs = [(int(rng.integers(0, 40)), int(rng.integers(0, 3))) for _ in range(700)]
    b = Batch(seqs, 2, 1, 64, 16, seed=4)
    check(attend(ctx, b), *b.attention())


def spread(n, rows, seed):
    """n sequences of up to 60 positions, but for long ones before, at and
    behind every 64th; rows(i) new ones each."""
    rng = np.random.default_rng(seed)
    kept = rng.integers(0, 60, n)
    for i, k in ((0, 1100), (62, 1500), (63, 900), (64, 2300), (n - 3, 3900), (n - 1, 1700)):
        kept[i] = k
    return [(int(kept[i]), rows(i)) for i in range(n)], [0, 1, 62, 63, 64, n - 3, n - 2, n - 1]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("n", [67, 130, 200])
def test_many_sequences_in_chunks(ctx, n, one, f16):
    """Long sequences on both sides of the 64th: their chunks' jobs, parts and
    arrivals follow those of all sequences before them."""
    seqs, _ = spread(n, (lambda i: 1) if one else (lambda i: i % 3), n)
    b = Batch(seqs, 4, 2, 64, 16, f16, seed=n, one=one, spare_rows=1)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("hd", [64, 128])
def test_many_sequences_in_wide_blocks(ctx, hd):
    """The same among prompt chunks of f16 pages."""
    seqs, at = spread(130, lambda i: (0, 1, 5, 1)[i % 4] if i not in (1, 63, 64, 128) else 40, 51)
    b = Batch(seqs, 14, 2, hd, 16, True, seed=52)
    only = [int(b.start[i]) + j for i in at for j in range(int(b.new[i]))]
    ref, tol = b.attention(only=only)
    got = attend(ctx, b)
    assert np.all(np.isfinite(got))
    check(got[only], ref[only], tol[only])


@pytest.mark.parametrize("f16", [False, True])
def test_many_sequences_unsplit(ctx, f16):
    """So many KV heads and sequences that no block is split."""
    seqs, at = spread(140, lambda i: 1, 53)
    b = Batch(seqs, 32, 32, 64, 16, f16, seed=54, one=True)
    ref, tol = b.attention(only=at)
    got = attend(ctx, b)
    assert np.all(np.isfinite(got))
    check(got[at], ref[at], tol[at])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,KVH,hd", [(71, 1, 64), (80, 2, 128), (130, 1, 64)])
@pytest.mark.parametrize("P", [0, 70])
def test_many_heads_of_a_group(ctx, H, KVH, hd, P, f16):
    """One row a sequence fills a wide block, or more than one."""
    seqs = [(0, 1), (16, 1), (200, 1), (1900, 1)]
    if P:
        b, table, *kv = shared_batch(seqs, P, H, KVH, hd, 16, f16, seed=H, one=True)
    else:
        b, table, kv = Batch(seqs, H, KVH, hd, 16, f16, seed=H, one=True), None, []
    check(attend(ctx, b, shared=(table, P) if P else None), *b.attention(*kv))


@pytest.mark.parametrize("f16,new", [(False, 3), (True, 3), (True, 40)])
def test_tables_without_a_place(ctx, f16, new):
    """No table: nothing is seen or stored."""
    b = Batch([(20, new), (0, 1)], 14, 2, 64, 16, f16, seed=55)
    batch = b.upload(ctx)
    batch.table, batch.table_stride = None, 0
    assert np.all(attend(ctx, b, batch) == 0.0)
    ones = ctx.buffer_from(np.ones((b.R, 2, 64), np.float32))
    d.rope_kv_append_paged_f32(ctx, batch, ctx.buffer_from(b.q), ones, ones, ctx.new_buffer(4 * b.q.size), 14, 1e4)
    ctx.flush()
    assert np.array_equal(b.bk.read(b.k.dtype), b.k.ravel(), equal_nan=True)


@pytest.mark.parametrize("f16", [False, True])
def test_page_stride(ctx, f16):
    """Pools with other things between the pages."""
    b = Batch([(100, 1), (30, 9)], 8, 2, 64, 32, f16, seed=5, gap=4096 + 8)
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("f16,new", [(False, 3), (True, 3), (True, 40)])
def test_pages_behind_four_billion_elements(ctx, f16, new):
    """The same bytes as from a small pool, appended and read."""
    H, KVH, hd, ps, far = 14, 2, 64, 16, 2 ** 32 + 64
    b = Batch([(50, new)], H, KVH, hd, ps, f16, seed=34)
    rng = np.random.default_rng(35)
    kv = [ctx.buffer_from(rng.standard_normal((new, KVH, hd)).astype(np.float32)) for _ in range(2)]
    size, outs = b.k.dtype.itemsize, []
    end = (50 + new - 1) // ps
    first, last = b.table[0, 0], b.table[0, end]
    table = np.full(b.table.size, NONE, np.uint32)
    table[0], table[end] = 0, 1  # the sequence's other pages are none
    for stride in (b.page, far):
        pools = [ctx.new_buffer((stride + b.page) * size) for _ in range(2)]
        for pool, data in zip(pools, (b.k, b.v)):
            pool.write(data[first])
            pool.write(data[last], stride * size)
        batch = d.PagedBatch(*pools, "f16" if f16 else "f32", 2, ps, KVH, hd, ctx.buffer_from(table), table.size, 1,
                             ctx.buffer_from(b.kv.astype(np.uint32)), rows=new,
                             row_start=ctx.buffer_from(b.start.astype(np.uint32)), page_stride=stride)
        q, o = ctx.buffer_from(b.q[:new]), ctx.new_buffer(4 * new * H * hd)
        d.rope_kv_append_paged_f32(ctx, batch, q, *kv, q, H, 1e6)
        d.paged_attention_f32(ctx, batch, q, o, H)
        ctx.flush()
        outs.append(o.read(np.float32))
        for x in pools:
            x.free()
    assert np.all(np.isfinite(outs[0])) and np.array_equal(*outs)


@pytest.mark.parametrize("f16", [False, True])
def test_missing_pages(ctx, f16):
    """Ids that are no page: their positions are not seen; a row that sees
    nothing gives zeros."""
    b = Batch([(200, 1), (40, 3), (31, 1)], 14, 2, 64, 16, f16, seed=6)
    keys = [b.get(b.k, s) for s in range(3)]
    vals = [b.get(b.v, s) for s in range(3)]
    for s, page, bad in ((0, 0, NONE), (0, 5, b.total), (1, 1, 0x80000000), (2, 0, NONE), (2, 1, NONE)):
        b.table[s, page] = bad
        keys[s][page * 16:page * 16 + 16] = np.nan
    ref, tol = b.attention(keys, vals)
    got = attend(ctx, b)
    assert np.all(got[4] == 0.0)
    check(got, ref, tol)


def test_rows_before_the_first_position(ctx):
    """kv_len below a sequence's rows: those at positions below 0 see nothing."""
    b = Batch([(0, 6), (9, 2)], 4, 2, 64, 16, seed=7)
    b.kv[0] = 4
    ref, tol = b.attention()
    got = attend(ctx, b)
    assert np.all(got[:2] == 0.0)
    check(got, ref, tol)


def test_length_beyond_the_table(ctx):
    """Positions that the table has no room for are not seen."""
    b = Batch([(60, 4)], 4, 2, 64, 16, seed=8)
    b.stride = 3  # 48 positions
    b.table = np.ascontiguousarray(b.table[:, :3])
    keys, vals = [b.get(b.k, 0)], [b.get(b.v, 0)]
    check(attend(ctx, b), *b.attention(keys, vals))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_later_values_stay_with_the_rows_that_see_them(ctx, bad, f16):
    """A value that is not finite, in a tile that earlier rows see in part."""
    b = Batch([(20, 12), (3, 1)], 4, 2, 64, 16, f16, seed=9)
    b.cells(b.v)[b.table[0, 27 // 16], 1, 27 % 16, 5] = bad
    got = attend(ctx, b)
    b.cells(b.v)[b.table[0, 27 // 16], 1, 27 % 16, 5] = 0
    ref, tol = b.attention()
    sees = np.zeros(got.shape, bool)
    sees[7:12, 2:, 5] = True  # rows at positions 27 .. 31, the second KV head's
    assert np.all(np.isnan(got[sees]) if bad != bad else got[sees] == bad)
    check(got[~sees], ref[~sees], tol[~sees])


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (14, 2, 128), (10, 1, 256)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_later_values_in_wide_blocks(ctx, H, KVH, hd, bad):
    """The same where many rows' columns share the tiles."""
    G = H // KVH
    b = Batch([(20, 60), (3, 1)], H, KVH, hd, 16, True, seed=31)
    at = (b.table[0, 61 // 16], KVH - 1, 61 % 16, 5)
    b.cells(b.v)[at] = bad
    got = attend(ctx, b)
    b.cells(b.v)[at] = 0
    ref, tol = b.attention()
    sees = np.zeros(got.shape, bool)
    sees[41:60, (KVH - 1) * G:, 5] = True  # rows at positions 61 .. 79
    assert np.all(np.isnan(got[sees]) if bad != bad else got[sees] == bad)
    check(got[~sees], ref[~sees], tol[~sees])


@pytest.mark.parametrize("f16,new", [(False, 1), (False, 40), (True, 1), (True, 40)])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("kept,P", [(50, 0), (3000, 0), (0, 300)])
def test_queries_that_are_not_finite(ctx, bad, f16, new, kept, P):
    """They cost their own row and head its outputs, and no other's: in one
    chunk, in several, over a shared prefix."""
    seqs, args = [(kept, new), (9, 2)], (14, 2, 64, 16, f16)
    if P:
        b, table, *kv = shared_batch(seqs, P, *args, seed=33)
    else:
        b, table, kv = Batch(seqs, *args, seed=33), None, []
    b.q[new - 1, 3, 7] = bad
    got = attend(ctx, b, shared=(table, P) if P else None)
    assert not np.any(np.isfinite(got[new - 1, 3]))
    b.q[new - 1, 3, 7] = 0.0
    ref, tol = b.attention(*kv)
    rest = np.ones(got.shape, bool)
    rest[new - 1, 3] = False
    check(got[rest], ref[rest], tol[rest])


@pytest.mark.parametrize("hd,rows", [(64, 376), (128, 256), (256, 128)])
def test_wide_blocks_of_long_chunks(ctx, hd, rows):
    """As many blocks as fit at once: each takes its whole sequence, of 140
    tiles, in one chunk."""
    b = Batch([(2240 - rows, rows)], 256, 16, hd, 64, True, seed=hd)
    b.table[0, 33] = NONE
    keys, vals = [b.get(b.k, 0)], [b.get(b.v, 0)]
    keys[0][33 * 64:34 * 64] = np.nan
    only = [0, 1, rows // 2, rows - 1]
    ref, tol = b.attention(keys, vals, only)
    check(attend(ctx, b)[only], ref[only], tol[only])


@pytest.mark.parametrize("f16", [False, True])
def test_values_far_apart(ctx, f16):
    """A heavy weight on tiny values, a light one on the largest, large and
    tiny queries and keys."""
    b = Batch([(150, 2), (40, 20)], 8, 2, 64, 32, f16, seed=10)
    for s in range(2):
        for p in range(int(b.kv[s])):
            page, at = b.table[s, p // 32], p % 32
            b.cells(b.v)[page, :, at] *= np.float32(2.0 ** -12 if p % 7 else 2.0 ** 12)
            b.cells(b.k)[page, :, at] *= np.float32(2.0 ** (p % 5 - 3))
    b.q[::3] *= 2.0 ** 3
    b.q[1::3] *= 2.0 ** -20
    check(attend(ctx, b), *b.attention())


@pytest.mark.parametrize("f16,new", [(False, 1), (False, 5), (True, 1), (True, 40)])
@pytest.mark.parametrize("at", [70, 100])
def test_the_largest_values(ctx, at, f16, new):
    """A value of almost the type's largest where the scores have risen a
    little, in a later tile: its share of the output is no more than it."""
    b = Batch([(120 - new, new), (9, 1)], 4, 2, 64, 16, f16, seed=58)
    for s in range(2):
        n, dt = int(b.kv[s]), b.k.dtype
        K, V = np.zeros((n, 2, 64), dt), np.zeros((n, 2, 64), dt)
        if s == 0:
            K[at, :, 0] = 2.5 * np.log(2) * 8
            V[at] = 0.97 * np.finfo(dt).max * b.rng.choice([-1, 1], (2, 64))
        b.put(b.k, s, 0, K)
        b.put(b.v, s, 0, V)
    b.q[:] = 0
    b.q[:, :, 0] = 1.0
    check(attend(ctx, b), *b.attention())


def shared_batch(seqs, P, H, KVH, hd, ps, f16, seed, **kw):
    """Sequences (P + kept, new) whose first P positions are the same; the
    shared table, and own tables that hold nothing there but their last page."""
    b = Batch([(P + k, n) for k, n in seqs], H, KVH, hd, ps, f16, seed=seed, **kw)
    K, V = b.get(b.k, 0)[:P], b.get(b.v, 0)[:P]
    table = b.table[0, :-(-P // ps)].copy()
    keys, vals = [b.get(b.k, s) for s in range(len(seqs))], [b.get(b.v, s) for s in range(len(seqs))]
    for s in range(len(seqs)):
        n = min(P, int(b.kv[s]))
        keys[s][:n], vals[s][:n] = K[:n], V[:n]
        b.table[s, :P // ps] = NONE
        if s:  # what is before the shared length in the page where it ends is not read
            for pool in (b.k, b.v):
                if P % ps and int(b.kv[s]) > P // ps * ps:
                    b.cells(pool)[b.table[s, P // ps], :, :P % ps] = np.nan
    return b, table, keys, vals


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("P,ps", [(1, 16), (64, 32), (133, 16), (1000, 64)])
def test_shared_prefix(ctx, H, KVH, hd, P, ps, f16):
    seqs = [(0, 1), (17, 1), (3, 5), (30, 0), (0, 20), (100, 1)]
    b, table, keys, vals = shared_batch(seqs, P, H, KVH, hd, ps, f16, seed=P + hd, spare_rows=1)
    check(attend(ctx, b, shared=(table, P)), *b.attention(keys, vals))


@pytest.mark.parametrize("f16", [False, True])
def test_shared_prefix_wide_batch(ctx, f16):
    """One row of 70 sequences over a long prefix."""
    rng = np.random.default_rng(11)
    b, table, keys, vals = shared_batch([(int(k), 1) for k in rng.integers(0, 90, 70)], 2048, 14, 2, 64, 64, f16,
                                        seed=12, one=True)
    check(attend(ctx, b, shared=(table, 2048)), *b.attention(keys, vals))


@pytest.mark.parametrize("f16", [False, True])
def test_shared_prefix_ragged_batch(ctx, f16):
    """Rows of more than 64 sequences, some without any, over a prefix that
    ends inside a page."""
    rng = np.random.default_rng(56)
    seqs = [(int(k), i % 4 if i < 131 else 0) for i, k in enumerate(rng.integers(0, 60, 140))]
    b, table, keys, vals = shared_batch(seqs, 1003, 4, 2, 64, 16, f16, seed=57, spare_rows=2)
    check(attend(ctx, b, shared=(table, 1003)), *b.attention(keys, vals))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("mag", [26, 28, 31, 34])
@pytest.mark.parametrize("seqs,P,H,KVH,hd", [
    ([(0, 1), (16, 1), (129, 1), (3000, 1)], 0, 14, 2, 64),
    ([(300, 60), (3, 1)], 0, 14, 2, 64),
    ([(300, 60), (3, 1)], 0, 10, 1, 256),
    ([(5, 1), (40, 12), (0, 60)], 300, 28, 4, 128),
])
def test_large_scores(ctx, seqs, P, H, KVH, hd, mag, f16):
    """Scores of about 2^mag log 2, each row's largest far above the others: its
    value is the output, however the maximum itself is rounded.  A weight as a
    pair of f16 is off by at most 2^-21 of it, product, sums over waves and
    chunks and the division are less than eight roundings, 2^-21; the other
    weights are e^ of minus thousands."""
    ps, rng = 16, np.random.default_rng(mag)
    if P:
        b, table, *_ = shared_batch(seqs, P, H, KVH, hd, ps, f16, seed=mag)
    else:
        b, table = Batch(seqs, H, KVH, hd, ps, f16, seed=mag), np.zeros(0, np.uint32)
    sign = rng.choice([-1.0, 1.0], hd)
    page = lambda s, p: table[p // ps] if p < P else b.table[s, p // ps]
    shared = {0, *rng.integers(0, P, 8).tolist()} if P else set()
    best = []  # of each sequence: up to each position, the one with the largest score
    for s in range(len(seqs)):
        n, up, last = int(b.kv[s]), 0, -1
        larger = shared | {P, *rng.integers(P, n, 8).tolist()}  # than all before them
        best.append([])
        for i in range(n):
            up, last = (up + 1, i) if i in larger else (up, last)
            best[s].append(last)
            t = 0.5 + up / 64 if last == i else 0.25 * rng.random()
            if i >= P or not s:
                b.cells(b.k)[page(s, i), :, i % ps] = (256 * t * sign * rng.uniform(1, 1.01, (KVH, hd))).astype(b.k.dtype)
    a = 2.0 ** (mag - 8) / (1.4427 * np.sqrt(hd))
    b.q[:] = a * sign * rng.uniform(1, 1.01, b.q.shape)
    got = attend(ctx, b, shared=(table, P) if P else None)
    for s in range(len(seqs)):
        for i in range(int(b.new[s])):
            at = best[s][int(b.kv[s] - b.new[s]) + i]
            v = np.repeat(b.cells(b.v)[page(s, at), :, at % ps].astype(np.float64), H // KVH, 0)
            check(got[int(b.start[s]) + i], v, np.abs(v) * 2.0 ** -20, what=(s, i))


def test_shared_prefix_rows_inside_it(ctx):
    """Rows whose position is inside the shared positions see their part."""
    b, table, keys, vals = shared_batch([(0, 4), (5, 2)], 50, 4, 2, 64, 16, False, seed=13)
    b.kv[0] = 30
    keys[0], vals[0] = keys[0][:30], vals[0][:30]
    check(attend(ctx, b, shared=(table, 50)), *b.attention(keys, vals))
    b.kv[0] = 0  # an idle place of the batch
    keys[0], vals[0] = keys[0][:0], vals[0][:0]
    got = attend(ctx, b, shared=(table, 50))
    assert np.all(got[:4] == 0.0)
    check(got, *b.attention(keys, vals))


def test_shared_prefix_of_nothing_is_the_attention(ctx):
    b = Batch([(100, 1), (30, 9)], 8, 2, 64, 32, seed=14)
    a = attend(ctx, b)
    c = attend(ctx, b, shared=(b.table[0], 0))
    assert np.array_equal(a, c)


def test_attention_repeats_and_replays(ctx):
    """Equal results call for call; a captured graph follows the lengths."""
    b = Batch([(900, 1), (10, 1), (333, 1)], 14, 2, 64, 16, seed=15, one=True)
    other = Batch([(10, 1), (5, 1), (7, 1)], 14, 2, 64, 16, seed=16, one=True)
    first = attend(ctx, b)
    batch, bq = b.upload(ctx), ctx.buffer_from(b.q)
    bo = ctx.new_buffer(4 * b.q.size)
    obatch, oq, oo = other.upload(ctx), ctx.buffer_from(other.q), ctx.new_buffer(4 * other.q.size)
    graphs = []
    for args in ((batch, bq, bo), (obatch, oq, oo)):  # two graphs with one workspace
        ctx.capture_begin()
        d.paged_attention_f32(ctx, *args, 14)
        graphs.append(ctx.capture_end())
    for n in (901, 901, 64, 17, 500):
        b.kv[0] = n
        b.bl.write(b.kv.astype(np.uint32))
        graphs[1].launch()
        graphs[0].launch()
        graphs[1].launch()
        ctx.flush()
        got = bo.read(np.float32).reshape(first.shape)
        if n == 901:
            assert np.array_equal(got, first)
        check(got, *b.attention(), what=n)
        check(oo.read(np.float32).reshape(3, 14, 64), *other.attention(), what=n)


@pytest.mark.parametrize("P", [0, 133])
def test_wide_blocks_replay(ctx, P):
    """A captured call of wide blocks follows the lengths too, with an eager
    call of another batch over the same workspace between the replays."""
    seqs, args = [(700, 40), (10, 1)], (14, 2, 64, 16, True)
    if P:
        b, table, keys, vals = shared_batch(seqs, P, *args, seed=36)
        bt = ctx.buffer_from(table.astype(np.uint32))
        call = lambda *x: d.shared_prefix_attention_f32(ctx, *x, 14, bt, P)
    else:
        b = Batch(seqs, *args, seed=36)
        keys, vals = [b.get(b.k, s) for s in range(2)], [b.get(b.v, s) for s in range(2)]
        call = lambda *x: d.paged_attention_f32(ctx, *x, 14)
    other = Batch([(300, 30), (5, 9)], *args, seed=37)
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
        ref = b.attention([keys[0][:n], keys[1]], [vals[0][:n], vals[1]])
        check(got.reshape(b.q.shape)[:b.R], *ref, what=n)


# ───────────────────────────── append ─────────────────────────────

@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,KVH,hd,ps", [(14, 2, 64, 16), (28, 4, 128, 64), (3, 1, 256, 32), (80, 16, 64, 16)])
@pytest.mark.parametrize("one", [False, True])
def test_append(ctx, H, KVH, hd, ps, f16, one):
    seqs = [(0, 1), (15, 1), (16, 1), (500, 1)] if one else [(0, 1), (9, 0), (14, 40), (0, 0), (300, 3), (31, 1)]
    b = Batch(seqs, H, KVH, hd, ps, f16, seed=hd + ps, one=one, spare_rows=2, gap=8)
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((b.rows, KVH, hd)).astype(np.float32) for _ in range(2))
    dt = b.k.dtype
    for s in range(len(seqs)):  # the new rows' places hold nothing yet
        n = int(b.new[s])
        for pool in (b.k, b.v):
            b.put(pool, s, int(b.kv[s]) - n, np.full((n, KVH, hd), np.nan, dt))
    batch, bq = b.upload(ctx), ctx.buffer_from(b.q)
    bo = ctx.buffer_from(np.full(b.q.shape, MARK, np.float32))
    theta = 10000.0
    before_k, before_v = b.k.copy(), b.v.copy()
    d.rope_kv_append_paged_f32(ctx, batch, bq, ctx.buffer_from(k), ctx.buffer_from(v), bo, H, theta)
    ctx.flush()
    got = bo.read(np.float32).reshape(b.q.shape)
    gk, gv = (x.read(dt).reshape(b.k.shape) for x in (b.bk, b.bv))
    assert np.all(got[b.R:] == MARK)
    seq = np.repeat(np.arange(len(seqs)), b.new)
    pos = b.kv[seq] - b.new[seq] + np.arange(b.R) - b.start[seq]
    # the angle to 2^-24 of half a turn, its sine and cosine, two products and a sum
    bound = lambda x: np.repeat((np.abs(x[..., :hd // 2]) + np.abs(x[..., hd // 2:]))[..., None, :], 2, -2).reshape(
        x.shape) * 2.0 ** -20
    assert np.all(np.abs(got[:b.R] - rope64(b.q[:b.R], pos, theta)) <= bound(b.q[:b.R]))
    rk = rope64(k[:b.R], pos, theta)
    tol = bound(k[:b.R]) + (np.abs(rk) * 2.0 ** -11 + 2.0 ** -25 if f16 else 0)
    ck, cv = b.cells(gk), b.cells(gv)
    ek, ev = before_k.copy(), before_v.copy()
    for r in range(b.R):
        at = (b.table[seq[r], pos[r] // ps], slice(None), pos[r] % ps)
        assert np.all(np.abs(ck[at] - rk[r]) <= tol[r]), r
        assert np.array_equal(cv[at], v[r].astype(dt)), r
        b.cells(ek)[at], b.cells(ev)[at] = ck[at], cv[at]
    assert np.array_equal(gk, ek, equal_nan=True) and np.array_equal(gv, ev, equal_nan=True), "another place was written"
    # in place
    d.rope_kv_append_paged_f32(ctx, batch, bq, ctx.buffer_from(k), ctx.buffer_from(v), bq, H, theta)
    ctx.flush()
    again = bq.read(np.float32).reshape(b.q.shape)
    assert np.array_equal(again[:b.R], got[:b.R]) and np.array_equal(again[b.R:], b.q[b.R:])


def test_append_far_positions(ctx):
    """Angles of hundreds of thousands of radians."""
    b = Batch([(0, 1)], 2, 1, 128, 1024, seed=3, one=True)
    for n in (100_001, 262_144):
        batch = b.upload(ctx)
        b.bl.write(np.array([n], np.uint32))
        bo = ctx.new_buffer(4 * b.q.size)
        kv = ctx.buffer_from(np.ones((1, 1, 128), np.float32))
        d.rope_kv_append_paged_f32(ctx, batch, ctx.buffer_from(b.q), kv, kv, bo, 2, 1e6)
        ctx.flush()
        ref = rope64(b.q, np.array([n - 1]), 1e6)
        lim = np.tile(np.abs(b.q[..., :64]) + np.abs(b.q[..., 64:]), 2) * 2.0 ** -20
        assert np.all(np.abs(bo.read(np.float32).reshape(ref.shape) - ref) <= lim)
        # beyond the table: nothing was stored
        assert np.array_equal(b.bk.read(np.float32), b.k.ravel(), equal_nan=True)


def test_append_without_a_page(ctx):
    b = Batch([(20, 3), (16, 4)], 4, 2, 64, 16, seed=5)
    b.table[0, 1] = NONE
    b.kv[1] = 2  # two of its four rows are before the first position
    ones = ctx.buffer_from(np.ones((b.R, 2, 64), np.float32))
    batch, bo = b.upload(ctx), ctx.new_buffer(4 * b.q.size)
    d.rope_kv_append_paged_f32(ctx, batch, ctx.buffer_from(b.q), ones, ones, bo, 4, 1e4)
    ctx.flush()
    want = b.v.copy()
    b.cells(want)[b.table[1, 0], :, :2] = 1.0
    assert np.array_equal(b.bv.read(np.float32).reshape(want.shape), want, equal_nan=True)


# ───────────────────────────── together, refusals ─────────────────────────────

@pytest.mark.parametrize("f16", [False, True])
def test_append_then_attention(ctx, f16):
    """Decode steps: each appends a row to every sequence and attends, against
    the same from one growing reference cache."""
    H, KVH, hd, ps, theta = 14, 2, 64, 16, 1e6
    b = Batch([(14, 1), (0, 1), (31, 1)], H, KVH, hd, ps, f16, seed=20, one=True)
    b.table = np.arange(12, dtype=np.uint32).reshape(3, 4)[:, ::-1].copy()
    b.stride, b.total = 4, 12
    b.k, b.v = (np.full((12, b.page), np.nan, b.k.dtype) for _ in range(2))
    kept = [14, 0, 31]
    rng = np.random.default_rng(21)
    for s, n in enumerate(kept):
        for pool in (b.k, b.v):
            b.put(pool, s, 0, rng.standard_normal((n, KVH, hd)).astype(b.k.dtype))
    batch = b.upload(ctx)
    for step in range(20):
        b.kv = np.array(kept) + step + 1
        b.bl.write(b.kv.astype(np.uint32))
        q, k, v = (rng.standard_normal((3, h, hd)).astype(np.float32) for h in (H, KVH, KVH))
        bq, bo = ctx.buffer_from(q), ctx.new_buffer(4 * q.size)
        d.rope_kv_append_paged_f32(ctx, batch, bq, ctx.buffer_from(k), ctx.buffer_from(v), bq, H, theta)
        d.paged_attention_f32(ctx, batch, bq, bo, H)
        ctx.flush()
        b.q = bq.read(np.float32).reshape(q.shape)
        pos = b.kv - 1
        assert np.max(np.abs(b.q - rope64(q, pos, theta))) <= 2.0 ** -20 * 2 * np.abs(q).max()
        b.k, b.v = (x.read(b.k.dtype).reshape(b.k.shape) for x in (b.bk, b.bv))
        for s in range(3):
            got = b.get(b.k, s)[-1]
            assert np.max(np.abs(got - rope64(k[s:s + 1], pos[s:s + 1], theta)[0])) <= (2.0 ** -10 if f16 else 2.0 ** -18) * 8
        check(bo.read(np.float32).reshape(q.shape), *b.attention(), what=step)


def test_workspace_of_growing_calls():
    """Calls that each need a little more than the one before keep memory in
    proportion to the largest, not to the number of sizes."""
    hip = d.load_library()

    def free():
        hip.hipDeviceSynchronize()
        n, total = ctypes.c_size_t(), ctypes.c_size_t()
        assert hip.hipMemGetInfo(ctypes.byref(n), ctypes.byref(total)) == 0
        return n.value

    def taken(sizes):
        with d.HipContext() as ctx:
            b = Batch([(60, 1)] * 40, 28, 4, 128, 16, True, seed=38, one=True)
            batch, q, o = b.upload(ctx), ctx.buffer_from(b.q), ctx.new_buffer(4 * b.q.size)
            before = free()
            for n in sizes:
                batch.n_seqs = batch.rows = n
                d.shared_prefix_attention_f32(ctx, batch, q, o, 28, b.bt, 48)
            return before - free()

    once = taken([40])
    assert 0 < once and taken(range(1, 41)) <= 4 * once + (8 << 20)


def test_a_context_leaves_no_error():
    """What a context's start looks for and does not find is not reported to
    the next user of the device."""
    hip = d.load_library()  # (its dependency's symbols too)
    hip.hipGetLastError()
    with d.HipContext():
        assert hip.hipPeekAtLastError() == 0


def test_refusals(ctx):
    b = Batch([(20, 1)], 4, 2, 64, 16, seed=30, one=True)
    q, o = ctx.buffer_from(b.q), ctx.new_buffer(4 * b.q.size)

    def refused(what, fn=None, H=4, q=q, o=o, **kw):
        batch = b.upload(ctx)
        for k, v in kw.items():
            setattr(batch, k, v)
        n = d.launch_count(ctx)
        with pytest.raises(d.Dispatch, match=what):
            (fn or (lambda bt: d.paged_attention_f32(ctx, bt, q, o, H)))(batch)
        assert d.launch_count(ctx) == n

    refused("head_dim=80", head_dim=80)
    refused("not a multiple", H=3)
    refused("num_heads=0", H=0)
    refused("page_size=8 ", page_size=8)
    refused("page_size=48", page_size=48)
    refused("num_pages=0", num_pages=0)
    refused("page_stride=100", page_stride=100)
    refused("page_stride=2052", page_stride=2052)
    refused("address space", page_stride=1 << 59)
    refused("exceed 2.28", table_stride=1 << 26)
    refused("too many", rows=1 << 24)
    refused("f16=2", f16=2)
    refused("null buffer", kv_len=None)
    refused("null buffer", table=None)
    refused("16-byte aligned", k_pages=b.bk.ptr + 4)
    refused("16-byte aligned", q=q.ptr + 4)
    refused("alias", o=q)
    refused("0 rows for 1|rows for", n_seqs=5)
    refused("null buffer", fn=lambda bt: d.shared_prefix_attention_f32(ctx, bt, q, o, 4, None, 16))
    refused("shared_len=64", fn=lambda bt: d.shared_prefix_attention_f32(ctx, bt, q, o, 4, b.bt, 64))
    refused("theta", fn=lambda bt: d.rope_kv_append_paged_f32(ctx, bt, q, q, q, o, 4, -1.0))
    refused("null buffer", fn=lambda bt: d.rope_kv_append_paged_f32(ctx, bt, q, None, q, o, 4, 1e4))
    with pytest.raises(d.Dispatch, match="null batch"):
        ctx._check(ctx.lib.rt_paged_attention_f32(ctx.handle, None, q.ptr, o.ptr, 4))
    with pytest.raises(ValueError):
        d.PagedBatch(b.bk, b.bv, "bf16", 1, 16, 1, 64, b.bt, 1, 1, b.bl)
    # nothing to do: no launch
    n = d.launch_count(ctx)
    for kw in (dict(n_seqs=0), dict(rows=0, n_seqs=0)):
        batch = b.upload(ctx)
        for k, v in kw.items():
            setattr(batch, k, v)
        d.paged_attention_f32(ctx, batch, q, o, 4)
        d.rope_kv_append_paged_f32(ctx, batch, q, q, q, o, 4, 1e4)
    assert d.launch_count(ctx) == n
