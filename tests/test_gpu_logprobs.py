"""rt_token_logprobs_f32 / _f16 against 64 bits: sizes around the vectors and
segments, odd strides, ties, infinities, NaN, token ids out of range."""
import numpy as np
import pytest

from runit_mac_amd import dispatch as d

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


def run(ctx, x, tokens, top, stride=None, extras=True):
    rows, n = len(tokens), x.shape[1] if stride is None else stride[1]
    call = d.token_logprobs_f16 if x.dtype == np.float16 else d.token_logprobs_f32
    bx, bt = ctx.buffer_from(x), ctx.buffer_from(np.asarray(tokens, np.uint32))
    lp, en = (ctx.buffer_from(np.full(rows + 1, 7.0, np.float32)) for _ in range(2))
    rk = ctx.buffer_from(np.full(rows + 1, 77, np.uint32))
    ids = ctx.buffer_from(np.full(rows * top + 1, 77, np.uint32))
    tl = ctx.buffer_from(np.full(rows * top + 1, 7.0, np.float32))
    call(ctx, bx, bt, rows, n, lp, entropy=en if extras else None, rank=rk if extras else None, top=top,
         top_ids=ids if top else None, top_logprobs=tl if top else None,
         row_stride=None if stride is None else stride[0])
    ctx.flush()
    got = [b.read(t) for b, t in ((lp, np.float32), (en, np.float32), (rk, np.uint32), (ids, np.uint32),
                                  (tl, np.float32))]
    for g in got:
        assert g[-1] in (7.0, 77), "past the last row"
    if not extras:
        assert np.all(got[1] == 7.0) and np.all(got[2] == 77)
    return got[0][:-1], got[1][:-1], got[2][:-1], got[3][:-1].reshape(rows, top), got[4][:-1].reshape(rows, top)


def check(x, tokens, top, got):
    lp, en, rk, ids, tl = got
    n = x.shape[1]
    for r, t in enumerate(tokens):
        v = x[r].astype(np.float64)
        m = v.max()
        e = np.exp(v - m)
        z = np.log(e.sum())
        p = e / e.sum()
        with np.errstate(invalid="ignore"):
            dist = np.where(p > 0, m - v, 0.0)
        # a term e^-d: the argument's roundings 4·d and 8 of its own; sums of at
        # most n / 64 + 64 terms one after the other
        rel = float(p @ (4 * dist + 8)) * F32 + (n / 64 + 64) * F32
        xt = v[t] if t < n else -np.inf
        if np.isfinite(xt):
            assert abs(lp[r] - (xt - m - z)) <= rel + 4 * F32 * (abs(xt - m) + abs(z) + 1), r
        else:
            assert lp[r] == -np.inf, r
        ent = z + p @ dist
        assert abs(en[r] - ent) <= rel * (1 + 2 * p @ dist) + float(p @ (dist * (4 * dist + 8))) * F32 + 8 * F32 * (
            abs(z) + ent + 1), r
        assert rk[r] == np.sum(v > xt), r
        if top:
            order = np.argsort(-v, kind="stable")[:top]
            assert np.array_equal(ids[r], order), r
            want = v[order] - m - z
            fin = np.isfinite(want)
            assert np.all(np.abs(tl[r][fin] - want[fin]) <= rel + 4 * F32 * (np.abs(want[fin]) + abs(z) + 1)), r
            assert np.all(tl[r][~fin] == -np.inf)


def logits(rng, rows, n, half, std=2.5):
    x = (std * rng.standard_normal((rows, n))).astype(np.float32)
    return x.astype(np.float16) if half else x


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,n,top", [
    (1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 64, 64), (5, 255, 7), (4, 257, 1), (2, 1023, 20), (1, 2049, 64),
    (7, 4095, 5), (2, 8192, 33), (3, 50001, 20), (1, 151936, 5), (40, 32007, 0), (1100, 300, 3), (600, 9001, 2),
])
def test_sizes(ctx, rows, n, top, half):
    rng = np.random.default_rng(rows + n)
    x = logits(rng, rows, n, half)
    tokens = rng.integers(0, n, rows)
    tokens[::3] = x[::3].argmax(1)
    check(x, tokens, top, run(ctx, x, tokens, top))


@pytest.mark.parametrize("half", [False, True])
def test_strides(ctx, half):
    """Rows apart by an odd number, what is between them NaN; starts at odd places."""
    rng = np.random.default_rng(2)
    rows, n, st = 5, 5003, 5017
    x = logits(rng, rows, n, half)
    buf = np.full(rows * st, np.nan, x.dtype)
    for r in range(rows):
        buf[r * st:r * st + n] = x[r]
    tokens = rng.integers(0, n, rows)
    check(x, tokens, 9, run(ctx, buf.reshape(1, -1), tokens, 9, stride=(st, n)))


@pytest.mark.parametrize("half", [False, True])
def test_rows_four_billion_apart(ctx, half):
    """A row behind 2^32 elements is the same row as one beside it."""
    n, far, dt = 5003, 2 ** 32 + 5, np.float16 if half else np.float32
    x = np.random.default_rng(40).standard_normal((2, n)).astype(dt)
    tok, outs = ctx.buffer_from(np.array([7, 4000], np.uint32)), []
    for stride in (n, far):
        buf = ctx.new_buffer((stride + n) * x.itemsize)
        buf.write(x[0])
        buf.write(x[1], stride * x.itemsize)
        lp, ids, tops = ctx.new_buffer(8), ctx.new_buffer(24), ctx.new_buffer(24)
        (d.token_logprobs_f16 if half else d.token_logprobs_f32)(ctx, buf, tok, 2, n, lp, top=3, top_ids=ids,
                                                                  top_logprobs=tops, row_stride=stride)
        ctx.flush()
        outs.append([lp.read(np.float32), ids.read(np.uint32), tops.read(np.float32)])
        buf.free()
    assert all(np.array_equal(*p) for p in zip(*outs)) and np.all(np.isfinite(outs[0][0]))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n", [700, 20001])
def test_ties(ctx, n, half):
    """Few different values, both zeros among them: equal logits go by the lower id."""
    rng = np.random.default_rng(n)
    x = rng.integers(-2, 3, (4, n)).astype(np.float16 if half else np.float32) * 0.5
    x[x == 0] *= np.where(rng.random(np.sum(x == 0)) < 0.5, 1, -1).astype(x.dtype)
    x[1] = 3.25  # all alike
    tokens = rng.integers(0, n, 4)
    check(x, tokens, 64, run(ctx, x, tokens, 64))


@pytest.mark.parametrize("order", [1, -1])
def test_sorted_rows(ctx, order):
    """Every value, or none, beats those before it."""
    x = np.linspace(-30, 5, 30011, dtype=np.float32)[::order].reshape(1, -1).copy()
    check(x, [17], 50, run(ctx, x, [17], 50))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n", [900, 20001])
def test_masked_vocabulary(ctx, n, half):
    """Most logits −inf: probability 0, last in the order, by id; and the
    type's lowest value in their place."""
    rng = np.random.default_rng(n + 1)
    x = logits(rng, 3, n, half)
    x[0, rng.random(n) < 0.9] = -np.inf
    x[1, 3:] = -np.inf
    x[2, rng.random(n) < 0.9] = np.finfo(x.dtype).min
    tokens = [int(np.flatnonzero(np.isinf(x[0]))[0]), 1, int(x[2].argmax())]
    check(x, tokens, 10, run(ctx, x, tokens, 10))


def test_confident_and_far(ctx):
    """One logit far above the others; all far from zero; far below."""
    rng = np.random.default_rng(5)
    x = logits(rng, 4, 30000, False, 1.0)
    x[0, 777] = 60.0
    x[1] += 10000.0
    x[2] -= 10000.0
    x[3] *= 1e30
    tokens = [777, 3, 4, int(x[3].argmax())]
    check(x, tokens, 3, run(ctx, x, tokens, 3))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n", [500, 20001])
def test_rows_without_a_distribution(ctx, n, half):
    rng = np.random.default_rng(6)
    x = logits(rng, 4, n, half)
    x[0, n // 2] = np.nan
    x[1, n // 3] = np.inf
    x[2] = -np.inf
    tokens = [1, n // 3, 5, 6]
    lp, en, rk, ids, tl = run(ctx, x, tokens, 4)
    assert np.all(np.isnan(lp[:3])) and np.all(np.isnan(en[:3])) and np.all(np.isnan(tl[:3]))
    order = np.argsort(-np.where(np.isnan(x[0]), -np.inf, x[0]).astype(np.float64), kind="stable")[:4]
    assert np.array_equal(ids[0], order) and ids[1, 0] == n // 3 and rk[1] == 0
    assert np.array_equal(ids[2], [0, 1, 2, 3])
    check(x[3:], tokens[3:], 4, (lp[3:], en[3:], rk[3:], ids[3:], tl[3:]))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n,top", [(500, 0), (500, 4), (20001, 0), (20001, 4)])
def test_tokens_that_are_nan(ctx, n, top, half):
    """A given token whose own logit is NaN ranks as one at -inf does: below
    every logit above -inf, in one segment and in several."""
    rng = np.random.default_rng(41)
    x = logits(rng, 3, n, half)
    x[0, 7] = np.nan
    x[1, n - 1], x[1, : n // 2] = np.nan, -np.inf
    x[2, [3, n // 2]] = np.nan, np.inf
    tokens = [7, n - 1, 3]
    lp, en, rk, _, tl = run(ctx, x, tokens, top)
    assert np.array_equal(rk, (x > -np.inf).sum(1))
    assert np.all(np.isnan(lp)) and np.all(np.isnan(en)) and np.all(np.isnan(tl))


def test_tokens_out_of_range(ctx):
    rng = np.random.default_rng(7)
    x = logits(rng, 3, 5000, False)
    tokens = np.array([5000, 0xFFFFFFFF, 4999])
    check(x, tokens, 2, run(ctx, x, tokens, 2))


def test_without_extras_and_repeats(ctx):
    rng = np.random.default_rng(8)
    x = logits(rng, 2, 152064, False)
    a = run(ctx, x, [5, 6], 8)
    b = run(ctx, x, [5, 6], 8)
    c = run(ctx, x, [5, 6], 0, extras=False)
    assert all(np.array_equal(p, q) for p, q in zip(a, b)) and np.array_equal(a[0], c[0])


def test_replay(ctx):
    """A captured call follows logits and tokens; two graphs share the workspace."""
    rng = np.random.default_rng(9)
    n, top = 50001, 6
    sets = []
    for rows in (2, 5):
        x = logits(rng, rows, n, False)
        bx, bt = ctx.buffer_from(x), ctx.buffer_from(np.zeros(rows, np.uint32))
        outs = [ctx.new_buffer(4 * rows * k) for k in (1, 1, 1, top, top)]
        args = (bx, bt, rows, n, outs[0])
        kw = dict(entropy=outs[1], rank=outs[2], top=top, top_ids=outs[3], top_logprobs=outs[4])
        d.token_logprobs_f32(ctx, *args, **kw)
        ctx.flush()
        sets.append([x, bx, bt, outs, args, kw])
    graphs = []
    for s in sets:
        ctx.capture_begin()
        d.token_logprobs_f32(ctx, *s[4], **s[5])
        graphs.append(ctx.capture_end())
    for turn in range(4):
        toks = []
        for s in sets:
            s[0] = logits(rng, s[0].shape[0], n, False)
            toks.append(rng.integers(0, n, s[0].shape[0]))
            s[1].write(s[0])
            s[2].write(toks[-1].astype(np.uint32))
        for g in graphs:
            g.launch()
        ctx.flush()
        for s, t in zip(sets, toks):
            rows = len(t)
            got = [o.read(k) for o, k in zip(s[3], (np.float32, np.float32, np.uint32, np.uint32, np.float32))]
            check(s[0], t, top, (*got[:3], got[3].reshape(rows, top), got[4].reshape(rows, top)))


def test_refusals(ctx):
    x, t, o = ctx.new_buffer(4000), ctx.new_buffer(4), ctx.new_buffer(4000)

    def refused(what, *args, **kw):
        n = d.launch_count(ctx)
        with pytest.raises(d.Dispatch, match=what):
            d.token_logprobs_f32(ctx, *args, **kw)
        assert d.launch_count(ctx) == n

    refused("n=0", x, t, 1, 0, o)
    refused("row_stride=99", x, t, 1, 100, o, row_stride=99)
    refused("65535", x, t, 65536, 10, o)
    refused("top=65", x, t, 1, 100, o, top=65, top_ids=o, top_logprobs=o)
    refused("top=11", x, t, 1, 10, o, top=11, top_ids=o, top_logprobs=o)
    refused("null buffer", None, t, 1, 10, o)
    refused("null buffer", x, None, 1, 10, o)
    refused("null buffer", x, t, 1, 10, None)
    refused("null buffer", x, t, 1, 10, o, top=2, top_ids=o)
    refused("misaligned", x.ptr + 2, t, 1, 10, o)
    n = d.launch_count(ctx)
    d.token_logprobs_f32(ctx, x, t, 0, 10, o)
    assert d.launch_count(ctx) == n
