"""Rules on logits (rt_adjust_logits_f32 / _f16) against 64 bits: sizes around the
vectors and segments, odd strides, lists that overlap, repeat, leave the
vocabulary or their buffer, masks, values that are not finite."""
import numpy as np
import pytest

from runit_mac_amd import dispatch as d

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


class Rules:
    """Random rules for `rows` rows of n logits; lists of up to `seen` tokens and `biases`."""

    def __init__(self, rows, n, seen=0, biases=0, masks=0, seed=0, prompt=True):
        r = self.r = np.random.default_rng(seed)
        self.rows, self.n = rows, n
        size = lambda most: np.where(r.random(rows) < 0.2, 0, r.integers(0, most + 1, rows)) if most else None
        self.tokens = self.biases = self.mask = None
        if seen:
            self.len = size(seen)
            self.len[0] = seen
            self.start = r.integers(0, seen, rows)  # (lists overlap)
            self.tokens = (n * r.random(2 * seen) ** 3).astype(np.uint32)
            self.prompt = (self.len * r.random(rows)).astype(np.int64) if prompt else np.zeros(rows, np.int64)
            self.pen = [r.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.4), (-0.2, 0.5), (-0.2, 0.7))]
        if biases:
            self.blen = size(biases)
            self.blen[0] = biases
            self.bstart = r.integers(0, biases, rows)
            self.bids = r.integers(0, n, 2 * biases).astype(np.uint32)
            self.biases = r.normal(0, 3, 2 * biases).astype(np.float32)
        if masks:
            self.mask = r.integers(0, 1 << 32, (masks, -(-n // 32) + 1), np.uint32)
            self.mask_row = r.integers(0, masks + 1, rows).astype(np.uint32)  # (the last: none)
            self.mask_row[0] = 0

    def upload(self, ctx):
        u = lambda a: ctx.buffer_from(np.asarray(a).astype(np.uint32))
        kw = {}
        if self.tokens is not None:
            p = [ctx.buffer_from(x) for x in self.pen]
            kw.update(tokens=u(self.tokens), n_tokens=self.tokens.size, token_start=u(self.start),
                      token_len=u(self.len), prompt_len=u(self.prompt) if self.prompt.any() else None,
                      repetition=p[0], frequency=p[1], presence=p[2])
        if self.biases is not None:
            kw.update(bias_ids=u(self.bids), bias=ctx.buffer_from(self.biases), n_bias=self.biases.size,
                      bias_start=u(self.bstart), bias_len=u(self.blen))
        if self.mask is not None:
            kw.update(mask=u(self.mask), mask_rows=len(self.mask), mask_row=u(self.mask_row),
                      mask_stride=self.mask.shape[1])
        return d.LogitRules(**kw)

    def apply(self, x):
        """The logits in 64 bits, what an f32 computation of them may be off by, and
        which ones a rule names."""
        y, tol, named = x.astype(np.float64), np.zeros(x.shape), np.zeros(x.shape, bool)
        n = self.n
        with np.errstate(all="ignore"):
            for r in range(self.rows):
                if self.tokens is not None:
                    ids = self.tokens[self.start[r]:self.start[r] + self.len[r]].astype(np.int64)
                    said = ids[self.prompt[r]:]
                    count = np.bincount(said[said < n], minlength=n)
                    some = np.unique(ids[ids < n])
                    rep, freq, pres = (float(p[r]) for p in self.pen)
                    v = y[r, some]
                    y[r, some] = np.where(v > 0, v / rep, v * rep)
                    # a rounding of the quotient, of the product and of each sum
                    tol[r, some] = np.abs(y[r, some]) * 3 + (np.abs(freq) * count[some] * 3 + 2 * abs(pres))
                    y[r] -= freq * count + pres * (count > 0)
                    named[r, some] = True
                if self.biases is not None:
                    ids = self.bids[self.bstart[r]:self.bstart[r] + self.blen[r]].astype(np.int64)
                    b = self.biases[self.bstart[r]:self.bstart[r] + self.blen[r]].astype(np.float64)
                    ok = ids < n
                    np.add.at(y[r], ids[ok], b[ok])
                    k = np.bincount(ids[ok], minlength=n)
                    tol[r] += np.bincount(ids[ok], weights=np.nan_to_num(np.abs(b[ok]), posinf=0), minlength=n) * (k + 1)
                    tol[r] += np.where(k, np.nan_to_num(np.abs(y[r]), posinf=0, neginf=0), 0)
                    named[r, ids[ok]] = True
                if self.mask is not None and self.mask_row[r] < len(self.mask):
                    bits = np.unpackbits(self.mask[self.mask_row[r]].view(np.uint8), bitorder="little")[:n]
                    y[r, bits == 0] = -np.inf
                    named[r, bits == 0] = True
        return y, np.nan_to_num(tol, posinf=0) * F32, named


def run(ctx, rules, x, inplace, stride=None, handle=None):
    rows, n = x.shape
    stride = stride or n
    full = np.full((rows, stride), 7.0, x.dtype)
    full[:, :n] = x
    a = ctx.buffer_from(full)
    b = a if inplace else ctx.buffer_from(np.full((rows, stride), 9.0, x.dtype))
    call = d.adjust_logits_f16 if x.dtype == np.float16 else d.adjust_logits_f32
    call(ctx, a, b, rows, n, handle or rules.upload(ctx), row_stride=stride)
    ctx.flush()
    got = b.read(x.dtype).reshape(rows, stride)
    assert np.all(got[:, n:] == (7.0 if inplace else 9.0)), "between the rows"
    if not inplace:
        assert np.array_equal(a.read(x.dtype).reshape(full.shape), full, equal_nan=True), "the logits"
    return got[:, :n]


def check(got, x, rules):
    y, tol, named = rules.apply(x)
    bits = np.uint16 if x.dtype == np.float16 else np.uint32
    assert np.array_equal(got.view(bits)[~named], x.view(bits)[~named]), "a logit that no rule names"
    g = got.astype(np.float64)
    assert np.array_equal(np.isnan(g), np.isnan(y))
    # (computed in f32: what rounds beyond its largest, 2^128 - 2^104, is infinite)
    y = np.where(np.abs(y) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, y), y)
    if x.dtype == np.float16:
        tol = tol + np.where(named, np.nan_to_num(np.abs(y), posinf=0, neginf=0), 0) * 2.0 ** -11 + 2.0 ** -25
        y = np.where(np.abs(y) >= 65520, np.copysign(np.inf, y), y)
    fine = np.isfinite(y)
    assert np.array_equal(g[~fine], y[~fine], equal_nan=True)
    bad = np.abs(g[fine] - y[fine]) > tol[fine]
    assert not bad.any(), (int(bad.sum()), float(np.abs(g[fine] - y[fine]).max()))


def logits(rows, n, f16, seed=1):
    x = np.random.default_rng(seed).normal(0, 2.5, (rows, n))
    return x.astype(np.float16 if f16 else np.float32)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("n", [1, 5, 31, 32, 33, 1000, 4095, 4096, 4097, 9001, 50001])
def test_sizes(ctx, n, inplace, f16):
    rules = Rules(4, n, 300, 40, 2, seed=n)
    x = logits(4, n, f16)
    check(run(ctx, rules, x, inplace, n + 3), x, rules)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("seen,biases,masks", [(500, 0, 0), (0, 90, 0), (0, 0, 3), (500, 0, 3), (0, 90, 3), (500, 90, 0),
                                               (1, 1, 1)])
def test_each_rule(ctx, seen, biases, masks, inplace, f16):
    rules = Rules(9, 10007, seen, biases, masks, seed=seen + biases + masks)
    x = logits(9, 10007, f16)
    check(run(ctx, rules, x, inplace), x, rules)


@pytest.mark.parametrize("f16", [False, True])
def test_a_vocabulary(ctx, f16):
    """Histories of thousands of tokens, hundreds of biases, the largest vocabulary."""
    rules = Rules(6, 152064, 9000, 400, 3, seed=2)
    x = logits(6, 152064, f16)
    check(run(ctx, rules, x, False), x, rules)
    check(run(ctx, rules, x, True), x, rules)


def test_repeated_tokens(ctx):
    """One token thousands of times, biases of one token in their order."""
    rules = Rules(2, 700, 5000, 600, 0, seed=3)
    rules.tokens[:] = np.where(rules.r.random(rules.tokens.size) < 0.9, 13, rules.tokens)
    rules.bids[:] = np.where(rules.r.random(rules.bids.size) < 0.5, 13, rules.bids)
    rules.biases[:] = rules.r.choice([1e4, -1e4, 1.0, 2.0 ** -9], rules.biases.size)
    x = logits(2, 700, False)
    first = run(ctx, rules, x, False)
    check(first, x, rules)
    a, b = rules.bstart[0], rules.blen[0]
    total = np.float32(0)
    for i, v in zip(rules.bids[a:a + b], rules.biases[a:a + b]):
        total = np.float32(total + v) if i == 13 else total
    alone = Rules(1, 700, 0, 600, 0, seed=4)
    alone.bstart, alone.blen, alone.bids, alone.biases = rules.bstart[:1], rules.blen[:1], rules.bids, rules.biases
    assert run(ctx, alone, x[:1], False)[0, 13] == np.float32(x[0, 13] + total)
    for _ in range(3):
        assert np.array_equal(run(ctx, rules, x, False), first)


def test_ids_and_lists_beyond_their_ends(ctx):
    """Ids that are no token are passed over; lists end with their buffer."""
    rules = Rules(5, 300, 50, 30, 2, seed=5)
    rules.tokens[::3] = rules.r.choice([300, 301, 0x7FFFFFFF, 0xFFFFFFFF], rules.tokens[::3].size)
    rules.bids[::4] = 0xFFFFFFFE
    rules.len[1], rules.start[1] = 4_000_000_000, 90  # (90 .. 99 are there)
    rules.blen[1], rules.bstart[1] = 0xFFFFFFFF, 59
    rules.len[2], rules.start[2] = 20, 4_000_000_000
    rules.blen[2], rules.bstart[2] = 20, 60
    rules.prompt[3] = 4_000_000_000
    rules.mask_row[:] = [0, 1, 2, 0xFFFFFFFF, 1]
    for inplace in (False, True):
        x = logits(5, 300, False)
        check(run(ctx, rules, x, inplace), x, rules)


@pytest.mark.parametrize("f16", [False, True])
def test_values_that_are_not_finite(ctx, f16):
    """Infinities and NaN stay what the formula makes of them; where a mask forbids
    them they are −inf."""
    rules = Rules(6, 500, 400, 60, 3, seed=6)
    rules.biases[::5], rules.biases[1::7] = -np.inf, np.inf
    x = logits(6, 500, f16)
    for i, v in enumerate((np.inf, -np.inf, np.nan, np.finfo(x.dtype).max, np.finfo(x.dtype).min, 0.0, -0.0)):
        x[:, i::40] = v
    for inplace in (False, True):
        check(run(ctx, rules, x, inplace), x, rules)


def test_masks_that_forbid_everything_or_nothing(ctx):
    rules = Rules(3, 4100, 0, 0, 2, seed=7)
    rules.mask[0], rules.mask[1] = 0, 0xFFFFFFFF
    rules.mask_row[:] = [0, 1, 2]
    for inplace in (False, True):
        x = logits(3, 4100, False)
        got = run(ctx, rules, x, inplace)
        assert np.all(got[0] == -np.inf) and np.array_equal(got[1:], x[1:])


def test_without_rules(ctx):
    """No rule: a copy; in place nothing at all."""
    x = logits(3, 777, False)
    assert np.array_equal(run(ctx, None, x, False, handle=d.LogitRules()), x)
    n = d.launch_count(ctx)
    assert np.array_equal(run(ctx, None, x, True, handle=d.LogitRules()), x)
    assert d.launch_count(ctx) == n


def test_penalties_alone(ctx):
    """Lists without penalties change nothing; each penalty alone, no prompt."""
    x = logits(2, 600, False)
    for which in range(4):
        rules = Rules(2, 600, 100, seed=8, prompt=False)
        h = rules.upload(ctx)
        for i, name in enumerate(("repetition", "frequency", "presence")):
            if i != which:
                rules.pen[i][:] = 1.0 if i == 0 else 0.0
                setattr(h, name, None)
        got = run(ctx, rules, x, False, handle=h)
        check(got, x, rules)
        assert np.array_equal(got, x) == (which == 3)


def test_masks_of_their_rows(ctx):
    """Without mask_row, row r has mask r; rows behind the last have none."""
    rules = Rules(5, 1000, 0, 0, 3, seed=9)
    rules.mask_row = np.arange(5).astype(np.uint32)
    h = rules.upload(ctx)
    h.mask_row = None
    x = logits(5, 1000, True)
    check(run(ctx, rules, x, True, handle=h), x, rules)


def test_replays_follow_the_lists(ctx):
    """A captured call takes the lists' lengths and masks as they are then; the chosen
    token and its probability are those of what is left."""
    n, rows = 5000, 3
    rules = Rules(rows, n, 200, 20, 2, seed=10)
    x = logits(rows, n, False)
    h, a, b = rules.upload(ctx), ctx.buffer_from(x), ctx.new_buffer(4 * rows * n)
    lens, best, lp = ctx.buffer_from(rules.len.astype(np.uint32)), ctx.new_buffer(4 * rows), ctx.new_buffer(4 * rows)
    h.token_len = lens.ptr
    d.adjust_logits_f32(ctx, a, b, rows, n, h)
    d.argmax_rows_first_f32(ctx, b, best, rows, n)
    d.token_logprobs_f32(ctx, b, best, rows, n, lp)
    ctx.capture_begin()
    d.adjust_logits_f32(ctx, a, b, rows, n, h)
    d.argmax_rows_first_f32(ctx, b, best, rows, n)
    d.token_logprobs_f32(ctx, b, best, rows, n, lp)
    graph = ctx.capture_end()
    for size in (0, 10, 200, 50):
        rules.len[:] = size
        lens.write(rules.len.astype(np.uint32))
        run(ctx, Rules(2, 900, 30, 3, 1, seed=size), logits(2, 900, False), True)
        graph.launch()
        ctx.flush()
        got = b.read(np.float32).reshape(rows, n)
        check(got, x, rules)
        assert np.array_equal(best.read(np.uint32), got.argmax(1))
        m = got.max(1).astype(np.float64)
        assert np.allclose(lp.read(np.float32), -np.log(np.exp(got - m[:, None]).sum(1)), rtol=0, atol=1e-5)


def test_rows_behind_four_billion_bytes(ctx):
    n, stride = 900, 2 ** 30 + 7
    rules = Rules(2, n, 100, 10, 1, seed=11)
    x = logits(2, n, False)
    a = ctx.new_buffer(4 * (stride + n))
    for r in range(2):
        a.write(x[r], 4 * r * stride)
    d.adjust_logits_f32(ctx, a, a, 2, n, rules.upload(ctx), row_stride=stride)
    ctx.flush()
    check(np.stack([a.read(np.float32, n, 4 * r * stride) for r in range(2)]), x, rules)
    a.free()


def test_refusals(ctx):
    rules = Rules(2, 64, 5, 5, 2, seed=12)
    a, b = ctx.buffer_from(np.zeros(130, np.float32)), ctx.new_buffer(520)

    def refused(what, x=a, out=b, rows=2, n=64, stride=None, **kw):
        h = rules.upload(ctx)
        for k, v in kw.items():
            setattr(h, k, v)
        before = d.launch_count(ctx)
        with pytest.raises(d.Dispatch, match=what):
            d.adjust_logits_f32(ctx, x, out, rows, n, h, row_stride=stride)
        assert d.launch_count(ctx) == before

    refused("null buffer", x=None)
    refused("null buffer", out=None)
    refused("misaligned", x=a.ptr + 2)
    refused("n=0", n=0)
    refused("row_stride=63", stride=63)
    refused("row_stride", stride=1 << 41)
    refused("rows=65536", rows=65536)
    refused("too many", out=a, rows=65535, n=600_000, mask_rows=0)
    refused("overlaps", out=a.ptr + 4)
    refused("overlaps", out=a.ptr + 4 * 127)
    refused("tokens in no list", tokens=None)
    refused("tokens in no list", token_len=None)
    refused("biases in no list", bias=None)
    refused("2 masks", mask=None)
    refused("2 masks", mask_stride=1)
    with pytest.raises(d.Dispatch, match="null rules"):
        ctx._check(ctx.lib.rt_adjust_logits_f32(ctx.handle, a.ptr, b.ptr, 2, 64, 64, None))
    n = d.launch_count(ctx)
    d.adjust_logits_f32(ctx, None, None, 0, 64, rules.upload(ctx))
    assert d.launch_count(ctx) == n


@pytest.mark.parametrize("n", [0xFFFF0001, 0xFFFFFFFF, 1 << 32, 1 << 40])
def test_lists_of_almost_32_bits(ctx, n):
    """Refused: places within them are 32-bit numbers that step on by thousands."""
    buf = ctx.buffer_from(np.zeros(64, np.float32))
    before = d.launch_count(ctx)
    for kw in (dict(tokens=buf, n_tokens=n, token_start=buf, token_len=buf),
               dict(bias_ids=buf, bias=buf, n_bias=n, bias_start=buf, bias_len=buf)):
        for call in (d.adjust_logits_f32, d.adjust_logits_f16):
            with pytest.raises(d.Dispatch, match="too many"):
                call(ctx, buf, buf, 1, 16, d.LogitRules(**kw))
    assert d.launch_count(ctx) == before
    # (the most that there may be, of which the list takes four)
    x = ctx.buffer_from(np.zeros(16, np.float32))
    u = lambda *v: ctx.buffer_from(np.array(v, np.uint32))
    d.adjust_logits_f32(ctx, x, x, 1, 16, d.LogitRules(tokens=u(3, 4, 3, 9), n_tokens=0xFFFF0000, token_start=u(0), token_len=u(4),
                                                       frequency=ctx.buffer_from(np.ones(1, np.float32))))
    ctx.flush()
    assert list(x.read(np.float32)) == [0, 0, 0, -2, -1, 0, 0, 0, 0, -1, 0, 0, 0, 0, 0, 0]
