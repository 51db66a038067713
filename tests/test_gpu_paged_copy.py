"""Pages copied through pools (rt_paged_copy) against the same on the host, one after
another: forks, chains, cycles, pages written twice, ids that are none."""
import numpy as np
import pytest

from runit_mac_amd import dispatch as d

pytestmark = pytest.mark.gpu

#       type   KVH, page size, head size
SHAPES = [("q4", 1, 16, 64), ("q4", 4, 64, 128), ("f16", 2, 64, 64), ("f32", 3, 32, 256), ("f32", 8, 128, 128)]


class Pools:
    def __init__(self, ctx, kind, KVH, ps, hd, pages, layers, gap=0, seed=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.pages = ctx, pages
        self.page = d.PagedBatch.page_bytes(kind, KVH, ps, hd)
        el = {"f32": 4, "f16": 2, "q4": 1}[kind]
        self.host = rng.integers(0, 256, (2 * layers, pages, self.page + gap), np.uint8)
        self.bufs = [ctx.buffer_from(h) for h in self.host]
        self.batches = [d.PagedBatch(k, v, kind, pages, ps, KVH, hd, None, 0, 0, None,
                                     page_stride=(self.page + gap) // el if gap else 0)
                        for k, v in zip(self.bufs[::2], self.bufs[1::2])]

    def copy(self, src, dst):
        src, dst = np.asarray(src, np.uint32), np.asarray(dst, np.uint32)
        for s, t in zip(src, dst):
            if s < self.pages and t < self.pages:
                self.host[:, t, :self.page] = self.host[:, s, :self.page]
        d.paged_copy(self.ctx, self.batches, self.ctx.buffer_from(src), self.ctx.buffer_from(dst), len(src))
        self.ctx.flush()

    def check(self):
        for h, b in zip(self.host, self.bufs):
            assert np.array_equal(b.read(np.uint8).reshape(h.shape), h)


LISTS = {
    "fork": ([3, 3, 5, 3], [7, 8, 9, 10]),
    "one": ([0], [11]),
    "itself": ([4, 4], [4, 6]),
    "chain": ([0, 1, 2, 3], [1, 2, 3, 4]),
    "chain back": ([1, 2, 3, 4], [0, 1, 2, 3]),
    "swap": ([0, 1, 9, 5], [9, 0, 1, 6]),
    "twice": ([0, 1, 2], [5, 5, 6]),
    "late": ([0, 1, 2, 7, 8], [3, 4, 5, 8, 9]),
    "none": ([0xFFFFFFFF, 2, 12, 1], [5, 12, 6, 7]),
    "none in a chain": ([0, 0xFFFFFFFF, 6], [6, 6, 0x80000000]),
}


@pytest.mark.parametrize("kind,KVH,ps,hd", SHAPES)
@pytest.mark.parametrize("name", LISTS)
def test_lists(ctx, name, kind, KVH, ps, hd):
    p = Pools(ctx, kind, KVH, ps, hd, 12, 2, gap=32 if name in ("fork", "chain") else 0, seed=hd)
    p.copy(*LISTS[name])
    p.check()
    if name == "fork":
        p.copy(*LISTS["chain"])
        p.check()


@pytest.mark.parametrize("pages,n", [(40, 700), (3000, 900), (5000, 1100)])
def test_long_lists(ctx, pages, n):
    """More entries than threads, some of them meeting others, or almost all."""
    rng = np.random.default_rng(n)
    p = Pools(ctx, "q4", 1, 16, 64, pages, 2, seed=n)
    p.copy(rng.integers(0, pages + 2, n), rng.integers(0, pages + 2, n))
    p.check()


@pytest.mark.parametrize("shift", [0, 1])
def test_lists_of_several_launches(ctx, shift):
    """Thousands of entries: each page once, then every page one place on (a chain
    through all of them)."""
    n = 9001
    p = Pools(ctx, "q4", 1, 16, 64, 2 * n, 1, seed=shift)
    ids = np.random.default_rng(shift).permutation(2 * n)
    p.copy(*((ids[:n], ids[n:]) if not shift else (np.arange(n), np.arange(n) + 1)))
    p.check()


def test_more_pools_than_a_launch_takes(ctx):
    p = Pools(ctx, "q4", 1, 16, 64, 9, 150, seed=3)
    n = d.launch_count(ctx)
    p.copy([0, 1, 1], [1, 2, 5])
    assert d.launch_count(ctx) == n + 2
    p.check()


def test_pages_behind_four_billion_bytes(ctx):
    stride, page = 2 ** 32 + 256, d.PagedBatch.page_bytes("f16", 1, 16, 64)
    bufs = [ctx.new_buffer(stride + page) for _ in range(2)]
    rows = [np.random.default_rng(i).integers(0, 256, page, np.uint8) for i in range(2)]
    for b, r in zip(bufs, rows):
        b.write(r)
    batch = d.PagedBatch(*bufs, "f16", 2, 16, 1, 64, None, 0, 0, None, page_stride=stride // 2)
    d.paged_copy(ctx, batch, ctx.buffer_from(np.zeros(1, np.uint32)), ctx.buffer_from(np.ones(1, np.uint32)), 1)
    ctx.flush()
    for b, r in zip(bufs, rows):
        assert np.array_equal(b.read(np.uint8, page, stride), r)
        b.free()


def test_replays_follow_the_lists(ctx):
    p = Pools(ctx, "f16", 2, 16, 64, 20, 3, seed=5)
    src, dst = ctx.buffer_from(np.zeros(3, np.uint32)), ctx.buffer_from(np.zeros(3, np.uint32))
    ctx.capture_begin()
    d.paged_copy(ctx, d.PagedBatch.array(p.batches), src, dst, 3)
    graph = ctx.capture_end()
    for s, t in (([1, 2, 3], [4, 5, 6]), ([4, 5, 9], [9, 4, 5]), ([0, 0, 0], [7, 8, 19])):
        src.write(np.array(s, np.uint32)), dst.write(np.array(t, np.uint32))
        graph.launch()
        ctx.flush()
        for a, b in zip(s, t):
            p.host[:, b] = p.host[:, a]
        p.check()
        p.copy([10], [11])


def test_refusals(ctx):
    p = Pools(ctx, "q4", 1, 16, 64, 4, 2)
    ids = ctx.buffer_from(np.zeros(4, np.uint32))

    def refused(what, src=ids, n=1, first=True, **kw):
        batches = d.PagedBatch.array(p.batches)
        for k, v in kw.items():
            setattr(batches[0 if first else 1], k, v)
        before = d.launch_count(ctx)
        with pytest.raises(d.Dispatch, match=what):
            d.paged_copy(ctx, batches, src, ids, n)
        assert d.launch_count(ctx) == before

    refused("null buffer", src=None)
    refused("exceed 65535", n=65536)
    refused("null buffer", k_pages=None)
    refused("16-byte aligned", v_pages=p.bufs[1].ptr + 8)
    refused("page_size=8", page_size=8)
    refused("num_pages=0", num_pages=0)
    refused("f16=2", f16=2)
    refused("head_dim=80", head_dim=80)
    refused("num_kv_heads=0", num_kv_heads=0)
    refused("page_stride=100", page_stride=100)
    refused("differ from", first=False, num_pages=3)
    refused("differ from", first=False, f16=1)
    refused("pool is there twice", first=False, k_pages=p.bufs[0].ptr)
    refused("too many|pages of", n=65535, page_size=1 << 25, num_pages=1, k_pages=p.bufs[0].ptr)
    n = d.launch_count(ctx)
    d.paged_copy(ctx, [], ids, ids, 1)
    d.paged_copy(ctx, p.batches, None, None, 0)
    assert d.launch_count(ctx) == n
    p.check()


def test_pools_that_overlap(ctx):
    """Refused where their pages do; pools whose pages take turns are apart."""
    p = Pools(ctx, "q4", 1, 16, 64, 4, 1)
    src, dst = ctx.buffer_from(np.array([1], np.uint32)), ctx.buffer_from(np.array([3], np.uint32))
    page, raw = p.page, np.random.default_rng(7).integers(0, 256, (4, 2, p.page), np.uint8)
    both = ctx.buffer_from(raw)
    make = lambda at: d.PagedBatch(both.ptr, both.ptr + at, "q4", 4, 16, 1, 64, None, 0, 0, None, page_stride=2 * page)
    n = d.launch_count(ctx)
    with pytest.raises(d.Dispatch, match="overlap"):
        d.paged_copy(ctx, make(page - 16), src, dst, 1)
    assert d.launch_count(ctx) == n
    d.paged_copy(ctx, make(page), src, dst, 1)
    ctx.flush()
    raw[3] = raw[1]
    assert np.array_equal(both.read(np.uint8).reshape(raw.shape), raw)


@pytest.mark.parametrize("layers", [1, 20])
def test_pools_that_overlap_anywhere(ctx, layers):
    """Pools shifted by whole pages, or into the gaps of others that are too
    narrow, are refused; those that end where the next begins, or in wide gaps, copied."""
    page = d.PagedBatch.page_bytes("q4", 1, 16, 64)
    raw = np.random.default_rng(8).integers(0, 256, (2 * layers + 1) * 4 * 2 * page, np.uint8)
    buf = ctx.buffer_from(raw)
    ids = ctx.buffer_from(np.array([1], np.uint32)), ctx.buffer_from(np.array([3], np.uint32))

    def copy(starts, stride, pages=4):
        """The last layer's values take the last start; the others are apart from both of its pools."""
        make = lambda k, v: d.PagedBatch(buf.ptr + k, buf.ptr + v, "q4", pages, 16, 1, 64, None, 0, 0, None, page_stride=stride)
        d.paged_copy(ctx, [make(k, v) for k, v in zip(starts[::2], starts[1::2])], *ids, 1)
        ctx.flush()

    whole = [4 * page * i for i in range(2 * layers)]
    turns = [2 * page * 4 * i for i in range(2 * layers)]
    for bad in (*((whole, s, 0) for s in (1, 2, 3)), *((whole, s, page) for s in (1, 3)), (whole, 3.5, 0),
                (turns, 0.5, 2 * page), (turns, 1.5, 2 * page), (turns, 2, 2 * page), (turns, 4.5, 2 * page), (turns, 6, 2 * page)):
        starts, shift, stride = bad
        n = d.launch_count(ctx)
        with pytest.raises(d.Dispatch, match="overlap"):
            copy([*starts[:-1], starts[-2] + int(shift * page)], stride)
        assert d.launch_count(ctx) == n
    assert np.array_equal(buf.read(np.uint8), raw)
    for starts, shift, stride in ((whole, 4, 0), (turns, 1, 2 * page), (turns, 5, 2 * page), (turns, 7, 2 * page)):
        at = [*starts[:-1], starts[-2] + shift * page]
        copy(at, stride)
        for k in at:
            raw[k + 3 * (stride or page):][:page] = raw[k + (stride or page):][:page]
        assert np.array_equal(buf.read(np.uint8), raw)
    copy([0, page], 0, 1)  # (one page each: one behind the other)


@pytest.mark.parametrize("kind", ["q4", "f16", "f32"])
def test_sizes_beyond_64_bits(ctx, kind):
    """Pages whose bytes do not fit 64 bits are refused, by every call over pages."""
    buf = ctx.new_buffer(1 << 16)
    n = d.launch_count(ctx)
    for heads, ps in ((1 << 25, 1 << 31), (1 << 31, 1 << 31), (1 << 29, 1 << 27), (1 << 31, 1 << 28)):
        b = d.PagedBatch(buf, buf.ptr + 256, kind, 1, ps, heads, 256, None, 0, 1, buf)
        for call in (lambda: d.paged_copy(ctx, b, buf, buf, 1), lambda: d.paged_gather_f32(ctx, b, buf, buf),
                     lambda: d.rope_kv_append_paged_f32(ctx, b, buf, buf, buf, buf, heads, 1e4),
                     lambda: d.paged_attention_f32(ctx, b, buf, buf.ptr + 4096, heads)):
            with pytest.raises(d.Dispatch, match="address space"):
                call()
    assert d.launch_count(ctx) == n


@pytest.mark.parametrize("n", [32_767, 40_000])
def test_long_lists_of_large_pages(ctx, n):
    """Pages of 8 MB (512 workgroups each), most entries without one."""
    p = Pools(ctx, "f32", 2, 16384, 64, 4, 1, seed=n)
    src, dst = np.full(n, 0xFFFFFFFF, np.uint32), np.zeros(n, np.uint32)
    for at, s, t in ((7, 0, 1), (1023, 1, 2), (1024, 2, 0), (n - 1, 3, 2)):
        src[at], dst[at] = s, t
    p.copy(src, dst)
    p.check()


def test_lists_of_the_largest_pages(ctx):
    """Pages of 1.2 GB are 73,728 workgroups' each: fewer entries a launch."""
    p = d.PagedBatch.page_bytes("q4", 1, 1 << 25, 64)
    bufs = [ctx.new_buffer(2 * p) for _ in range(2)]
    rows = np.random.default_rng(1).integers(0, 256, (2, 1 << 20), np.uint8)
    for b, r in zip(bufs, rows):
        b.write(r), b.write(r[::-1], p - r.size)
    batch = d.PagedBatch(*bufs, "q4", 2, 1 << 25, 1, 64, None, 0, 0, None)
    n, src = d.launch_count(ctx), np.full(300, 0xFFFFFFFF, np.uint32)
    src[299] = 0
    d.paged_copy(ctx, batch, ctx.buffer_from(src), ctx.buffer_from(np.ones(300, np.uint32)), 300)
    ctx.flush()
    assert d.launch_count(ctx) == n + 4  # (2^24 workgroups: 227 entries of a pool)
    for b, r in zip(bufs, rows):
        assert np.array_equal(b.read(np.uint8, r.size, p), r) and np.array_equal(b.read(np.uint8, r.size, 2 * p - r.size), r[::-1])
        b.free()
