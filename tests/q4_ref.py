"""Pages of 4 bits for the tests: codes and scale words in 64 bits, the pages'
layout, and batches over such pages."""
from __future__ import annotations

import numpy as np

from paged_ref import Batch
from runit_mac_amd import dispatch as d


def up7(x):
    """The next number of seven significant bits, a multiple of 2^-20."""
    m, e = np.frexp(x)
    unit = np.maximum(np.ldexp(1.0, e - 7), 2.0 ** -20)
    return np.ceil(x / unit) * unit


def step(word):
    return (word & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)


def encode(x):
    """Codes [...][hd] and scale words [...][hd / 32]; groups with a value that is
    not finite or beyond 32,768: NaN."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(g) <= 32768).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    lo, hi = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
    dd = up7((hi - lo) / 15)
    safe = np.where(dd > 0, dd, 1.0)
    z = np.rint(-lo / safe)
    n = np.clip(np.rint(g / safe[..., None]) + z[..., None], 0, 15).astype(np.uint8)
    w = dd.astype(np.float16).view(np.uint16) | z.astype(np.uint16)
    return n.reshape(x.shape), np.where(bad, 0xFFFF, w).astype(np.uint16)


def decode(n, w):
    g = n.reshape(*n.shape[:-1], -1, 32).astype(np.float64) - (w & 15)[..., None]
    with np.errstate(invalid="ignore"):
        return (g * step(w)[..., None]).reshape(n.shape)


def pack(n, w, values):
    """A KV head's part of a page: codes [ps][hd], words [ps][hd / 32] as bytes."""
    ps, hd = n.shape
    if values:
        q = 1 if hd == 64 else 2
        # [tile][g][pair][position][block][chunk][half][element] → [tile][block][g][chunk][pair][half][position][element]
        t = n.reshape(ps // 16, 4, 2, 2, hd // (64 * q), 16, q, 4).transpose(0, 4, 1, 5, 2, 6, 3, 7)
        words = w.reshape(ps // 16, 16, -1).transpose(0, 2, 1)
    else:
        t = n.reshape(ps, hd // 8, 4, 2).swapaxes(2, 3)
        words = w
    t = np.ascontiguousarray(t).reshape(-1, 2)
    return np.concatenate([t[:, 0] | t[:, 1] << 4, np.ascontiguousarray(words).reshape(-1).view(np.uint8)])


def unpack(part, ps, hd, values):
    half = ps * hd // 2
    t = np.stack([part[:half] & 15, part[:half] >> 4], -1)
    w = np.ascontiguousarray(part[half:half + ps * hd // 16]).view(np.uint16)
    if values:
        q = 1 if hd == 64 else 2
        t = t.reshape(ps // 16, hd // (64 * q), 4, 16, 2, q, 2, 4).transpose(0, 2, 4, 6, 1, 3, 5, 7)
        w = w.reshape(ps // 16, -1, 16).transpose(0, 2, 1)
    else:
        t = t.reshape(ps, hd // 8, 2, 4).swapaxes(2, 3)
    return np.ascontiguousarray(t).reshape(ps, hd), np.ascontiguousarray(w).reshape(ps, hd // 32)


class Batch4(Batch):
    """A Batch whose pool holds what 4 bits hold; k and v are their values
    (f16), NaN where nothing is."""

    def __init__(self, *args, gap=0, **kw):
        super().__init__(*args, True, **kw)
        self.gap = gap
        self.words = {}
        for name in "kv":
            c = self.cells(getattr(self, name))
            n, w = encode(c.astype(np.float64))
            c[:] = decode(n, w)
            self.words[name] = [n, w]

    def bytes_of(self, name):
        n, w = self.words[name]
        pages = [np.concatenate([pack(n[p, h], w[p, h], name == "v") for h in range(self.KVH)] +
                                [np.full(self.gap, 0xA5, np.uint8)]) for p in range(self.total)]
        return np.stack(pages)

    def upload(self, ctx):
        self.raw = {x: self.bytes_of(x) for x in "kv"}
        self.bk, self.bv = (ctx.buffer_from(self.raw[x]) for x in "kv")
        self.bt, self.bl = ctx.buffer_from(self.table), ctx.buffer_from(self.kv.astype(np.uint32))
        self.bs = None if self.one else ctx.buffer_from(self.start.astype(np.uint32))
        return d.PagedBatch(self.bk, self.bv, "q4", self.total, self.ps, self.KVH, self.hd, self.bt, self.stride,
                            len(self.seqs), self.bl, rows=self.rows, row_start=self.bs,
                            page_stride=self.raw["k"].shape[1] if self.gap else 0)

    def read(self, name):
        """Codes and words of the pool as it is on the device, [page][KV head]."""
        raw = (self.bk if name == "k" else self.bv).read(np.uint8).reshape(self.raw[name].shape)
        part = self.ps * self.hd * 9 // 16
        got = [[unpack(raw[p, h * part:(h + 1) * part], self.ps, self.hd, name == "v") for h in range(self.KVH)]
               for p in range(self.total)]
        return raw, np.array([[x[0] for x in p] for p in got]), np.array([[x[1] for x in p] for p in got])
