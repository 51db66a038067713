"""Batches over a paged cache for the tests: a pool whose unwritten places hold
NaN, and append and attention in 64 bits."""
from __future__ import annotations

import numpy as np

from runit_mac_amd import dispatch as d

NONE = 0xFFFFFFFF
F32 = 2.0 ** -24  # half a step of f32


class Batch:
    """seqs: (kept, new) positions of each sequence; new rows are its last
    positions.  one: no row_start (each sequence brings one row)."""

    def __init__(self, seqs, H, KVH, hd, ps, f16=False, seed=0, spare_rows=0, one=False, gap=0, vscale=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.H, self.KVH, self.hd, self.ps, self.f16 = seqs, H, KVH, hd, ps, f16
        self.new = np.array([n for _, n in seqs])
        self.kv = np.array([k + n for k, n in seqs])
        self.start = np.concatenate([[0], np.cumsum(self.new)])
        self.R, self.rows, self.one = int(self.start[-1]), int(self.start[-1]) + spare_rows, one
        per = -(-self.kv // ps)
        self.stride = int(max(per.max(initial=0), 1)) + 1
        total = int(per.sum()) + 2
        order = rng.permutation(total)
        self.table = np.full((len(seqs), self.stride), NONE, np.uint32)
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.total, self.gap = total, gap
        dt = np.float16 if f16 else np.float32
        self.page = KVH * ps * hd + gap
        self.k, self.v = (np.full((total, self.page), np.nan, dt) for _ in range(2))
        for s in range(len(seqs)):
            for pool, sc in ((self.k, 1.0), (self.v, vscale)):
                self.put(pool, s, 0, (sc * rng.standard_normal((int(self.kv[s]), KVH, hd))).astype(dt))
        self.q = rng.standard_normal((self.rows, H, hd)).astype(np.float32)

    def cells(self, pool):
        n = self.KVH * self.ps * self.hd
        return pool[:, :n].reshape(self.total, self.KVH, self.ps, self.hd)

    def put(self, pool, s, p0, rows):
        c = self.cells(pool)
        for i, r in enumerate(rows):
            c[self.table[s, (p0 + i) // self.ps], :, (p0 + i) % self.ps] = r

    def get(self, pool, s, table=None):
        """[positions][KVH][hd] in 64 bits; no page: NaN."""
        c, L = self.cells(pool), int(self.kv[s])
        t = self.table[s] if table is None else table
        out = np.full((L, self.KVH, self.hd), np.nan)
        for p in range(0, L, self.ps):
            if p // self.ps < len(t) and t[p // self.ps] < self.total:
                n = min(self.ps, L - p)
                out[p:p + n] = c[t[p // self.ps], :, :n].transpose(1, 0, 2)
        return out

    def upload(self, ctx):
        self.bk, self.bv = ctx.buffer_from(self.k), ctx.buffer_from(self.v)
        self.bt, self.bl = ctx.buffer_from(self.table), ctx.buffer_from(self.kv.astype(np.uint32))
        self.bs = None if self.one else ctx.buffer_from(self.start.astype(np.uint32))
        return d.PagedBatch(self.bk, self.bv, "f16" if self.f16 else "f32", self.total, self.ps, self.KVH,
                            self.hd, self.bt, self.stride, len(self.seqs), self.bl, rows=self.rows,
                            row_start=self.bs, page_stride=self.page if self.gap else 0)

    def attention(self, keys=None, vals=None, only=None):
        """The outputs in 64 bits, and a bound of an f32 computation's error:
        scores of hd + 16 roundings of Σ|qk|, a weight and their sum e^ of that
        each, sums of L terms and 64 more roundings, all of Σ w|v|.  f16 pages:
        weights as pairs of f16, the largest scaled to 2^12 or more, the smaller half's last place
        2^-24: an absolute 2^-37 of the largest weight, and that of the values.
        `only`: of these rows (the others' are zeros)."""
        H, KVH, hd, G = self.H, self.KVH, self.hd, self.H // self.KVH
        out, tol = np.zeros((self.R, H, hd)), np.zeros((self.R, H, hd))
        for s in range(len(self.seqs)):
            K = self.get(self.k, s) if keys is None else keys[s]
            V = self.get(self.v, s) if vals is None else vals[s]
            for i in range(int(self.new[s])):
                r, p = int(self.start[s]) + i, int(self.kv[s] - self.new[s]) + i
                seen = np.flatnonzero(~np.isnan(K[:p + 1, 0, 0])) if p >= 0 else np.zeros(0, int)
                if not len(seen) or only is not None and r not in only:
                    continue
                for h in range(H):
                    k, v = K[seen, h // G], V[seen, h // G]
                    q = self.q[r, h].astype(np.float64)
                    x = k @ q / np.sqrt(hd)
                    w = np.exp(x - x.max())
                    out[r, h] = w @ v / w.sum()
                    mag = (np.abs(k) @ np.abs(q)).max() / np.sqrt(hd)
                    tol[r, h] = w @ np.abs(v) / w.sum() * (2 * (hd + 16) * mag + len(seen) + 64) * F32
                    if self.f16:
                        tol[r, h] += len(seen) * np.abs(v).max(0) * w.max() / w.sum() * 2.0 ** -37
        return out, tol


def rope64(x, pos, theta):
    """x [rows][heads][hd] at pos [rows], pairs (d, d + hd/2)."""
    half = x.shape[-1] // 2
    a = pos[:, None] * theta ** (-2.0 * np.arange(half) / (2 * half))
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    lo, hi = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    return np.concatenate([lo * c - hi * s, lo * s + hi * c], -1)
