"""Many sequences decoded together over a paged cache (no counterpart in the
reference, whose engine holds one sequence in one KvCache).

A BatchDecoder takes a DecodeModel's weights and gives its sequences pages of
one pool as they grow.  Each pass runs any number of rows of any of them
together: prompts, single tokens, drafts to verify.  All sequences may begin
with the same prompt, held once and read for all together.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from . import dispatch as d
from .decode import Arena, DecodeModel, accept_drafts

NO_PAGE = 0xFFFFFFFF


class PagePool:
    """The page ids 0 .. num_pages - 1, given out and taken back."""

    def __init__(self, num_pages: int):
        self.num_pages = num_pages
        self._free = list(range(num_pages - 1, -1, -1))

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise d.BufferSize(f"buffer size mismatch: expected {n} free pages, got {len(self._free)}")
        return [self._free.pop() for _ in range(n)]

    def give(self, pages) -> None:
        self._free.extend(reversed(pages))


@dataclass
class TokenScores:
    """Of each of a sequence's tokens: its log probability given those before
    it, the distribution's entropy (nats), how many tokens were likelier, and
    the likeliest ones with their log probabilities ([tokens][top])."""
    tokens: np.ndarray
    logprob: np.ndarray
    entropy: np.ndarray
    rank: np.ndarray
    top_ids: np.ndarray
    top_logprobs: np.ndarray


class _Sequence:
    def __init__(self, length: int):
        self.len = length
        self.pages: list[int] = []  # from the prefix's last whole page on


class BatchDecoder:
    """`max_seqs` sequences of up to `max_len` positions over `num_pages` pages
    of `page_size` positions (f16 or f32) a layer; passes of up to `max_rows`
    rows, the logits of up to `max_logits` of them at once, up to `max_top`
    alternatives.  Longer prompts run in several passes."""

    def __init__(self, model: DecodeModel, max_seqs: int, num_pages: int, page_size: int = 64,
                 kv: str = "f16", max_len: int | None = None, max_rows: int = 512,
                 max_logits: int = 64, max_top: int = 20):
        c = model.cfg
        max_len = c.max_seq if max_len is None else max_len
        if min(max_seqs, num_pages, max_len, max_rows, max_logits) < 1 or max_top < 0:
            raise ValueError("batch decoder: sizes must be positive")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"batch decoder: page_size {page_size} is not a power of two from 16 on")
        if kv not in ("f16", "f32"):
            raise ValueError(f"batch decoder: kv {kv!r}: 'f16' or 'f32' expected")
        if c.head_dim not in (64, 128, 256):
            raise ValueError(f"batch decoder: head size {c.head_dim}: 64, 128 or 256 expected")
        if model.lm_fmt in ("f16", "f32"):
            raise ValueError(f"LM head in {model.lm_fmt}: no f16/f32-weight GEMM here")
        if any(F["gate"] != F["up"] for F in model.fmts):
            raise ValueError("gate and up in different formats: no fused gate+up+SiLU")
        self.model, self.ctx, self.kv, self.page_size = model, model.ctx, kv, page_size
        # (the embedding takes 65,535 rows, the argmax of rows 14,336)
        max_rows, max_logits = min(max_rows, 65535), min(max_logits, 14336)
        self.max_seqs, self.max_len, self.max_rows = max_seqs, max_len, max_rows
        self.max_logits, self.max_top = min(max_logits, max_rows), min(max_top, c.vocab, 64)
        self.stride = -(-max_len // page_size)
        self.pool = PagePool(num_pages)
        self._seqs: dict[int, _Sequence] = {}
        self._next = 0
        self._prefix_pages: list[int] = []
        self.prefix_len = 0
        page = c.kv_heads * page_size * c.head_dim * (2 if kv == "f16" else 4)
        # what a pass reads of its sequences, written in one piece: tokens, kept rows, targets, lengths, row
        # starts, tables
        R, words = max_rows, 0
        self._meta = {}
        for name, n in (("tok", R), ("keep", R), ("target", R), ("kv_len", max_seqs), ("start", max_seqs + 1),
                        ("shared", self.stride), ("table", max_seqs * self.stride)):
            self._meta[name] = words
            words += -(-n // 64) * 64
        self._host = np.zeros(words, np.uint32)
        dims = dict(x=c.hidden, xn=c.hidden, q=c.q_dim, k=c.kv_dim, v=c.kv_dim, att=c.q_dim, p=c.hidden, g=c.ff,
                    u=c.ff, idx=1, logprob=1, entropy=1, rank=1, top_ids=self.max_top, top_logprobs=self.max_top)
        up = lambda n: (n + 255) & ~255
        a = self.arena = Arena(self.ctx, sum(up(4 * R * n) for n in dims.values()) + up(4 * words) +
                               up(4 * self.max_logits * c.vocab) + 2 * c.layers * up(page * num_pages))
        self._b = {k: a.take(4 * R * n) for k, n in dims.items()}
        self._b["logits"] = a.take(4 * self.max_logits * c.vocab)
        self._dev = a.take(4 * words)
        self._at = {k: self._dev + 4 * o for k, o in self._meta.items()}
        self._pages = [d.PagedBatch(a.take(page * num_pages), a.take(page * num_pages), kv, num_pages, page_size,
                                    c.kv_heads, c.head_dim, self._at["table"], self.stride, 0, self._at["kv_len"])
                       for _ in range(c.layers)]

    # ───────────────────────────── sequences ─────────────────────────────

    def open(self) -> int:
        """A new sequence, empty but for the shared prompt."""
        if len(self._seqs) >= self.max_seqs:
            raise d.BufferSize(f"buffer size mismatch: expected room for another sequence, got {self.max_seqs}")
        self._next += 1
        self._seqs[self._next] = _Sequence(self.prefix_len)
        return self._next

    def close(self, seq: int) -> None:
        self.pool.give(self._seq(seq).pages)
        del self._seqs[seq]

    def length(self, seq: int) -> int:
        return self._seq(seq).len

    def trim(self, seq: int, length: int) -> None:
        """Forgets a sequence's positions from `length` on."""
        s = self._seq(seq)
        if not self.prefix_len <= length <= s.len:
            raise ValueError(f"trim: {length} is not within {self.prefix_len} .. {s.len}")
        s.len = length
        keep = -(-length // self.page_size) - self.prefix_len // self.page_size if length > self.prefix_len else 0
        self.pool.give(s.pages[keep:])
        del s.pages[keep:]

    def share_prefix(self, tokens) -> None:
        """Runs `tokens` as the beginning of every sequence to come, in pages
        of their own.  While no sequence is open; no tokens: none any more.
        Refused, it leaves the former ones; if a pass fails, there are none."""
        if self._seqs:
            raise ValueError("share_prefix: sequences are open")
        toks = self._tokens(tokens)
        if toks.size > self.max_len:
            raise ValueError(f"share_prefix: {toks.size} tokens exceed max_len {self.max_len}")
        need, there = -(-toks.size // self.page_size), self.pool.free + len(self._prefix_pages)
        if need > there:
            raise d.BufferSize(f"buffer size mismatch: expected {need} free pages, got {there}")
        self.pool.give(self._prefix_pages)
        self._prefix_pages, self.prefix_len = [], 0
        if toks.size == 0:
            return
        seq = self.open()
        try:
            self._run({seq: toks}, None)
        except BaseException:
            self.close(seq)
            raise
        s = self._seqs.pop(seq)
        self._prefix_pages, self.prefix_len = s.pages, s.len

    def _seq(self, seq: int) -> _Sequence:
        if seq not in self._seqs:
            raise ValueError(f"sequence {seq!r} is not open")
        return self._seqs[seq]

    def _tokens(self, tokens) -> np.ndarray:
        ids = np.asarray(tokens)
        ids = ids.astype(np.int64, casting="same_kind" if ids.size else "unsafe").ravel()
        # (the embedding reads its table at the id unchecked)
        if np.any(ids < 0) or np.any(ids >= self.model.cfg.vocab):
            raise ValueError(f"token id out of range [0, {self.model.cfg.vocab})")
        return ids.astype(np.uint32)

    # ────────────────────────────── passes ──────────────────────────────

    def step(self, work: dict, top: int | None = None) -> dict:
        """Appends tokens to sequences ({sequence: tokens}) and returns the
        likeliest next token of each; with `top`, pairs of it and its
        TokenScores with that many alternatives."""
        work = self._checked(work)
        if any(t.size == 0 for t in work.values()):
            raise ValueError("step: empty sequence of tokens")
        got = self._run(work, {s: range(t.size - 1, t.size) for s, t in work.items()}, top)
        if top is None:
            return {s: int(g.tokens[0]) for s, g in got.items()}
        return {s: (int(g.tokens[0]), g) for s, g in got.items()}

    def score(self, work: dict, top: int = 0) -> dict:
        """Appends tokens to sequences and returns the TokenScores of each's
        tokens but the first (whose logits came with the token before it)."""
        work = self._checked(work)
        if any(t.size == 0 for t in work.values()):
            raise ValueError("score: empty sequence of tokens")
        return self._run(work, {s: range(t.size - 1) for s, t in work.items()}, top, given=True)

    def verify(self, work: dict) -> dict:
        """verify_draft (forward.rs:2118-2309) of several sequences at once:
        {sequence: (token, drafts)} → {sequence: (accepted, next token)}; each
        sequence keeps its token and its accepted drafts."""
        drafts = {s: self._tokens(dr) for s, (_, dr) in work.items()}
        rows = self._checked({s: np.concatenate([self._tokens([t]), drafts[s]]) for s, (t, _) in work.items()})
        base = {s: self._seq(s).len for s in rows}
        got = self._run(rows, {s: range(t.size) for s, t in rows.items()})
        out = {}
        for s, g in got.items():
            out[s] = accept_drafts(g.tokens, drafts[s])
            self.trim(s, base[s] + 1 + out[s][0])
        return out

    def _checked(self, work: dict) -> dict:
        work = {s: self._tokens(t) for s, t in work.items()}
        need = 0
        for s, t in work.items():
            q = self._seq(s)
            if q.len + t.size > self.max_len:
                raise ValueError(f"sequence {s}: {q.len} + {t.size} tokens exceed max_len {self.max_len}")
            need += self._more_pages(q, t.size)
        if need > self.pool.free:
            raise d.BufferSize(f"buffer size mismatch: expected {need} free pages, got {self.pool.free}")
        return work

    def _more_pages(self, q: _Sequence, n: int) -> int:
        if n == 0:
            return 0
        return -(-(q.len + n) // self.page_size) - self.prefix_len // self.page_size - len(q.pages)

    def _run(self, work: dict, keep: dict | None, top: int | None = None, given: bool = False) -> dict:
        """The passes over `work`; of the tokens in `keep`'s ranges the argmax,
        or (`given`) the token that follows, and with `top` its scores.  If one
        fails, the sequences are as they were before all of them."""
        if top is not None and not 0 <= top <= self.max_top:
            raise ValueError(f"top {top} is not within 0 .. {self.max_top}")
        before = {s: self._seqs[s].len for s in work}
        try:
            return self._passes(work, keep, top, given)
        except BaseException:
            for s, n in before.items():
                self.trim(s, n)
            raise

    def _passes(self, work: dict, keep: dict | None, top: int | None, given: bool) -> dict:
        parts = {s: [] for s in work}
        left = [(s, 0) for s, t in work.items() if t.size]
        while left:
            rows, batch = 0, []
            while left and rows < self.max_rows:
                s, at = left.pop(0)
                n = min(work[s].size - at, self.max_rows - rows)
                batch.append((s, at, n))
                rows += n
                if at + n < work[s].size:
                    left.insert(0, (s, at + n))
            # (rows in the batch's order; a sequence is in a pass once)
            picks, targets, owner, row = [], [], [], 0
            for s, at, n in batch:
                kept = range(max(at, keep[s].start), min(at + n, keep[s].stop)) if keep else ()
                picks += [row + i - at for i in kept]
                owner += [s] * len(kept)
                targets += [work[s][i + 1] for i in kept] if given else ()
                row += n
            self._place(batch, work, picks, targets)
            got = self._launch(batch, row, picks, targets if given else None, top)
            for s, _, n in batch:
                self._seqs[s].len += n
            owner = np.array(owner)
            for s, _, _ in batch:
                if np.any(owner == s):
                    parts[s].append([g[owner == s] for g in got])
        empty = [np.zeros(0, np.uint32), np.zeros(0, np.float32), np.zeros(0, np.float32), np.zeros(0, np.uint32),
                 np.zeros((0, top or 0), np.uint32), np.zeros((0, top or 0), np.float32)]
        return {s: TokenScores(*(np.concatenate(x) for x in zip(*p))) if p else TokenScores(*empty)
                for s, p in parts.items()}

    def _place(self, batch, work, picks, targets) -> None:
        """The pages and the host's arrays of a pass: batch of (sequence, first
        token, tokens)."""
        host, meta, W = self._host, self._meta, self.stride
        first = self.prefix_len // self.page_size
        table = host[meta["table"]:meta["table"] + len(batch) * W].reshape(len(batch), W)
        table[:] = NO_PAGE
        put = lambda name, at, v: host.__setitem__(slice(meta[name] + at, meta[name] + at + len(v)), v)
        row = 0
        for i, (s, at, n) in enumerate(batch):
            q = self._seqs[s]
            q.pages += self.pool.take(self._more_pages(q, n))
            put("start", i, [row, row + n])
            put("kv_len", i, [q.len + n])
            put("tok", row, work[s][at:at + n])
            table[i, first:first + len(q.pages)] = q.pages
            row += n
        put("keep", 0, picks)
        put("target", 0, targets)
        put("shared", 0, self._prefix_pages)

    def _launch(self, batch, rows, picks, targets, top):
        m, c, ctx, B, at = self.model, self.model.cfg, self.ctx, self._b, self._at
        used = self._meta["table"] + len(batch) * self.stride
        ctx._check(ctx.lib.rt_upload(ctx.handle, self._dev, self._host.ctypes.data, 4 * used))
        start = None if rows == len(batch) else at["start"]
        h, form = c.hidden, m.row_form(rows)
        d.embed_rows_f32(ctx, m.embd_fmt, m.embd, at["tok"], B["x"], h, rows)
        for L, F, pages in zip(m.layers, m.fmts, self._pages):
            if form == "rows":
                m.qkv_rows(L, F, B, rows)
            else:
                d.gemm_set_f32(ctx, (F["q"], F["k"], F["v"]), (L["wq"], L["wk"], L["wv"]), (B["q"], B["k"], B["v"]),
                               (c.q_dim, c.kv_dim, c.kv_dim), B["x"], rows, h, biases=(L["bq"], L["bk"], L["bv"]),
                               gamma=L["attn_norm"], eps=c.eps, xn=B["xn"])
            pages.n_seqs, pages.rows, pages.row_start = len(batch), rows, start
            d.rope_kv_append_paged_f32(ctx, pages, B["q"], B["k"], B["v"], B["q"], c.heads, c.theta)
            if self.prefix_len:
                d.shared_prefix_attention_f32(ctx, pages, B["q"], B["att"], c.heads, at["shared"], self.prefix_len)
            else:
                d.paged_attention_f32(ctx, pages, B["q"], B["att"], c.heads)
            if form == "rows":
                m.out_ffn_rows(L, F, B, rows)
            else:
                d.gemm_ffn_block_f32(ctx, (F["o"], F["gate"], F["up"], F["down"]), L["wo"], L["wg"], L["wu"], L["wd"],
                                     B["att"], B["x"], B["p"], L["ffn_norm"], c.eps, B["g"], B["u"], B["xn"], rows, h,
                                     c.q_dim, c.ff)
        if not picks:
            return ()
        x, nk = B["x"], len(picks)
        if picks != list(range(rows)):
            # the kept rows together (a table of f32 rows, read at their numbers)
            d.embed_rows_f32(ctx, "f32", B["x"], at["keep"], B["p"], h, nk)
            x = B["p"]
        wanted = B["idx"] if targets is None else at["target"]
        for r in range(0, nk, self.max_logits):
            n = min(nk - r, self.max_logits)
            m.head_rows(m.row_form(n), x + 4 * r * h, B["logits"], B["xn"], n)
            if targets is None:
                d.argmax_rows_first_f32(ctx, B["logits"], B["idx"] + 4 * r, n, c.vocab)
            if top is not None:
                d.token_logprobs_f32(ctx, B["logits"], wanted + 4 * r, n, c.vocab, B["logprob"] + 4 * r,
                                     entropy=B["entropy"] + 4 * r, rank=B["rank"] + 4 * r, top=top,
                                     top_ids=B["top_ids"] + 4 * r * top, top_logprobs=B["top_logprobs"] + 4 * r * top)
        tokens = np.array(targets, np.uint32) if targets is not None else self._read("idx", nk, np.uint32)
        ns, f32, u32 = 0 if top is None else nk, np.float32, np.uint32
        return (tokens, self._read("logprob", ns, f32, nk), self._read("entropy", ns, f32, nk),
                self._read("rank", ns, u32, nk), self._read("top_ids", ns * (top or 0), u32).reshape(nk, -1),
                self._read("top_logprobs", ns * (top or 0), f32).reshape(nk, -1))

    def _read(self, name, n, dtype, size=0):
        """The first n elements of a result (and zeros up to size)."""
        out = np.zeros(max(n, size), dtype)
        if n:
            self.ctx._check(self.ctx.lib.rt_download(self.ctx.handle, out.ctypes.data, self._b[name], 4 * n))
        return out

    def free(self) -> None:
        self.arena.buf.free()
