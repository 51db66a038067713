"""Many sequences decoded together over a paged cache (no counterpart in the
reference, whose engine holds one sequence in one KvCache).

A BatchDecoder takes a DecodeModel's weights and gives its sequences pages of
one pool as they grow.  Each pass runs any number of rows of any of them
together: prompts, single tokens, drafts to verify.  All sequences may begin
with the same prompt, held once and read for all together; a sequence may go on
as several, which share its pages until they write to them.  Rules on a
sequence's next token (penalties, biases, a grammar's mask) come before the
choice.
"""
from __future__ import annotations

from ctypes import c_float
from dataclasses import dataclass

import numpy as np

from . import dispatch as d
from .decode import Arena, DecodeModel, accept_drafts

NO_PAGE = 0xFFFFFFFF
NO_BIASES = np.zeros(0, np.int64), np.zeros(0, np.float32)


class PagePool:
    """The page ids 0 .. num_pages - 1, given out and taken back; a page that
    several hold is free when each has given it."""

    def __init__(self, num_pages: int):
        self.num_pages = num_pages
        self._free = list(range(num_pages - 1, -1, -1))
        self._holders: dict[int, int] = {}

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise d.BufferSize(f"buffer size mismatch: expected {n} free pages, got {len(self._free)}")
        pages = [self._free.pop() for _ in range(n)]
        self._holders.update(dict.fromkeys(pages, 1))
        return pages

    def give(self, pages) -> None:
        for p in reversed(pages):
            self._holders[p] -= 1
            if not self._holders[p]:
                del self._holders[p]
                self._free.append(p)

    def share(self, pages) -> None:
        """Another holder of pages that are held."""
        for p in pages:
            self._holders[p] += 1

    def holders(self, page: int) -> int:
        return self._holders.get(page, 0)

    def compaction(self) -> dict[int, int]:
        """Where the held pages would go ({from: to}) to be the first ones."""
        n = len(self._holders)
        return dict(zip(sorted(p for p in self._holders if p >= n), sorted(p for p in self._free if p < n)))

    def move(self, moves: dict[int, int]) -> None:
        """Held pages have moved to free ones."""
        self._holders = {moves.get(p, p): k for p, k in self._holders.items()}
        self._free = sorted(set(range(self.num_pages)) - set(self._holders), reverse=True)


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


@dataclass
class Rules:
    """What holds for a sequence's next token, in this order: penalties for the
    tokens that it has (rt_logit_rules: `repetition` for all of them, `frequency`
    a time and `presence` once for those behind the first `prompt_len`), biases
    ({token: value}), the tokens that a grammar allows ([vocab] truth values, or
    bits in ceil(vocab / 32) u32 words)."""
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    prompt_len: int = 0
    bias: dict | None = None
    allowed: np.ndarray | None = None

    def checked(self, vocab: int) -> "Rules":
        rep, freq, pres = self.penalties()
        if not (0 < rep < np.inf and abs(freq) < np.inf and abs(pres) < np.inf):
            raise ValueError(f"rules: penalties {self.repetition}, {self.frequency}, {self.presence}")
        if not self.prompt_len >= 0 or self.prompt_len % 1:
            raise ValueError(f"rules: prompt_len {self.prompt_len}")
        if any(not 0 <= t < vocab or t % 1 for t in self.bias or ()):
            raise ValueError(f"rules: a bias's token is none of [0, {vocab})")
        left = self.left(vocab) if self.allowed is not None else None
        if self.bias:
            ids, bias = self.biases()
            if np.isnan(bias).any():
                raise ValueError("rules: a bias is NaN")
            never = ids[bias == -np.inf]
            if never.size:
                left = np.ones(vocab, bool) if left is None else left.copy()
                left[never] = False
        if left is not None and not left.any():
            raise ValueError("rules: no token is allowed")
        return self

    def penalties(self) -> tuple:
        """Repetition, frequency and presence as the 32-bit numbers that they become."""
        return c_float(self.repetition).value, c_float(self.frequency).value, c_float(self.presence).value

    def penalises(self) -> bool:
        """Whether the sequence's tokens change anything."""
        return self.penalties() != (1, 0, 0)

    def biases(self) -> tuple[np.ndarray, np.ndarray]:
        """The biases' tokens and, in 32 bits, values."""
        b = self.bias or {}
        with np.errstate(over="ignore", under="ignore"):
            return np.array(list(b), np.int64), np.array(list(b.values()), np.float64).astype(np.float32)

    def forbids(self, token: int) -> bool:
        """Whether the mask or a bias of -inf forbids a token."""
        ids, bias = self.biases()
        a = None if self.allowed is None else np.asarray(self.allowed)
        off = a is not None and not (a[token] if a.dtype == bool else a[token // 32] >> token % 32 & 1)
        return bool(off or np.any(bias[ids == token] == -np.inf))

    def left(self, vocab: int) -> np.ndarray:
        """The mask's tokens as [vocab] truth values."""
        a, words = np.asarray(self.allowed), -(-vocab // 32)
        if a.dtype == np.uint32 and a.shape == (words,):
            return np.unpackbits(np.ascontiguousarray(a).view(np.uint8), bitorder="little")[:vocab].view(bool)
        if a.dtype != bool or a.shape != (vocab,):
            raise ValueError(f"rules: allowed is neither {vocab} truth values nor {words} u32 words")
        return a

    def mask(self, vocab: int) -> np.ndarray:
        """The mask's tokens as bits in u32 words."""
        a, words = np.asarray(self.allowed), -(-vocab // 32)
        if a.dtype == np.uint32 and a.shape == (words,):
            return a
        bits = np.zeros(32 * words, bool)
        bits[:vocab] = self.left(vocab)
        return np.packbits(bits, bitorder="little").view(np.uint32)


class _Tokens:
    """Token ids in an array that grows; equal to a list of the same."""

    def __init__(self, ids=()):
        self._room = np.array(ids, np.uint32)
        self._n = self._room.size

    @property
    def ids(self) -> np.ndarray:
        return self._room[:self._n]

    def __len__(self) -> int:
        return self._n

    def __eq__(self, other) -> bool:
        return np.array_equal(self.ids, other.ids if isinstance(other, _Tokens) else other)

    def extend(self, ids) -> None:
        n = self._n + len(ids)
        if n > self._room.size:
            room = np.empty(n + n // 2, np.uint32)
            room[:self._n] = self.ids
            self._room = room
        self._room[self._n:n] = ids
        self._n = n

    def cut(self, n: int) -> None:
        self._n = min(self._n, n)


class _Sequence:
    def __init__(self, tokens: _Tokens):
        self.tokens = _Tokens(tokens.ids)
        self.len = len(tokens)
        self.pages: list[int] = []  # from the prefix's last whole page on


class BatchDecoder:
    """`max_seqs` sequences of up to `max_len` positions over `num_pages` pages
    of `page_size` positions (f16, f32 or, q4, 4 bits: less memory, faster decoding over long
    contexts, prompts a little slower) a layer; passes of up to `max_rows` rows, the logits
    of up to `max_logits` of them at once, up to `max_top` alternatives.  Longer prompts run
    in several passes."""

    def __init__(self, model: DecodeModel, max_seqs: int, num_pages: int, page_size: int = 64,
                 kv: str = "f16", max_len: int | None = None, max_rows: int = 512,
                 max_logits: int = 64, max_top: int = 20):
        c = model.cfg
        max_len = c.max_seq if max_len is None else max_len
        if min(max_seqs, num_pages, max_len, max_rows, max_logits) < 1 or max_top < 0:
            raise ValueError("batch decoder: sizes must be positive")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"batch decoder: page_size {page_size} is not a power of two from 16 on")
        if kv not in ("f16", "f32", "q4"):
            raise ValueError(f"batch decoder: kv {kv!r}: 'f16', 'f32' or 'q4' expected")
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
        self._prefix_tokens = _Tokens()
        self.prefix_len = 0
        self._copied: list = []  # of the call that runs: (sequence, place, the page before)
        self._pick_rules: list | None = None  # of the pass's kept rows: rules and tokens
        self._rules_buf: dict = {}
        page = d.PagedBatch.page_bytes(kv, c.kv_heads, page_size, c.head_dim)
        # what a pass reads of its sequences, written in one piece: tokens, kept rows, targets, lengths, row
        # starts, tables; and the pages that are copied
        R, words = max_rows, 0
        self._meta = {}
        for name, n in (("tok", R), ("keep", R), ("target", R), ("kv_len", max_seqs), ("start", max_seqs + 1),
                        ("shared", self.stride), ("table", max_seqs * self.stride),
                        ("src", max(max_seqs, num_pages)), ("dst", max(max_seqs, num_pages))):
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
        self._all_pages = d.PagedBatch.array(self._pages)

    # ───────────────────────────── sequences ─────────────────────────────

    def open(self) -> int:
        """A new sequence, empty but for the shared prompt."""
        if len(self._seqs) >= self.max_seqs:
            raise d.BufferSize(f"buffer size mismatch: expected room for another sequence, got {self.max_seqs}")
        self._next += 1
        self._seqs[self._next] = _Sequence(self._prefix_tokens)
        return self._next

    def fork(self, seq: int) -> int:
        """A new sequence that goes on from where `seq` is.  Their pages are the
        same ones until either writes to one, which is copied first."""
        s = self._seq(seq)
        new = self.open()
        f = self._seqs[new]
        f.tokens, f.len, f.pages = _Tokens(s.tokens.ids), s.len, list(s.pages)
        self.pool.share(f.pages)
        return new

    def compact(self) -> int:
        """Moves the pages in use to the pools' beginning; how many they are."""
        moves = self.pool.compaction()
        if moves:
            self._copy_pages(list(moves), list(moves.values()))
            for s in self._seqs.values():
                s.pages = [moves.get(p, p) for p in s.pages]
            self._prefix_pages = [moves.get(p, p) for p in self._prefix_pages]
            self.pool.move(moves)
        return self.pool.num_pages - self.pool.free

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
        s.tokens.cut(length)
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
        self._prefix_pages, self._prefix_tokens, self.prefix_len = [], _Tokens(), 0
        if toks.size == 0:
            return
        seq = self.open()
        try:
            self._run({seq: toks}, None)
        except BaseException:
            self.close(seq)
            raise
        s = self._seqs.pop(seq)
        self._prefix_pages, self._prefix_tokens, self.prefix_len = s.pages, s.tokens, s.len

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

    def step(self, work: dict, top: int | None = None, rules: dict | None = None) -> dict:
        """Appends tokens to sequences ({sequence: tokens}) and returns the
        likeliest next token of each that its `rules` ({sequence: Rules}) leave
        (ValueError if they leave none with a logit above -inf); with `top`,
        pairs of it and its TokenScores with that many alternatives, the model's
        own: without the rules."""
        work = self._checked(work)
        if any(t.size == 0 for t in work.values()):
            raise ValueError("step: empty sequence of tokens")
        for s, r in (rules or {}).items():
            if s not in work:
                raise ValueError(f"rules: sequence {s!r} is not in the step")
            r.checked(self.model.cfg.vocab)
        got = self._run(work, {s: range(t.size - 1, t.size) for s, t in work.items()}, top, rules=rules)
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
        need, writers = 0, {}
        for s, t in work.items():
            q = self._seq(s)
            if q.len + t.size > self.max_len:
                raise ValueError(f"sequence {s}: {q.len} + {t.size} tokens exceed max_len {self.max_len}")
            need += self._more_pages(q, t.size)
            if t.size and self._shared_end(q) is not None:
                writers[q.pages[-1]] = writers.get(q.pages[-1], 0) + 1
        # (one of a page's holders keeps it)
        need += sum(min(n, self.pool.holders(p) - 1) for p, n in writers.items())
        if need > self.pool.free:
            raise d.BufferSize(f"buffer size mismatch: expected {need} free pages, got {self.pool.free}")
        return work

    def _shared_end(self, q: _Sequence) -> int | None:
        """The page that the sequence's next position is in, if others hold it too."""
        begun = q.pages and q.len % self.page_size
        return q.pages[-1] if begun and self.pool.holders(q.pages[-1]) > 1 else None

    def _more_pages(self, q: _Sequence, n: int) -> int:
        if n == 0:
            return 0
        return -(-(q.len + n) // self.page_size) - self.prefix_len // self.page_size - len(q.pages)

    def _run(self, work: dict, keep: dict | None, top: int | None = None, given: bool = False,
             rules: dict | None = None) -> dict:
        """The passes over `work`; of the tokens in `keep`'s ranges the argmax,
        or (`given`) the token that follows, and with `top` its scores.  If one
        fails, the sequences are as they were before all of them."""
        if top is not None and not 0 <= top <= self.max_top:
            raise ValueError(f"top {top} is not within 0 .. {self.max_top}")
        before = {s: self._seqs[s].len for s in work}
        self._copied = []
        try:
            return self._passes(work, keep, top, given, rules or {})
        except BaseException:
            for s, n in before.items():
                self.trim(s, n)
            # (of a page that was copied nobody has written to the positions of those that held it)
            for q, at, page in reversed(self._copied):
                self.pool.share([page])
                self.pool.give([q.pages[at]])
                q.pages[at] = page
            raise
        finally:
            self._copied = []

    def _passes(self, work: dict, keep: dict | None, top: int | None, given: bool, rules: dict) -> dict:
        parts = {s: [] for s in work}
        left = [(s, 0) for s, t in work.items() if t.size]
        self._own_ends([self._seqs[s] for s, _ in left])
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
            upto = {s: at + n for s, at, n in batch}
            said = lambda s, n: _Tokens(np.concatenate([self._seqs[s].tokens.ids, work[s][upto[s] - n:upto[s]]]))
            self._pick_rules = [(rules[s], said(s, n) if rules[s].penalises() else _Tokens()) if s in rules else None
                                for s, _, n in batch if s in owner] if any(s in rules for s in owner) else None
            got = self._launch(batch, row, picks, targets if given else None, top)
            # (a row of -inf and NaN has the first token for its likeliest)
            for s, r, t in zip(owner, self._pick_rules or (), got[0] if got else ()):
                if t == 0 and r is not None and r[0].forbids(0):
                    raise ValueError(f"rules: they leave sequence {s} no token with a logit")
            for s, at, n in batch:
                self._seqs[s].len += n
                self._seqs[s].tokens.extend(work[s][at:at + n])
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

    def _own_ends(self, seqs) -> None:
        """Copies the pages that these sequences, all that a call appends to, write to
        next and others hold.  A page that all of its holders write to is kept by the
        longest: it stores nothing before the others' ends, so that they can have the
        page back if the call fails."""
        by_page, writers = {}, []
        for q in seqs:
            page = self._shared_end(q)
            if page is not None:
                by_page.setdefault(page, []).append(q)
        for page, qs in by_page.items():
            keeper = max(reversed(qs), key=lambda q: q.len) if len(qs) == self.pool.holders(page) else None
            writers += [(q, page) for q in qs if q is not keeper]
        if not writers:
            return
        fresh = self.pool.take(len(writers))
        try:
            self._copy_pages([page for _, page in writers], fresh)
        except BaseException:
            self.pool.give(fresh)
            raise
        for (q, page), new in zip(writers, fresh):
            self._copied.append((q, len(q.pages) - 1, page))
            q.pages[-1] = new
            self.pool.give([page])

    def _copy_pages(self, src, dst) -> None:
        """Pages of every layer, of the same lengths, none both read and written."""
        ctx = self.ctx
        for name, ids in (("src", src), ("dst", dst)):
            at, n = self._meta[name], len(ids)
            self._host[at:at + n] = ids
            ctx._check(ctx.lib.rt_upload(ctx.handle, self._at[name], self._host[at:].ctypes.data, 4 * n))
        for i in range(0, len(src), 65535):  # (of a call)
            d.paged_copy(ctx, self._all_pages, self._at["src"] + 4 * i, self._at["dst"] + 4 * i, min(65535, len(src) - i))

    def _rules(self, rows):
        """LogitRules of rows of (rules, tokens) or None, their arrays on the device."""
        vocab, n = self.model.cfg.vocab, len(rows)
        rules = [r[0] if r else Rules() for r in rows]
        lists = [(r[1] if r else _Tokens()).ids for r in rows]
        penalties = np.array([r.penalties() for r in rules], np.float32).view(np.uint32)
        ids, biases = zip(*(r.biases() if r.bias else NO_BIASES for r in rules))
        masks = [r.mask(vocab) for r in rules if r.allowed is not None]
        starts = lambda x: np.concatenate([[0], np.cumsum([len(v) for v in x])[:-1]])
        u32 = lambda v: np.asarray(v, np.int64).astype(np.uint32)
        parts = dict(
            tokens=np.concatenate(lists), token_start=u32(starts(lists)), token_len=u32([len(v) for v in lists]),
            prompt_len=u32([min(r.prompt_len, 0xFFFFFFFF) for r in rules]), repetition=penalties[:, 0],
            frequency=penalties[:, 1], presence=penalties[:, 2],
            bias_ids=u32(np.concatenate(ids)), bias=np.concatenate(biases).view(np.uint32),
            bias_start=u32(starts(ids)), bias_len=u32([len(t) for t in ids]),
            mask=np.concatenate(masks) if masks else u32([]),
            mask_row=u32(np.where([r.allowed is not None for r in rules],
                                  np.cumsum([r.allowed is not None for r in rules]) - 1, NO_PAGE)))
        host, at = np.concatenate(list(parts.values())), {}
        for k, v in parts.items():
            at[k] = sum(x.size for x in list(parts.values())[:len(at)])
        buf = self._rules_buf.get("lists")
        if buf is None or buf.nbytes < host.nbytes:
            self.ctx.flush()  # (calls before may read the old one)
            buf = self._rules_buf["lists"] = self.ctx.new_buffer(2 * host.nbytes)
        buf.write(host)
        p = {k: buf.ptr + 4 * v for k, v in at.items()}
        return d.LogitRules(n_tokens=parts["tokens"].size, n_bias=parts["bias"].size, mask_rows=len(masks), **p)

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
                logits, rules = B["logits"], self._pick_rules
                if rules is not None and any(rules[r:r + n]):
                    if top is not None:  # (the scores are of the logits as they are)
                        if "logits" not in self._rules_buf:
                            self._rules_buf["logits"] = ctx.new_buffer(4 * self.max_logits * c.vocab)
                        logits = self._rules_buf["logits"].ptr
                    d.adjust_logits_f32(ctx, B["logits"], logits, n, c.vocab, self._rules(rules[r:r + n]))
                d.argmax_rows_first_f32(ctx, logits, B["idx"] + 4 * r, n, c.vocab)
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
        for b in self._rules_buf.values():
            b.free()
        self._rules_buf = {}
