"""Operators of serving many sequences over caches of 4 bits, as cases that can
be timed and checked.

* append: the rotary embedding of a ragged batch's new queries and keys, keys
  and values stored into pages of 4 bits, and read back from them as f16;
* attention: the causal attention of the batch's rows over pages of 4 bits, from
  one new row a sequence (a decode step) to prompt chunks, also where all
  sequences begin with one long prefix;
* copy: pages of all layers' pools copied, as sequences fork or the pool is
  compacted;
* rules: penalties for repeated tokens, biases and grammar masks on logits.

A page of 4 bits holds, for each KV head, the codes of its positions and behind
them their scales, one for each 32 elements of a head: a word with the step d
in the upper twelve bits of an f16 and the zero point z in the lower four.  A
code n stands for d·(n − z).  Head layouts are those of the 0.5B and 7B Qwen2.5
configurations that bench.py runs; drawn cases take other sizes of the same
ranges.  Where `own` is true the framework's entry points run, otherwise plain
torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

THETA = 1e6
HALF = dict(heads=14, kv_heads=2, head_dim=64)    # 0.5B
SEVEN = dict(heads=28, kv_heads=4, head_dim=128)  # 7B


def listed():
    return [
        # one decode step of a few sequences on the 0.5B model: latency
        dict(name="append_step_0p5b", kind="append", page=16, seqs=4, lo=60, hi=700, new=1, shape=1, **HALF),
        # the rows of prompt chunks and decoding sequences together, far positions
        dict(name="append_chunk_7b", kind="append", page=64, seqs=12, lo=100, hi=20000, new=700, shape=2, **SEVEN),
        # a decode step of three short chats on the 0.5B model: latency
        dict(name="attn_step_0p5b", kind="attention", page=16, seqs=3, lo=100, hi=600, new=1, shared=0, shape=3,
             **HALF),
        # a decode step of a serving batch with long contexts on the 7B model
        dict(name="attn_step_7b", kind="attention", page=64, seqs=32, lo=300, hi=16000, new=1, shared=0, shape=4,
             **SEVEN),
        # drafts to verify behind one book of an odd number of positions
        dict(name="attn_long_7b", kind="attention", page=256, seqs=1, lo=200003, hi=200003, new=2, shared=0, shape=5,
             **SEVEN),
        # prompt chunks and decoding sequences in one batch
        dict(name="attn_chunk_7b", kind="attention", page=32, seqs=6, lo=100, hi=4000, new=375, shared=0, shape=7,
             **SEVEN),
        # many answers to one long document on the 7B model
        dict(name="shared_step_7b", kind="attention", page=64, seqs=40, lo=20, hi=600, new=1, shared=8192, shape=8,
             **SEVEN),
        # the last pages of two sequences that eight go on from, all layers of the 0.5B model, f16 pages
        dict(name="copy_fork_0p5b", kind="copy", bits=16, page=64, layers=24, pages=64, copies=8, sources=2, **HALF),
        # a 7B model's pool of 4 bits compacted: the pages in use behind its first ones go there
        dict(name="copy_compact_7b", kind="copy", bits=4, page=64, layers=28, pages=600, copies=277, sources=277,
             **SEVEN),
        # grammar masks alone, in place, on the logits of a small batch: latency
        dict(name="rules_grammar_step", kind="rules", f16=False, rows=5, n=151936, seen=0, biases=0, masks=3,
             inplace=True, shape=10),
        # all rules on a serving batch of the 7B model, the logits kept: histories of thousands of tokens
        dict(name="rules_all_7b", kind="rules", f16=False, rows=120, n=152064, seen=9000, biases=300, masks=40,
             inplace=False, shape=11),
        # f16 logits of an odd vocabulary, penalties and biases only
        dict(name="rules_f16", kind="rules", f16=True, rows=37, n=50001, seen=1500, biases=20, masks=0,
             inplace=False, shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "append", "attention", "attention", "shared", "shared", "copy", "copy", "rules", "rules"))
    if kind == "rules":
        n = _log(rng, 1000, 152064)
        rows = _log(rng, 1, min(500, 18_000_000 // n))
        seen = rng.choice((0, _log(rng, 1, 9000), _log(rng, 1, 9000)))
        biases = rng.choice((0, _log(rng, 1, 300)))
        masks = rng.choice((0, _log(rng, 1, rows)))
        if not (seen or biases or masks):
            masks = 1
        return dict(kind=kind, f16=rng.random() < 0.4, rows=rows, n=n, seen=seen, biases=biases, masks=masks,
                    inplace=not (seen or biases) and rng.random() < 0.7, shape=rng.randrange(1 << 20))
    kv = rng.choice((1, 2, 4, 8))
    c = dict(kind=kind, page=rng.choice((16, 32, 64, 128, 256)), kv_heads=kv, heads=kv * rng.randint(1, 9),
             head_dim=rng.choice((64, 64, 128, 128, 256)))
    wide = c["kv_heads"] * c["head_dim"]
    if kind == "copy":
        c["bits"] = rng.choice((4, 4, 16, 32))
        c["layers"] = _log(rng, 1, 32)
        page = 2 * c["layers"] * wide * c["page"] * (4.5 if c["bits"] == 4 else c["bits"]) / 8
        c["copies"] = _log(rng, 1, max(2, min(300, int(280e6 / page))))
        c["sources"] = rng.choice((c["copies"], rng.randint(1, c["copies"])))
        c["pages"] = c["copies"] + c["sources"] + rng.randint(0, max(1, min(50, int(200e6 / page))))
        return c
    c["kind"] = "append" if kind == "append" else "attention"
    c["shape"] = rng.randrange(1 << 20)
    if kind == "append":
        c["new"] = rng.choice((1, _log(rng, 2, 300)))
        c["seqs"] = _log(rng, 1, 24)
        c["lo"] = _log(rng, 1, 500)
        # the pool of all sequences stays within that of the largest listed case
        c["hi"] = _log(rng, c["lo"], max(c["lo"] + 1, min(20000, 30_000_000 // (c["seqs"] * wide))))
        return c
    c["new"] = rng.choice((1, 1, rng.randint(2, 8), _log(rng, 9, 300)))
    c["seqs"] = _log(rng, 2 if kind == "shared" else 1, 40 if c["new"] <= 8 else 6)
    c["shared"] = 0
    rows = c["seqs"] * min(c["new"], 8) + c["new"]
    most = 40_000_000 // (wide * c["seqs"])  # positions a sequence, by its memory ...
    most = max(64, min(most, 80_000_000 // (c["seqs"] * c["new"] * c["heads"]),  # ... and by the scores,
                       5_000_000_000 // (rows * c["heads"] * c["head_dim"])))    # ... and the products
    if kind == "shared":
        c["shared"] = _log(rng, 33, max(34, min(8192, most * 3 // 4)))
        if rng.random() < 0.6:
            c["shared"] = max(c["page"], c["shared"] // c["page"] * c["page"])
        c["lo"], top = _log(rng, 1, 30), max(31, min(600, most // 4))
    else:
        c["lo"], top = _log(rng, 1, 300), max(301, min(100000, most))
    c["hi"] = _log(rng, c["lo"], top)
    return c


# ───────────────────────────── pages of 4 bits ─────────────────────────────

def _places(c, values, dev="cuda"):
    """Of a KV head's part of a page, in 16-bit words: the word of each
    position's each element, the element's place among its word's four codes,
    and the scale's word of each position's each group."""
    ps, hd = c["page"], c["head_dim"]
    p = torch.arange(ps, device=dev)[:, None]
    e = torch.arange(hd, device=dev)[None, :]
    u = torch.arange(hd // 32, device=dev)[None, :]
    if values:  # tiles of 16 positions: two positions by four elements a 32-bit word
        w = 4 if hd == 64 else 8
        quad = (e // (16 * w) * 4 + p % 16 // 4) * 16 + e // w % 16
        word = p // 16 * 4 * hd + ((quad * 2 + p % 4 // 2) * (w // 4) + e % w // 4) * 2 + p % 2
        scale = p // 16 * (hd // 2) + u * 16 + p % 16
        nib = e % 4
    else:  # rows of positions: eight elements a 32-bit word, even ones in its lower half
        word = p * (hd // 4) + e // 8 * 2 + e % 2
        scale = p * (hd // 32) + u
        nib = e % 8 // 2
    return word, nib.expand(ps, hd), ps * hd // 4 + scale


def _read(c, pages, places):
    """[pages][KV heads][words] as [pages][KV heads][positions][elements] in 32 bits."""
    word, nib, scale = places
    shape = (*pages.shape[:2], c["page"], c["head_dim"])
    n = (pages[..., word.reshape(-1)].int() >> (4 * nib.reshape(-1)).int() & 15).view(shape)
    w = pages[..., scale.reshape(-1)]
    d = (w & ~15).view(torch.float16).float().view(*shape[:3], -1, 1)
    return ((n.view(*shape[:3], -1, 32) - (w.int() & 15).view(*shape[:3], -1, 1)) * d).view(shape)


def _coded(x):
    """Codes and scale words of [...][elements], 32 a scale."""
    g = x.double().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True).clamp_max(0), g.amax(-1, keepdim=True).clamp_min(0)
    step = (hi - lo) / 15
    # up to seven significant bits, of 2^-20 at least
    unit = torch.exp2(torch.floor(torch.log2(step.clamp_min(2.0 ** -30))) - 6).clamp_min(2.0 ** -20)
    d = torch.ceil(step / unit) * unit
    over = torch.where(d > 0, 1 / d, 0.0)
    z = torch.round(-lo * over)
    n = (torch.round(g * over) + z).clamp(0, 15)
    return n.flatten(-2).int(), d[..., 0].half().view(torch.int16) | z[..., 0].to(torch.int16)


def _store(c, pages, places, page, slot, x):
    """x [rows][KV heads][elements] to (page, slot) of [pages][KV heads][words]."""
    word, nib, scale = places
    n, w = _coded(x)
    order = torch.argsort(word[0] * 4 + nib[0])  # the elements of each word together
    piece = (n[..., order].unflatten(-1, (-1, 4)) << (4 * torch.arange(4, device="cuda"))).sum(-1).to(torch.int16)
    heads = torch.arange(c["kv_heads"], device="cuda")[None, :, None]
    at = page[:, None, None], heads
    pages[at + (word[slot][:, order[::4]][:, None],)] = piece
    pages[at + (scale[slot][:, None],)] = w


# ───────────────────────────── inputs ─────────────────────────────

def _sizes(c):
    """New rows and positions (new ones included) of each sequence."""
    r = np.random.default_rng(c["shape"])
    n = c["seqs"]
    kept = np.exp(r.uniform(np.log(c["lo"]), np.log(c["hi"] + 1), n)).astype(np.int64)
    new = np.exp(r.uniform(0, np.log(c["new"] + 1), n)).astype(np.int64)
    new[0], kept[-1] = c["new"], c["hi"]
    if c["new"] == 1:
        new[:] = 1
    return new, c.get("shared", 0) + kept + new


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _pool(c, g, total, values):
    """Pages of normally distributed keys or values, a channel's own size each."""
    ps, kvh, hd = c["page"], c["kv_heads"], c["head_dim"]
    out = torch.empty(total, kvh, ps * hd * 9 // 32, dtype=torch.int16, device="cuda")
    size = torch.exp(_normal(g, kvh, 1, hd, std=0.3))
    places = _places(c, values)
    heads = torch.arange(kvh, device="cuda")[None, :, None]
    word, nib, scale = places
    order = torch.argsort(word.reshape(-1) * 4 + nib.reshape(-1))
    for a in range(0, total, max(1, (8 << 20) // (kvh * ps * hd))):
        b = min(total, a + max(1, (8 << 20) // (kvh * ps * hd)))
        n, w = _coded(_normal(g, b - a, kvh, ps, hd) * size)
        piece = n.flatten(2)[..., order].unflatten(-1, (-1, 4)) << (4 * torch.arange(4, device="cuda"))
        out[a:b, :, :ps * hd // 4] = piece.sum(-1).to(torch.int16)
        out[a:b, :, scale.reshape(-1)] = w.flatten(2)
    return out, places


def _lists(r, c, most, new):
    """Of each row the length of a list and where it begins."""
    n = np.exp(r.uniform(0, np.log(most + 1), c["rows"])).astype(np.int64) if most else np.zeros(c["rows"], np.int64)
    if most:
        n[-1] = most
        n[r.random(c["rows"]) < 0.1] = 0
        n[0] = most
    return n, np.concatenate([[0], np.cumsum(n)[:-1]])


def _prepare_rules(c, g, seed):
    s, r = dict(case=c), np.random.default_rng(c["shape"])
    cuda = lambda a, t=np.int32: torch.from_numpy(np.asarray(a).astype(t)).cuda()
    rows, n = c["rows"], c["n"]
    x = _normal(g, rows, n, std=2.5)
    s["logits"] = x.half() if c["f16"] else x
    s["out"] = s["logits"] if c["inplace"] else torch.empty_like(s["logits"])
    u = np.random.default_rng(seed)
    for name, most in (("token", c["seen"]), ("bias", c["biases"])):
        size, start = _lists(r, c, most, None)
        s[name + "_len"], s[name + "_start"] = cuda(size), cuda(start)
        s[name + "_row"] = cuda(np.repeat(np.arange(rows), size), np.int64)
        # few tokens make up most of a text
        s[name + "_ids"] = cuda(np.minimum(n * u.random(int(size.sum())) ** 3, n - 1))
    s["bias"] = cuda(u.normal(0, 3, s["bias_ids"].numel()), np.float32)
    s["bias"][u.random(s["bias"].numel()) < 0.05] = -math.inf  # a token that is not wanted at all
    s["prompt_len"] = cuda(s["token_len"].cpu().numpy() * r.random(rows))
    s["place"] = torch.arange(s["token_ids"].numel(), device="cuda") - s["token_start"].long()[s["token_row"]]
    s["repetition"], s["frequency"], s["presence"] = (cuda(u.uniform(a, b, rows), np.float32)
                                                      for a, b in ((1.0, 1.3), (0.0, 0.5), (0.0, 0.7)))
    words = -(-n // 32)
    if c["masks"]:
        # a grammar leaves a few tokens, or all but a few
        few = torch.rand(c["masks"], 1, generator=g, device="cuda") < 0.7
        a, b, d = (torch.randint(-(1 << 31), 1 << 31, (c["masks"], words), generator=g, device="cuda") for _ in range(3))
        s["mask"] = torch.where(few, a & b & d, a | b | d).int()
        s["mask_row"] = cuda(np.where(r.random(rows) < 0.2, -1, r.integers(0, c["masks"], rows)))
        s["mask_row"][0] = 0
    return s


def _prepare_copy(c, g, seed):
    s, r = dict(case=c), np.random.default_rng(seed)
    size = c["kv_heads"] * c["page"] * c["head_dim"]
    size = size * 9 // 16 if c["bits"] == 4 else size * c["bits"] // 8
    s["pools"] = torch.randint(-(1 << 62), 1 << 62, (c["layers"], 2, c["pages"], size // 8), generator=g, device="cuda")
    order = r.permutation(c["pages"])  # pages in use, and free ones that they go to
    src = order[:c["sources"]][np.arange(c["copies"]) % c["sources"]]
    s["src"], s["dst"] = (torch.from_numpy(a.astype(np.int32)).cuda()
                          for a in (src, order[c["sources"]:c["sources"] + c["copies"]]))
    return s


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] in ("rules", "copy"):
        s = (_prepare_rules if c["kind"] == "rules" else _prepare_copy)(c, g, seed)
        torch.cuda.synchronize()
        return s
    s = dict(case=c)
    new, kv = _sizes(c)
    S, ps, kvh, hd = c["seqs"], c["page"], c["kv_heads"], c["head_dim"]
    shared = c.get("shared", 0)
    per = -(-kv // ps)  # pages of a sequence, whole shared ones first
    whole, first = shared // ps, -(-shared // ps)
    total = first + int((per - whole).sum()) + 3
    order = np.random.default_rng(seed).permutation(total)  # where each page is in the pool
    table = np.full((S, int(per.max()) + 2), -1, np.int32)
    at = first
    for i in range(S):
        own_pages = int(per[i]) - whole
        table[i, :whole] = order[:whole]
        table[i, whole:per[i]] = order[at:at + own_pages]
        at += own_pages
    (s["k"], s["k_at"]), (s["v"], s["v_at"]) = _pool(c, g, total, False), _pool(c, g, total, True)
    s["table"] = torch.from_numpy(table).cuda()
    if shared:
        s["shared_table"] = torch.from_numpy(order[:first].astype(np.int32)).cuda()
        if shared % ps:  # the last page of the prefix, copied as each sequence went on behind it
            for p in (s["k"], s["v"]):
                p[s["table"][:, whole].long()] = p[int(order[whole])].clone()
    s["kv_len"] = torch.from_numpy(kv.astype(np.int32)).cuda()
    R = int(new.sum())
    s["rows"], s["most"] = R, int(new.max())
    start = np.concatenate([[0], np.cumsum(new)])
    if c["new"] > 1:
        s["row_start"] = torch.from_numpy(start.astype(np.int32)).cuda()
    # of each row: its sequence, its place among the sequence's new rows, its position
    seq = np.repeat(np.arange(S), new)
    place = np.arange(R) - start[seq]
    for name, v in (("seq", seq), ("place", place), ("pos", kv[seq] - new[seq] + place)):
        s[name] = torch.from_numpy(v).cuda()
    s["q"] = _normal(g, R, c["heads"], hd, std=2.0)
    s["q_out"] = torch.zeros_like(s["q"])
    if c["kind"] == "append":
        s["k_new"], s["v_new"] = _normal(g, R, kvh, hd), _normal(g, R, kvh, hd)
        s["k_back"], s["v_back"] = (torch.zeros(R, kvh, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()  # the framework has a stream of its own
    return s


# ───────────────────────────── one pass ─────────────────────────────

_ctx = None


def _own(s):
    """The framework's context, and what a program keeps: the batch's handle, its pools', the rules'."""
    global _ctx
    from runit_mac_amd import dispatch as d
    if _ctx is None:
        _ctx = d.HipContext()
    c = s["case"]
    p = lambda name: s[name].data_ptr() if name in s and s[name].numel() else None
    if "held" in s:
        return d
    if c["kind"] == "rules":
        seen, bias = c["seen"] > 0, c["biases"] > 0
        s["held"] = d.LogitRules(
            **(dict(tokens=p("token_ids"), n_tokens=s["token_ids"].numel(), token_start=p("token_start"),
                    token_len=p("token_len"), prompt_len=p("prompt_len"), repetition=p("repetition"),
                    frequency=p("frequency"), presence=p("presence")) if seen else {}),
            **(dict(bias_ids=p("bias_ids"), bias=p("bias"), n_bias=s["bias"].numel(), bias_start=p("bias_start"),
                    bias_len=p("bias_len")) if bias else {}),
            **(dict(mask=p("mask"), mask_rows=c["masks"], mask_row=p("mask_row")) if c["masks"] else {}))
    elif c["kind"] == "copy":
        # (a copy asks nothing of sequences)
        s["held"] = d.PagedBatch.array([
            d.PagedBatch(k_pages=k.data_ptr(), v_pages=v.data_ptr(), dtype={4: "q4", 16: "f16", 32: "f32"}[c["bits"]],
                         num_pages=c["pages"], page_size=c["page"], num_kv_heads=c["kv_heads"],
                         head_dim=c["head_dim"], table=None, table_stride=0, n_seqs=0, kv_len=None)
            for k, v in s["pools"]])
    else:
        s["held"] = d.PagedBatch(
            k_pages=s["k"].data_ptr(), v_pages=s["v"].data_ptr(), dtype="q4", num_pages=s["k"].shape[0],
            page_size=c["page"], num_kv_heads=c["kv_heads"], head_dim=c["head_dim"], table=s["table"].data_ptr(),
            table_stride=s["table"].shape[1], n_seqs=c["seqs"], kv_len=s["kv_len"].data_ptr(), rows=s["rows"],
            row_start=s["row_start"].data_ptr() if c["new"] > 1 else None)
    return d


def _run_own(s):
    d, c = _own(s), s["case"]
    if c["kind"] == "rules":
        call = d.adjust_logits_f16 if c["f16"] else d.adjust_logits_f32
        call(_ctx, s["logits"].data_ptr(), s["out"].data_ptr(), c["rows"], c["n"], s["held"])
        return s["out"]
    if c["kind"] == "copy":
        d.paged_copy(_ctx, s["held"], s["src"].data_ptr(), s["dst"].data_ptr(), c["copies"])
        return s["pools"]
    if c["kind"] == "append":
        d.rope_kv_append_paged_f32(_ctx, s["held"], s["q"].data_ptr(), s["k_new"].data_ptr(),
                                   s["v_new"].data_ptr(), s["q_out"].data_ptr(), c["heads"], THETA)
        d.paged_gather_f16(_ctx, s["held"], s["k_back"].data_ptr(), s["v_back"].data_ptr())
        return {"q": s["q_out"], "k": s["k_back"], "v": s["v_back"]}
    if c["shared"]:
        d.shared_prefix_attention_f32(_ctx, s["held"], s["q"].data_ptr(), s["q_out"].data_ptr(), c["heads"],
                                      s["shared_table"].data_ptr(), c["shared"])
    else:
        d.paged_attention_f32(_ctx, s["held"], s["q"].data_ptr(), s["q_out"].data_ptr(), c["heads"])
    return s["q_out"]


def _plain_append(s):
    c, half = s["case"], s["case"]["head_dim"] // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    a = s["pos"].double()[:, None, None] * THETA ** (-2 * i / c["head_dim"])
    cos, sin = a.cos(), a.sin()
    # (in 64 bits: a key next to the border of two codes goes to either)
    turn = lambda t: torch.cat([t[..., :half] * cos - t[..., half:] * sin,
                                t[..., :half] * sin + t[..., half:] * cos], -1)
    page = s["table"][s["seq"], s["pos"] // c["page"]].long()
    slot = s["pos"] % c["page"]
    back = {}
    for name, x in (("k", turn(s["k_new"].double())), ("v", s["v_new"])):
        _store(c, s[name], s[name + "_at"], page, slot, x)
        word, nib, scale = s[name + "_at"]
        at = page[:, None, None], torch.arange(c["kv_heads"], device="cuda")[None, :, None]
        n = s[name][at + (word[slot][:, None],)].int() >> (4 * nib[0]) & 15
        w = s[name][at + (scale[slot][:, None],)].repeat_interleave(32, -1)
        back[name] = ((n - (w.int() & 15)) * (w & ~15).view(torch.float16).float()).half()
    return {"q": turn(s["q"].double()).float(), **back}


def _plain_attention(s):
    c = s["case"]
    S, N, kvh, hd, group = c["seqs"], s["most"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    pages = s["table"].long().clamp_min(0)
    # [sequence][kv head][position][dim]
    k, v = (_read(c, s[x], s[x + "_at"])[pages].transpose(1, 2).reshape(S, kvh, -1, hd) for x in "kv")
    j = torch.arange(k.shape[2], device="cuda")
    there = j[None, :] < s["kv_len"].long()[:, None]
    v = v.masked_fill(~there[:, None, :, None], 0)
    q = torch.zeros(S, kvh, N, group, hd, device="cuda")
    q[s["seq"], :, s["place"]] = s["q"].view(-1, kvh, group, hd)
    pos = torch.full((S, N), -1, device="cuda")
    pos[s["seq"], s["place"]] = s["pos"]
    x = q.view(S, kvh, N * group, hd) @ k.transpose(2, 3).contiguous() / math.sqrt(hd)
    hidden = j[None, None, :] > pos[:, :, None]
    x = x.view(S, kvh, N, group, -1).masked_fill(hidden[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    o = e.view(S, kvh, N * group, -1) @ v / e.view(S, kvh, N * group, -1).sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(S, kvh, N, group, hd)[s["seq"], :, s["place"]].reshape(-1, c["heads"], hd)


def _plain_copy(s):
    # (no page is both copied and written)
    s["pools"][:, :, s["dst"].long()] = s["pools"][:, :, s["src"].long()]
    return s["pools"]


def _plain_rules(s):
    c, x = s["case"], s["logits"].float()
    rows, n = x.shape
    if c["seen"]:
        at = s["token_row"] * n + s["token_ids"].long()
        count = torch.zeros(rows * n, dtype=torch.int32, device="cuda")
        seen = count.index_add(0, at, torch.ones_like(at, dtype=torch.int32)).view(rows, n)
        said = count.index_add(0, at, (s["place"] >= s["prompt_len"].long()[s["token_row"]]).int()).view(rows, n)
        r = s["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * said - s["presence"][:, None] * (said > 0)
    if c["biases"]:
        more = torch.zeros(rows * n, dtype=torch.float64, device="cuda")  # (any order gives the same 32 bits)
        more.index_add_(0, s["bias_row"] * n + s["bias_ids"].long(), s["bias"].double())
        x = x + more.float().view(rows, n)
    if c["masks"]:
        bit = torch.arange(n, device="cuda")
        ok = (s["mask"][:, bit // 32] >> (bit % 32).int() & 1).bool()
        which = s["mask_row"].long()
        x = torch.where((which < 0)[:, None] | ok[which.clamp_min(0)], x, -math.inf)
    return s["out"].copy_(x.to(s["out"].dtype))


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attention": _plain_attention, "copy": _plain_copy,
            "rules": _plain_rules}[state["case"]["kind"]](state)


# ───────────────────────────── cost ─────────────────────────────

def work(case):
    c = case
    if c["kind"] == "rules":
        el, r = 2 if c["f16"] else 4, np.random.default_rng(c["shape"])
        seen, biases = (int(_lists(r, c, m, None)[0].sum()) for m in (c["seen"], c["biases"]))
        n = c["rows"] * c["n"]
        # (in place about half of the logits are written, those that the masks forbid)
        return {"bytes": (n // 2 if c["inplace"] else 2 * n) * el + 4 * seen + 8 * biases + c["masks"] * c["n"] // 8,
                "flops": n}
    if c["kind"] == "copy":
        size = c["kv_heads"] * c["page"] * c["head_dim"] * (4.5 if c["bits"] == 4 else c["bits"]) / 8
        return {"bytes": 2 * c["layers"] * size * (c["copies"] + c["sources"]), "flops": 0}
    new, kv = _sizes(c)
    R, wide = int(new.sum()), c["kv_heads"] * c["head_dim"]
    q = 4 * R * c["heads"] * c["head_dim"]
    if c["kind"] == "append":  # (stored and read back)
        return {"bytes": 2 * q + 2 * R * wide * (4 + 9 / 16 + 2), "flops": 6 * R * (c["heads"] * c["head_dim"] + 2 * wide)}
    seen = int(sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new.tolist(), kv.tolist())))
    held = int(kv.sum()) - (c["seqs"] - 1) * c["shared"]
    return {"bytes": 2 * q + 2 * held * wide * 9 / 16, "flops": 4 * seen * c["heads"] * c["head_dim"]}


# ───────────────────────────── the same in 64 bits ─────────────────────────────

def _exact_rows(c, pages, values):
    """[n][words] of a KV head's part of pages, as [n·page][elements] in 64 bits."""
    ps, hd, n = c["page"], c["head_dim"], pages.shape[0]
    half = ps * hd // 2
    b = pages.contiguous().view(torch.uint8)
    scale = b[:, half:].contiguous().view(torch.int16).long() & 0xFFFF
    nib = torch.stack([b[:, :half] & 15, b[:, :half] >> 4], -1)
    if values:
        w = 1 if hd == 64 else 2
        i = hd // (64 * w)
        # tile, block of elements, four positions, chunk, pair, half of the chunk, position, element
        nib = nib.reshape(n, ps // 16, i, 4, 16, 2, w, 2, 4).permute(0, 1, 3, 5, 7, 2, 4, 6, 8)
        scale = scale.view(n, ps // 16, hd // 32, 16).transpose(2, 3)
    else:
        nib = nib.reshape(n, ps, hd // 8, 2, 4).transpose(3, 4)
    nib, scale = nib.reshape(n * ps, hd // 32, 32).double(), scale.reshape(n * ps, hd // 32)
    m, e = scale >> 4 & 63, scale >> 10 & 31
    step = torch.where(e > 0, (64 + m) * torch.exp2(e - 21.0), m * 2.0 ** -20)
    return ((nib - (scale & 15)[..., None]) * step[..., None]).view(n * ps, hd)


def _exact_attention(s):
    c, ps = s["case"], s["case"]["page"]
    group, out = c["heads"] // c["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    new, kv = _sizes(c)
    r0 = 0
    for i in range(c["seqs"]):
        n, L = int(new[i]), int(kv[i])
        pages = s["table"][i, :-(-L // ps)].long()
        for h in range(c["kv_heads"]):
            k, v = (_exact_rows(c, s[x][pages, h], x == "v")[:L] for x in "kv")
            for a in range(0, n, 64):
                b = min(n, a + 64)
                q = s["q"][r0 + a:r0 + b, h * group:(h + 1) * group].double()
                sc = torch.tensordot(q, k, dims=([2], [1])) / math.sqrt(c["head_dim"])
                p = torch.arange(L - n + a, L - n + b, device="cuda")
                late = torch.arange(L, device="cuda")[None, None, :] > p[:, None, None]
                w = torch.softmax(sc.masked_fill(late, -math.inf), -1)
                out[r0 + a:r0 + b, h * group:(h + 1) * group] = torch.tensordot(w, v, dims=([2], [0]))
        r0 += n
    return out


def _exact_append(s):
    c, hd = s["case"], s["case"]["head_dim"]
    freq = torch.tensor([THETA ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * freq)[:, None]

    def rotate(t):
        z = torch.complex(t[..., :hd // 2].double(), t[..., hd // 2:].double()) * turn
        return torch.cat([z.real, z.imag], -1)

    def held(t):
        g = t.reshape(-1, 32).cpu().numpy().astype(np.float64)
        lo, hi = np.minimum(g.min(1), 0.0), np.maximum(g.max(1), 0.0)
        mant, ex = np.frexp((hi - lo) / 15)  # mant in [1/2, 1): seven bits are its 128ths
        ulp = np.maximum(np.ldexp(1.0, ex - 7), 2.0 ** -20)
        step = np.ceil((hi - lo) / 15 / ulp) * ulp
        some = step > 0
        safe = np.where(some, step, 1.0)
        zero = np.rint(-lo / safe)
        code = np.clip(np.rint(g / safe[:, None]) + zero[:, None], 0, 15)
        return torch.from_numpy(np.where(some, step, 0.0)[:, None] * (code - zero[:, None])).cuda().view(t.shape)

    return {"q": rotate(s["q"]), "k": held(rotate(s["k_new"])), "v": held(s["v_new"].double())}


def _exact_rules(s):
    c, out = s["case"], s["logits"].double().cpu().numpy()
    host = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k not in ("logits", "out")}
    for r in range(c["rows"]):
        x = out[r]
        if c["seen"]:
            ids = host["token_ids"][host["token_start"][r]:][:host["token_len"][r]]
            count = np.bincount(ids[host["prompt_len"][r]:], minlength=c["n"])
            some = np.unique(ids)
            p = host["repetition"][r].astype(np.float64)
            x[some] = np.minimum(x[some] / p, x[some] * p) if p >= 1 else np.maximum(x[some] / p, x[some] * p)
            x -= count * host["frequency"][r].astype(np.float64) + np.sign(count) * host["presence"][r].astype(np.float64)
        if c["biases"]:
            a, k = host["bias_start"][r], host["bias_len"][r]
            np.add.at(x, host["bias_ids"][a:a + k], host["bias"][a:a + k].astype(np.float64))
        if c["masks"] and host["mask_row"][r] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_row"][r]].view(np.uint8), bitorder="little")[:c["n"]]
            x[bits == 0] = -np.inf
    return torch.from_numpy(out)


def exact(case, seed):
    if case["kind"] == "copy":
        return None  # (bits: equal or not)
    s = prepare(case, seed)
    return {"rules": _exact_rules, "append": _exact_append, "attention": _exact_attention}[case["kind"]](s)
