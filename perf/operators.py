"""Operators of batched decoding, as cases that can be timed and checked.

Four operators of a batch of sequences whose keys and values live in pages:

* append: the rotary embedding of a ragged batch's new queries and keys, and
  the new keys and values stored into their pages (f32 or f16);
* attention: the causal attention of the batch's rows over those pages, from
  one new row a sequence (a decode step) to prompt chunks;
* shared: the same attention where every sequence begins with one long prefix;
* logprobs: log probabilities of given tokens, with the entropy, the token's
  rank and the most probable alternatives.

Head layouts are those of the 0.5B and 7B Qwen2.5 configurations that bench.py
runs; drawn cases take other sizes of the same ranges.  Where `own` is true
the framework's entry points run, otherwise plain torch operations.
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
        dict(name="append_step_0p5b", kind="append", f16=False, page=16, seqs=4, lo=60, hi=700,
             new=1, shape=1, **HALF),
        # the rows of prompt chunks and decoding sequences together, far positions
        dict(name="append_chunk_7b", kind="append", f16=True, page=64, seqs=12, lo=100, hi=20000,
             new=700, shape=2, **SEVEN),
        # a decode step of three short chats on the 0.5B model: latency
        dict(name="attn_step_0p5b", kind="attention", f16=False, page=16, seqs=3, lo=100, hi=600,
             new=1, shared=0, shape=3, **HALF),
        # a decode step of a serving batch on the 7B model, f16 pages
        dict(name="attn_step_7b", kind="attention", f16=True, page=64, seqs=24, lo=300, hi=8000,
             new=1, shared=0, shape=4, **SEVEN),
        # one sequence with a whole book before it, f32 pages
        dict(name="attn_long_7b", kind="attention", f16=False, page=256, seqs=1, lo=100003,
             hi=100003, new=1, shared=0, shape=5, **SEVEN),
        # drafts to verify on the 0.5B model, f32 pages
        dict(name="attn_verify_0p5b", kind="attention", f16=False, page=32, seqs=9, lo=200, hi=4000,
             new=8, shared=0, shape=6, **HALF),
        # prompt chunks and decoding sequences in one batch, f16 pages
        dict(name="attn_chunk_7b", kind="attention", f16=True, page=32, seqs=6, lo=100, hi=4000,
             new=375, shared=0, shape=7, **SEVEN),
        # many answers to one long document on the 7B model, f16 pages
        dict(name="shared_step_7b", kind="attention", f16=True, page=64, seqs=40, lo=20, hi=600,
             new=1, shared=8192, shape=8, **SEVEN),
        # a system prompt that ends inside a page, drafts to verify, f32 pages
        dict(name="shared_verify_0p5b", kind="attention", f16=False, page=16, seqs=18, lo=5,
             hi=300, new=4, shared=1803, shape=9, **HALF),
        # the tokens drawn in one step of a small batch, with 5 alternatives
        dict(name="logprobs_step", kind="logprobs", f16=False, rows=4, n=151936, top=5),
        # a scored prompt chunk of the 7B model, 20 alternatives
        dict(name="logprobs_prompt", kind="logprobs", f16=False, rows=500, n=152064, top=20),
        # f16 logits of an odd vocabulary, scored without alternatives
        dict(name="logprobs_f16", kind="logprobs", f16=True, rows=93, n=50001, top=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "shared", "shared", "logprobs", "logprobs"))
    if kind == "logprobs":
        n = _log(rng, 1000, 152064)
        return dict(kind=kind, f16=rng.random() < 0.4, rows=_log(rng, 1, min(500, 70_000_000 // n)), n=n,
                    top=rng.choice((0, 1, _log(rng, 2, 50))))
    kv = rng.choice((1, 2, 4, 8))
    c = dict(kind="append" if kind == "append" else "attention", f16=rng.random() < 0.5,
             page=rng.choice((16, 32, 64, 128, 256)), kv_heads=kv, heads=kv * rng.randint(1, 9),
             head_dim=rng.choice((64, 64, 128, 128, 256)), shape=rng.randrange(1 << 20))
    wide = c["kv_heads"] * c["head_dim"]
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
    most = 25_000_000 // (wide * c["seqs"])  # positions a sequence, by its memory ...
    most = max(64, min(most, 80_000_000 // (c["seqs"] * c["new"] * c["heads"]),  # ... and by the scores,
                       5_000_000_000 // (rows * c["heads"] * c["head_dim"])))    # ... and the products
    if kind == "shared":
        c["shared"] = _log(rng, 33, max(34, min(8192, most * 3 // 4)))
        if rng.random() < 0.6:
            c["shared"] = max(c["page"], c["shared"] // c["page"] * c["page"])
        c["lo"], top = _log(rng, 1, 30), max(31, min(600, most // 4))
    else:
        c["lo"], top = _log(rng, 1, 300), max(301, min(60000, most))
    c["hi"] = _log(rng, c["lo"], top)
    return c


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


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=c)
    if c["kind"] == "logprobs":
        x = _normal(g, c["rows"], c["n"], std=2.5)
        s["tokens"] = torch.randint(0, c["n"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        likely = torch.rand(c["rows"], generator=g, device="cuda") < 0.7
        s["tokens"] = torch.where(likely, x.argmax(1).int(), s["tokens"])
        s["logits"] = x.half() if c["f16"] else x
        f = lambda *shape, t=torch.float32: torch.empty(shape, device="cuda", dtype=t)
        s["out"] = dict(logprob=f(c["rows"]), entropy=f(c["rows"]), rank=f(c["rows"], t=torch.int32))
        if c["top"]:
            s["out"].update(top_ids=f(c["rows"], c["top"], t=torch.int32), top_logprobs=f(c["rows"], c["top"]))
        torch.cuda.synchronize()
        return s
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
    dt = torch.float16 if c["f16"] else torch.float32
    s["k"], s["v"] = (_normal(g, total, kvh, ps, hd).to(dt) for _ in range(2))
    s["table"] = torch.from_numpy(table).cuda()
    if shared:
        s["shared_table"] = torch.from_numpy(order[:first].astype(np.int32)).cuda()
        if shared % ps:  # the last page of the prefix, copied as each sequence went on behind it
            for p in (s["k"], s["v"]):
                p[s["table"][:, whole].long(), :, :shared % ps] = p[int(order[whole]), :, :shared % ps]
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
    torch.cuda.synchronize()  # the framework has a stream of its own
    return s


# ───────────────────────────── one pass ─────────────────────────────

_ctx = None


def _own(s):
    """The framework's context, and the batch's handle, which a program keeps with its pages."""
    global _ctx
    from runit_mac_amd import dispatch as d
    if _ctx is None:
        _ctx = d.HipContext()
    c = s["case"]
    if c["kind"] != "logprobs" and "batch" not in s:
        s["batch"] = d.PagedBatch(
            k_pages=s["k"].data_ptr(), v_pages=s["v"].data_ptr(), dtype="f16" if c["f16"] else "f32",
            num_pages=s["k"].shape[0], page_size=c["page"], num_kv_heads=c["kv_heads"],
            head_dim=c["head_dim"], table=s["table"].data_ptr(), table_stride=s["table"].shape[1],
            n_seqs=c["seqs"], kv_len=s["kv_len"].data_ptr(), rows=s["rows"],
            row_start=s["row_start"].data_ptr() if c["new"] > 1 else None)
    return d


def _run_own(s):
    d, c = _own(s), s["case"]
    if c["kind"] == "logprobs":
        o = s["out"]
        p = lambda name: o[name].data_ptr() if name in o else None
        call = d.token_logprobs_f16 if c["f16"] else d.token_logprobs_f32
        call(_ctx, s["logits"].data_ptr(), s["tokens"].data_ptr(), c["rows"], c["n"], p("logprob"),
             entropy=p("entropy"), rank=p("rank"), top=c["top"], top_ids=p("top_ids"),
             top_logprobs=p("top_logprobs"))
        return o
    if c["kind"] == "append":
        d.rope_kv_append_paged_f32(_ctx, s["batch"], s["q"].data_ptr(), s["k_new"].data_ptr(),
                                   s["v_new"].data_ptr(), s["q_out"].data_ptr(), c["heads"], THETA)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if c["shared"]:
        d.shared_prefix_attention_f32(_ctx, s["batch"], s["q"].data_ptr(), s["q_out"].data_ptr(), c["heads"],
                                      s["shared_table"].data_ptr(), c["shared"])
    else:
        d.paged_attention_f32(_ctx, s["batch"], s["q"].data_ptr(), s["q_out"].data_ptr(), c["heads"])
    return s["q_out"]


def _plain_append(s):
    c, half = s["case"], s["case"]["head_dim"] // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    a = s["pos"].double()[:, None, None] * THETA ** (-2 * i / c["head_dim"])
    cos, sin = a.cos().float(), a.sin().float()
    turn = lambda t: torch.cat([t[..., :half] * cos - t[..., half:] * sin,
                                t[..., :half] * sin + t[..., half:] * cos], -1)
    page = s["table"][s["seq"], s["pos"] // c["page"]].long()
    slot = s["pos"] % c["page"]
    s["k"][page, :, slot] = turn(s["k_new"]).to(s["k"].dtype)
    s["v"][page, :, slot] = s["v_new"].to(s["v"].dtype)
    return {"q": turn(s["q"]), "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    c = s["case"]
    S, N, kvh, hd, group = c["seqs"], s["most"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    pages = s["table"].long().clamp_min(0)
    # [sequence][kv head][position][dim]
    k, v = (p[pages].transpose(1, 2).reshape(S, kvh, -1, hd).float() for p in (s["k"], s["v"]))
    j = torch.arange(k.shape[2], device="cuda")
    there = j[None, :] < s["kv_len"].long()[:, None]
    v = v.masked_fill(~there[:, None, :, None], 0)
    q = torch.zeros(S, kvh, N, group, hd, device="cuda")
    q[s["seq"], :, s["place"]] = s["q"].view(-1, kvh, group, hd)
    pos = torch.full((S, N), -1, device="cuda")
    pos[s["seq"], s["place"]] = s["pos"]
    x = q.view(S, kvh, N * group, hd) @ k.transpose(2, 3) / math.sqrt(hd)
    hidden = j[None, None, :] > pos[:, :, None]
    x = x.view(S, kvh, N, group, -1).masked_fill(hidden[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    o = e.view(S, kvh, N * group, -1) @ v / e.view(S, kvh, N * group, -1).sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(S, kvh, N, group, hd)[s["seq"], :, s["place"]].reshape(-1, c["heads"], hd)


def _plain_logprobs(s):
    c, x = s["case"], s["logits"].float() + 0.0  # (one zero)
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1)
    z = torch.log(total)
    xt = x.gather(1, s["tokens"].long()[:, None])
    o = dict(logprob=(xt - m)[:, 0] - z, entropy=z + (e * (m - x)).sum(1) / total,
             rank=(x > xt).sum(1).int())
    if c["top"]:
        # whole numbers in the order of the floats, the index below them: no two alike
        b = x.view(torch.int32)
        b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
        key = (b << 20) + (c["n"] - 1 - torch.arange(c["n"], device="cuda"))
        ids = c["n"] - 1 - (key.topk(c["top"], 1).values & 0xFFFFF)
        o.update(top_ids=ids.int(), top_logprobs=x.gather(1, ids) - m - z[:, None])
    return o


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "append":
        return _plain_append(state)
    return _plain_logprobs(state) if kind == "logprobs" else _plain_attention(state)


# ───────────────────────────── cost ─────────────────────────────

def work(case):
    c = case
    if c["kind"] == "logprobs":
        n = c["rows"] * c["n"]
        return {"bytes": n * (2 if c["f16"] else 4) + c["rows"] * (16 + 8 * c["top"]), "flops": 6 * n}
    new, kv = _sizes(c)
    R, el, wide = int(new.sum()), 2 if c["f16"] else 4, c["kv_heads"] * c["head_dim"]
    q = 4 * R * c["heads"] * c["head_dim"]
    if c["kind"] == "append":
        return {"bytes": 2 * q + 2 * R * wide * (4 + el), "flops": 3 * R * (c["heads"] * c["head_dim"] + wide)}
    seen = int(sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new.tolist(), kv.tolist())))
    held = int(kv.sum()) - (c["seqs"] - 1) * c["shared"]
    return {"bytes": 2 * q + 2 * held * wide * el, "flops": 4 * seen * c["heads"] * c["head_dim"]}


# ───────────────────────────── the same in 64 bits ─────────────────────────────

def _exact_attention(s):
    c, ps = s["case"], s["case"]["page"]
    group, out = c["heads"] // c["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    new, kv = _sizes(c)
    r0 = 0
    for i in range(c["seqs"]):
        n, L = int(new[i]), int(kv[i])
        pages = s["table"][i, :-(-L // ps)].long()
        for h in range(c["kv_heads"]):
            k, v = (p[pages, h].reshape(-1, c["head_dim"])[:L].double() for p in (s["k"], s["v"]))
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

    k, v = s["k"].double(), s["v"].double()
    flat = s["table"][s["seq"], s["pos"] // c["page"]].long() * c["page"] + s["pos"] % c["page"]
    for pool, rows in ((k, rotate(s["k_new"])), (v, s["v_new"].double())):
        rows_of = pool.transpose(1, 2).reshape(-1, c["kv_heads"], hd)
        rows_of[flat] = rows
        pool.copy_(rows_of.view(pool.shape[0], c["page"], c["kv_heads"], hd).transpose(1, 2))
    return {"q": rotate(s["q"]), "k": k, "v": v}


def _exact_logprobs(s):
    c, o = s["case"], []
    for x, t in zip(s["logits"], s["tokens"].long()):
        lp = torch.log_softmax(x.double(), 0)
        row = [lp[t], -(lp.exp() * lp).sum(), lp.sort(descending=True).values[:c["top"]]]
        o.append(row)
    got = dict(logprob=torch.stack([r[0] for r in o]), entropy=torch.stack([r[1] for r in o]), rank=None)
    if c["top"]:
        got.update(top_ids=None, top_logprobs=torch.stack([r[2] for r in o]))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(s)
    return _exact_append(s) if case["kind"] == "append" else _exact_attention(s)
