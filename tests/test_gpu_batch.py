"""Sequences decoded together (BatchDecoder) against the CPU reference model
stepped through each of them alone."""
import numpy as np
import pytest

import oracle_lib as ora
from runit_mac_amd.batch import BatchDecoder
from runit_mac_amd.decode import Q4K_M, DecodeConfig, DecodeModel

pytestmark = pytest.mark.gpu

SMALL = dict(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, ff=1024, vocab=1000, max_seq=160)
TINY = dict(layers=2, hidden=896, heads=14, kv_heads=2, head_dim=64, ff=1024, vocab=2000, max_seq=160)


def host_logits(host, tokens):
    return np.stack([host.step(int(t), i, threads=8)[1] for i, t in enumerate(tokens)]).astype(np.float64)


def tolerance(logits, kv):
    """Of a logit: 1e-3 of the row's spread as for the single sequence's
    batched pass, whose projections these are; f16 pages add roundings of
    2^-11 to each key and value.  A value's changes the attention's output by
    2^-11 of it, a key's the scores by 2^-11·Σ|q·k|/√hd — below 4 with
    weights of N(0, 0.02) and normalised inputs —, the output by twice that:
    9·2^-11 a layer, two layers, 9e-3."""
    return (1e-3 + (9e-3 if kv == "f16" else 0.0)) * (logits.max(-1) - logits.min(-1))


def check_scores(got, logits, tokens, kv):
    """logits: of the rows that predict `tokens`.  A log probability moves by
    at most twice a logit's tolerance; likewise its place among the sorted."""
    m = logits.max(-1, keepdims=True)
    lp = logits - m - np.log(np.exp(logits - m).sum(-1, keepdims=True))
    tol = 2 * tolerance(logits, kv) + 1e-5
    assert np.array_equal(got.tokens, tokens)
    rows = np.arange(len(tokens))
    assert np.all(np.abs(got.logprob - lp[rows, tokens]) <= tol)
    best = -np.sort(-lp, axis=-1)[:, :got.top_ids.shape[1]]
    assert np.all(np.abs(got.top_logprobs - best) <= tol[:, None])
    assert np.all(np.abs(got.top_logprobs - np.take_along_axis(lp, got.top_ids.astype(np.int64), -1)) <= tol[:, None])
    own = lp[rows, tokens][:, None]
    assert np.all((lp > own + 2 * tol[:, None]).sum(-1) <= got.rank)
    assert np.all((lp > own - 2 * tol[:, None]).sum(-1) >= got.rank)
    # |d entropy| <= max |d ln p|·(1 + ...): Σ|Δp||ln p| + Σp|Δ ln p|, with |Δp| <= p·(e^tol − 1)
    ent = -(np.exp(lp) * lp).sum(-1)
    assert np.all(np.abs(got.entropy - ent) <= np.expm1(tol) * ent + tol + 1e-5)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("quant,cfg_kw,max_rows", [(None, TINY, 24), (Q4K_M, SMALL, 512), (Q4K_M, SMALL, 3)])
def test_scores_of_sequences_together(ctx, quant, cfg_kw, max_rows, kv):
    """Three sequences, in one call then each alone, in passes that cut them
    anywhere: every token's scores are those of the sequence by itself."""
    cfg = DecodeConfig(**cfg_kw)
    m = DecodeModel(ctx, cfg, seed=21, quant=quant)
    host = ora.HostStepModel.from_recipe(m)
    rng = np.random.default_rng(4)
    b = BatchDecoder(m, 3, 30, 16, kv=kv, max_rows=max_rows, max_logits=17, max_top=5)
    toks = [rng.integers(cfg.vocab, size=n) for n in (33, 2, 50)]
    more = [rng.integers(cfg.vocab, size=n) for n in (1, 4, 20)]
    seqs = [b.open() for _ in toks]
    got = b.score(dict(zip(seqs, toks)), top=5)
    again = b.score(dict(zip(seqs, more)), top=3)
    for s, t, u in zip(seqs, toks, more):
        ref = host_logits(host, np.concatenate([t, u]))
        check_scores(got[s], ref[:len(t) - 1], t[1:], kv)
        check_scores(again[s], ref[len(t):-1], u[1:], kv)
        assert b.length(s) == len(t) + len(u)
    b.free(), m.free()


@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_steps_and_a_shared_prompt(ctx, kv):
    """Sequences behind a common prompt (that ends inside a page), stepped
    together token by token, against each of them whole."""
    cfg = DecodeConfig(**SMALL)
    m = DecodeModel(ctx, cfg, seed=5, quant=Q4K_M)
    host = ora.HostStepModel.from_recipe(m)
    rng = np.random.default_rng(6)
    b = BatchDecoder(m, 7, 40, 16, kv=kv, max_rows=64, max_top=4)
    prefix = rng.integers(cfg.vocab, size=37)
    b.share_prefix(prefix)
    seqs = [b.open() for _ in range(7)]
    history = {s: list(prefix) for s in seqs}
    for i in range(6):
        work = {s: rng.integers(cfg.vocab, size=1 + (i * s) % 3 if i < 3 else 1) for s in seqs[:7 - i]}
        got = b.step(work, top=4)
        for s, t in work.items():
            history[s] += list(t)
            ref = host_logits(host, history[s])[-1:]
            token, scores = got[s]
            assert token == scores.top_ids[0, 0] and scores.rank[0] == 0
            check_scores(scores, ref, np.array([token]), kv)
    b.free(), m.free()


def test_few_rows_of_a_large_model(ctx):
    """Passes of one to five rows where the hidden size takes them to the
    batched GEMMs: steps of one sequence and of three, a draft to verify."""
    cfg = DecodeConfig(layers=2, hidden=1280, heads=10, kv_heads=2, head_dim=128, ff=1536, vocab=1000, max_seq=64)
    m = DecodeModel(ctx, cfg, seed=11, quant=Q4K_M)
    assert m.row_form(1) == m.row_form(5) == "gemm"
    host = ora.HostStepModel.from_recipe(m)
    rng = np.random.default_rng(12)
    b = BatchDecoder(m, 3, 12, 16, kv="f32", max_rows=8, max_top=4)
    seqs = [b.open() for _ in range(3)]
    history = {s: [] for s in seqs}
    for sizes in ((1,), (1, 1, 1), (2, 1, 2), (4,), (1, 1, 1)):
        work = {s: rng.integers(cfg.vocab, size=n) for s, n in zip(seqs, sizes)}
        got = b.step(work, top=4)
        for s, t in work.items():
            history[s] += list(t)
            token, scores = got[s]
            assert token == scores.top_ids[0, 0] and scores.rank[0] == 0
            check_scores(scores, host_logits(host, history[s])[-1:], np.array([token]), "f32")
    s = seqs[0]
    before = b.length(s)
    kept, following = b.verify({s: (3, [4, 5])})[s]
    logits = host_logits(host, history[s] + [3, 4, 5])[-3:]
    fits = [np.flatnonzero(x >= x.max() - 2 * tolerance(x, "f32")) for x in logits]
    assert all([4, 5][i] in fits[i] for i in range(kept)) and following in fits[kept]
    assert b.length(s) == before + 1 + kept
    b.free(), m.free()


def test_verify_of_several_sequences(ctx):
    """Drafts that the reference model would have decoded are kept up to the
    first that no logits within the tolerance allow, and the sequence goes on
    from there as if that had not been."""
    cfg = DecodeConfig(**TINY)
    m = DecodeModel(ctx, cfg, seed=8)
    host = ora.HostStepModel.from_recipe(m)
    rng = np.random.default_rng(9)
    b = BatchDecoder(m, 2, 24, 16, kv="f32", max_rows=64, max_top=2)
    work, seen, wrong = {}, {}, {}
    for n, bad in ((20, None), (9, 2)):
        s = b.open()
        seen[s] = list(rng.integers(cfg.vocab, size=n))
        path = list(seen[s])
        for i in range(6):
            logits = host_logits(host, path)[-1]
            path.append(int(np.argmin(logits) if i - 1 == bad else np.argmax(logits)))
        b.step({s: seen[s]})
        work[s], wrong[s] = (path[n], path[n + 1:]), bad
    got = b.verify(work)
    for s, (kept, following) in got.items():
        token, drafts = work[s]
        logits = host_logits(host, seen[s] + [token] + drafts)[len(seen[s]):]
        fits = [np.flatnonzero(x >= x.max() - 2 * tolerance(x, "f32")) for x in logits]
        sure = next((i for i, f in enumerate(fits) if len(f) > 1), len(fits))  # (drafts with one answer)
        assert kept >= min(sure, len(drafts) if wrong[s] is None else wrong[s])
        assert kept <= (len(drafts) if wrong[s] is None else wrong[s])
        assert all(drafts[i] in fits[i] for i in range(kept)) and following in fits[kept]
        assert b.length(s) == len(seen[s]) + 1 + kept
        # on behind the kept ones: the forgotten rows are overwritten
        scores = b.score({s: [following, 3, 4, 5]}, top=2)[s]
        ref = host_logits(host, seen[s] + [token] + drafts[:kept] + [following, 3, 4, 5])
        check_scores(scores, ref[-4:-1], np.array([3, 4, 5]), "f32")
    b.free(), m.free()
