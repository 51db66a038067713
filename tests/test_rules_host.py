"""Rules on a sequence's next token, before a GPU is asked for: what is refused
because no token, or no number, would be left."""
import numpy as np
import pytest

from runit_mac_amd.batch import Rules
from test_batch_fork_host import Ruled
from test_batch_host import CFG, decoder

N = CFG.vocab
only = lambda *t: np.isin(np.arange(N), t)
words = lambda a: Rules(allowed=a).mask(N)


@pytest.mark.parametrize("rules", [
    dict(allowed=only(3, 4), bias={3: -np.inf, 4: -np.inf}),
    dict(allowed=only(3, 4), bias={3: -np.inf, 4: -1e39}),  # (−inf in 32 bits)
    dict(allowed=words(only(3, 4)), bias={4: -1e39, 3: -np.inf, 9: 1.0}),
    dict(bias=dict.fromkeys(range(N), -np.inf)),
    dict(repetition=1e-50), dict(repetition=1e39),          # (0 and inf there)
    dict(frequency=1e39), dict(presence=-1e39),
])
def test_nothing_is_left(rules):
    b = decoder(Ruled)
    s = b.open()
    with pytest.raises(ValueError):
        b.step({s: [1]}, rules={s: Rules(**rules)})
    assert not b.passes and b.length(s) == 0


@pytest.mark.parametrize("rules", [
    dict(allowed=only(3, 4), bias={3: -np.inf}), dict(allowed=only(3, 4), bias={0: -np.inf, 4: -3e38}),
    dict(bias=dict.fromkeys(range(1, N), -np.inf)), dict(allowed=words(only(2)), bias={2: 5.0}),
    dict(repetition=3e38, frequency=-3e38, presence=3e38), dict(repetition=1e-38), dict(bias={3: 1e39}),
])
def test_something_is_left(rules):
    b = decoder(Ruled)
    s = b.open()
    b.step({s: [1]}, rules={s: Rules(**rules)})
    assert b.length(s) == 1


@pytest.mark.parametrize("rules", [dict(allowed=only(3, 4)), dict(allowed=words(only(3, 4))), dict(bias={0: -np.inf}),
                                   dict(bias={0: -1e39}, allowed=only(0, 7))])
def test_no_logit_is_left(rules):
    """Of a row of -inf and NaN the first token is the likeliest: an error where the rules
    forbid it, and the sequences of the call stay as they were."""
    b = decoder(Ruled, num_pages=12)
    s, t = b.open(), b.open()
    b.step({s: [1], t: [2]})
    with pytest.raises(ValueError, match="no token"):
        b.step({s: [5], t: np.append(np.arange(20), N - 1)}, rules={t: Rules(**rules)})  # (N - 1: after it comes 0)
    assert b.length(s) == b.length(t) == 1 and b.pool.free == 10
    assert b.step({s: [N - 1], t: [5]}, rules={t: Rules(frequency=1.0)}) == {s: 0, t: 6}
    assert b.step({t: [N - 1]}, rules={t: Rules(allowed=only(0, 7), bias={0: -3.0})}) == {t: 0}


@pytest.mark.parametrize("rules", [dict(bias={1.5: 1.0}), dict(bias={np.nan: 1.0}), dict(bias={0.25: -np.inf}),
                                   dict(prompt_len=1.5), dict(prompt_len=np.nan)])
def test_numbers_that_are_not_whole(rules):
    b = decoder(Ruled)
    s = b.open()
    with pytest.raises(ValueError):
        b.step({s: [1]}, rules={s: Rules(**rules)})
    assert not b.passes
    b.step({s: [1]}, rules={s: Rules(bias={np.int64(3): 1.0, 4.0: 2.0}, prompt_len=np.uint32(2))})


def test_masks_and_biases_need_no_tokens():
    """A sequence's tokens are counted only where a penalty is for them."""
    b = decoder(Ruled, max_rows=64)
    s, t, u = b.open(), b.open(), b.open()
    mask, bias, neutral = Rules(allowed=only(2, 6, 8)), Rules(bias={6: 1.0}, prompt_len=1), Rules(1.0, -0.0, 1e-50)
    b.step({s: [5, 1], t: [5, 7], u: [9]}, rules={s: mask, t: bias, u: neutral})
    assert b.seen[-1] == [(mask, []), (bias, []), (neutral, [])]
    for r in (Rules(repetition=1.1), Rules(frequency=-0.1), Rules(presence=1e-30)):
        b.step({s: [1], t: [7]}, rules={s: r, t: bias})
        assert b.seen[-1] == [(r, b._seqs[s].tokens.ids), (bias, [])]
