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
