"""The tests' own codes of 4 bits, and what the library refuses of them before a GPU
is asked for."""
import numpy as np
import pytest

from q4_ref import decode, encode, pack, step, unpack, up7
from runit_mac_amd import dispatch as d


def test_values_are_exact_in_f16_and_near():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((400, 64)) * 2.0 ** rng.integers(-26, 15, (400, 1))
    x[::3, 5] *= 30
    x[1::7] = np.abs(x[1::7])
    x = np.clip(x, -32768, 32768)
    n, w = encode(x)
    y = decode(n, w)
    assert np.array_equal(y.astype(np.float16).astype(np.float64), y)
    assert np.all(np.abs(y - x) <= np.repeat(step(w), 32, -1) / 2 * (1 + 1e-9))


def test_groups_that_nothing_holds():
    x = np.zeros((4, 32))
    x[1, 3], x[2, 3], x[3, 3] = np.inf, np.nan, 32769
    n, w = encode(x)
    y = decode(n, w)
    assert np.all(y[0] == 0) and np.all(np.isnan(y[1:]))


def test_steps():
    assert np.array_equal(up7(np.array([1.0, 1 + 2 ** -7, 1.9999, 3 * 2.0 ** -21, 0.0])),
                          [1.0, 1 + 2 ** -6, 2.0, 2 * 2.0 ** -20, 0.0])


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("values", [False, True])
def test_pages_are_permutations(hd, values):
    rng = np.random.default_rng(hd)
    n, w = rng.integers(0, 16, (48, hd), np.uint8), rng.integers(0, 1 << 16, (48, hd // 32), np.uint16)
    part = pack(n, w, values)
    assert part.size == d.PagedBatch.page_bytes("q4", 1, 48, hd)
    a, b = unpack(part, 48, hd, values)
    assert np.array_equal(a, n) and np.array_equal(b, w)
    # no byte is two positions'
    for p in (0, 17, 47):
        m, u = n.copy(), w.copy()
        m[p] ^= 15
        u[p] ^= 1
        assert np.sum(pack(m, u, values) != part) == hd // 2 + hd // 32


def test_types_of_pages():
    b = d.PagedBatch(16, 32, "q4", 1, 16, 1, 64, None, 0, 0, None)
    assert b.f16 == 4
    a = d.PagedBatch.array([b, b])
    assert len(a) == 2 and a[1].f16 == 4 and a[0].k_pages == 16
    with pytest.raises(ValueError):
        d.PagedBatch(16, 32, "q8", 1, 16, 1, 64, None, 0, 0, None)


@pytest.mark.parametrize("call", [
    lambda lib: lib.rt_paged_gather_f32(None, None, None, None),
    lambda lib: lib.rt_paged_gather_f16(None, None, None, None),
    lambda lib: lib.rt_paged_copy(None, None, 1, None, None, 1),
    lambda lib: lib.rt_adjust_logits_f32(None, None, None, 1, 1, 1, None),
    lambda lib: lib.rt_adjust_logits_f16(None, None, None, 1, 1, 1, None),
])
def test_no_context(call):
    lib = d.load_library()
    assert call(lib) == 5 and b"null context" in lib.rt_global_last_error()
