"""Every compiled form of the rotary append and of the attention, against float64: head sizes that fill a form's registers and that do
not, each type pair, and calls large enough to go past the caches.  The rules that choose a form are restated here, so that a case
that moves to another form is noticed."""
import numpy as np
import pytest

import test_paged_gpu
from test_paged_gpu import _attend, _compare

pytestmark = pytest.mark.gpu

PAIRS = [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "float32"), ("float32", "bfloat16")]
DIMS = [8, 40, 64, 80, 96, 128, 136, 192, 256]          # forms of 64, 128 and 256: padded and full ones
UNITS = 256


def _is_few(lens, heads, kvh, kind):
    """Single float32 rows and chunks, and small 16-bit calls, take the few-rows form (with hints)."""
    rows, keys = max(n for _, n in lens), max(c + n for c, n in lens)
    return kind == "float32" or (rows * (heads // kvh) <= 16 and keys <= 1024 and len(lens) * kvh <= UNITS)


@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 140)])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("kind,cache", PAIRS)
def test_few_rows(kind, cache, dim, window, sinks):
    """Single rows over several steps of keys, key heads shared by up to 16 rows; the window leaves whole steps out."""
    for lens, heads, kvh in (([(900, 1), (5, 1), (130, 1), (0, 1)], 4, 2), ([(517, 1), (64, 1)], 16, 1), ([(700, 3), (2, 2)], 4, 1)):
        assert _is_few(lens, heads, kvh, kind)
        _compare(*_attend(lens, heads, kvh, dim, 16, kind, cache, window, sinks), kind, dim)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("cache", ["float32", "bfloat16"])
def test_chunks_of_float_rows(cache, dim):
    """Float32 rows have the few-rows form alone: tiles of 16 packed rows at the causal edge, with and without a window."""
    for window, sinks in ((0, 0), (50, 20)):
        _compare(*_attend([(200, 40), (0, 19), (90, 1)], 4, 2, dim, 24, "float32", cache, window, sinks), "float32", dim)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
def test_chunks(kind, dim):
    lens = [(300, 70), (0, 150), (90, 1)]
    assert not _is_few(lens, 4, 2, kind)
    for window, sinks in ((0, 0), (100, 40)):
        _compare(*_attend(lens, 4, 2, dim, 24, kind, kind, window, sinks), kind, dim)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("lens", [[(100, 6), (30, 1)], [(100, 60), (30, 1)]])
def test_values_that_are_not_finite(kind, cache, dim, lens):
    """Keys and values that only the last rows see hold NaN and infinities, at the head's first and last places."""
    def poison(k, v, table, page, total):
        j = total[0] - 2
        at = table[0, j // page], j % page
        v[at][0, 0], v[at][0, dim - 1], v[at][1, dim // 2] = np.nan, np.inf, -np.inf
        j = total[0] - 1
        at = table[0, j // page], j % page
        k[at][0, dim - 1] = np.nan
        v[at][1, dim - 2] = np.inf

    _compare(*_attend(lens, 4, 2, dim, 16, kind, cache, 0, 0, poison=poison), kind, dim)


@pytest.mark.parametrize("dim", [64, 96, 128, 200, 256])
@pytest.mark.parametrize("kind,cache", PAIRS)
def test_splits(kind, cache, dim):
    """Long contexts cut into splits and merged."""
    _compare(*_attend([(6000, 1), (20, 1)], 4, 2, dim, 16, kind, cache, 0, 0), kind, dim)
    _compare(*_attend([(5000, 5)], 2, 2, dim, 16, kind, cache, 2500, 10), kind, dim)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("rot", [128, 64])
def test_rotary_past_the_caches(kind, cache, inter, rot):
    rows, heads, kvh, dim = 4100, 12, 4, 128
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    assert rows * dim * (2 * heads * size[kind] + 2 * kvh * (size[kind] + size[cache])) > 32 << 20
    test_paged_gpu.test_rotary_append((rows, heads, kvh, dim, rot, inter, kind, cache, 16, 3, 1.25), "fused")
