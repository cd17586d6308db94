"""ss_hip_sample_rows against 64 bits. The token has to be the same wherever the
draw and the cutoffs lie more than NEAR from a border (relative to the sum they
are compared with): the call's weights are whole multiples of 2^-44 of the
largest, so a sum of up to 2^19 of them is off by 2^-26 = 1.5e-8 of the largest
at most and by a random walk of that, 2^-35 = 3e-11, in earnest; the largest is
at most the sum. numpy's own running sums are off by 2^19 * 2^-53 = 6e-11. A
draw nearer than that says nothing and is counted; few may be."""
import numpy as np
import pytest

from tests.serving import sample_call, sample_exact

pytestmark = pytest.mark.gpu
NEAR = 1e-9

SETTINGS = [(0.7, 0, 1.0, 0.0), (1.0, 40, 0.9, 0.0), (1.3, 0, 0.5, 0.0), (0.8, 1, 0.999, 0.0), (1.0, 5, 1.0, 0.3),
            (1.1, 0, 1.0, 0.02), (0.6, 2, 0.95, 0.05), (1.5, 1500, 0.95, 0.0), (2.0, 0, 0.999, 1e-4), (1.0, 0, 1e-6, 0.0),
            (0.8, 0, 1.0, 1.0), (0.0, 40, 0.9, 0.1), (-1.0, 0, 1.0, 0.0), (1e-3, 100, 0.9, 0.0)]


def _logits(kind, rows, V, rng):
    x = (rng.standard_normal((rows, V)) * 2.5).astype(np.float32)
    if kind == "peaked":
        x[np.arange(rows), rng.integers(0, V, rows)] += 12.0
    elif kind == "ties":
        x = rng.integers(-3, 3, (rows, V)).astype(np.float32)
    elif kind == "flat":
        x[:] = np.float32(-0.25)
    elif kind == "masked":   # a grammar's mask, NaN among it
        x[rng.random((rows, V)) < 0.9] = -np.inf
        x[rng.random((rows, V)) < 0.05] = np.nan
        x[:, V // 2] = 1.0
    elif kind == "low":      # far below zero, the type's lowest value as a mask
        x -= np.float32(3e4)
        x[:, ::3] = np.finfo(np.float32).min
    return x


def _check(hip, x, setting, u, ld=None):
    got = sample_call(hip, x, setting[0], *setting[1:], u, ld)
    near = 0
    for r in range(x.shape[0]):
        want, gap = sample_exact(x[r], setting[0], *setting[1:], u[r])
        if gap > NEAR:
            assert got[r] == want, (setting, r, got[r], want, u[r], gap)
        else:
            near += 1
            assert 0 <= got[r] < x.shape[1]
    return near


@pytest.mark.parametrize("kind", ["normal", "peaked", "ties", "flat", "masked", "low"])
@pytest.mark.parametrize("rows,V,ld", [(1, 1, 1), (3, 2, 5), (2, 7, 7), (5, 1000, 1003), (2, 1024, 1024), (3, 1025, 1025),
                                       (2, 4097, 4100), (16, 32000, 32000), (3, 128256, 128257), (2, 262144, 262144)])
def test_rows_against_64_bits(hip, kind, rows, V, ld):
    rng = np.random.default_rng([rows, V, len(kind)])
    near = 0
    for setting in SETTINGS:
        print("sample rows", kind, rows, V, ld, setting, flush=True)
        u = rng.random(rows, np.float32)
        if setting == SETTINGS[0]:
            u[0] = 0.0
        near += _check(hip, _logits(kind, rows, V, rng), setting, u, ld)
    # equal logits put every border on a multiple of 1 / n, where a draw of 24 bits may fall
    assert near <= (rows * len(SETTINGS) // 4 if kind in ("ties", "flat") else 1 + rows * len(SETTINGS) // 50)


def test_ends_of_the_random_numbers(hip):
    print("sample rows, ends", flush=True)
    rng = np.random.default_rng(1)
    for V in (100, 5000):
        x = np.repeat(_logits("normal", 1, V, rng), 7, 0)
        u = np.array([0.0, -1.0, np.nan, 1.0 - 2.0 ** -24, 1.0, 2.0, np.inf], np.float32)
        for setting in ((1.0, 0, 1.0, 0.0), (1.0, 10, 0.9, 0.0), (0.7, 0, 0.8, 0.0)):
            got = sample_call(hip, x, *setting, u)
            first = sample_exact(x[0], *setting, 0.0)[0]
            last = sample_exact(x[0], *setting, 1.0)[0]
            assert list(got) == [first] * 3 + [last] * 4, (V, setting, got, first, last)


def test_rows_with_nothing_or_infinite(hip):
    print("sample rows, nothing left", flush=True)
    for V in (9, 3000):
        x = np.zeros((4, V), np.float32)
        x[0] = -np.inf
        x[1] = np.nan
        x[2, [3, 7]] = np.inf            # the infinite ones share the weight
        x[3] = -np.inf
        x[3, V - 1] = np.finfo(np.float32).min
        for setting in ((1.0, 0, 1.0, 0.0), (1.0, 4, 0.9, 0.1), (0.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.5)):
            got = sample_call(hip, x, *setting, np.full(4, 0.75, np.float32))
            assert list(got) == [-1, -1, 3 if setting[0] <= 0 else 7, V - 1], (V, setting, got)


def test_draws_follow_the_weights(hip):
    """Random numbers on a grid give each token as often as its weight asks, within one."""
    print("sample rows, grid", flush=True)
    x = np.repeat(np.log(np.array([[1, 2, 4, 8, 1]], np.float32)), 1600, 0)
    got = sample_call(hip, x, 1.0, 0, 1.0, 0.0, (np.arange(1600) + 0.5) / 1600)
    assert np.all(np.abs(np.bincount(got, minlength=5) - 100 * np.array([1, 2, 4, 8, 1])) <= 1)


@pytest.mark.parametrize("setting", [(6.0, 0, 0.9, 0.0), (6.0, 20000, 1.0, 0.0), (4.0, 30000, 0.7, 0.001), (40.0, 1, 1.0, 0.0),
                                     (40.0, 0, 0.999, 0.0), (9.0, 128000, 0.0, 0.3)], ids=str)
def test_more_entries_near_the_threshold_than_the_list_holds(hip, setting):
    """High temperatures bring tens of thousands of different logits within a quarter of one another."""
    print("sample rows, hot", setting, flush=True)
    rng = np.random.default_rng(int(10 * setting[0]))
    x = (2.5 * rng.standard_normal((5, 128256))).astype(np.float32)
    x[1, ::7] = np.nan
    x[2, ::2] = np.float32(0.5)
    u = rng.random(5, np.float32)
    u[3:] = 0.0, np.float32(1 - 2 ** -24)
    assert _check(hip, x, setting, u) <= 1
