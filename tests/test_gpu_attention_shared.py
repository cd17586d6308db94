"""ss_hip_attention_shared (sequences that continue one prompt) against 64 bits,
over both caches; tolerance in tests/serving.py. Positions past the prefix and
past a sequence's own length hold NaN."""
import numpy as np
import pytest

from tests.serving import TOL, cache, row_err, shared_call, shared_exact, spoil

pytestmark = pytest.mark.gpu

# H, KVH, hd, prefix, own_max, lengths
SHAPES = [
    (4, 4, 64, 0, 1, [1]), (4, 2, 128, 1, 1, [1, 1]), (8, 1, 256, 1, 3, [0, 3]), (32, 8, 128, 0, 7, [0, 7, 1]),
    (32, 4, 64, 200, 35, [32, 1, 17, 35]), (32, 8, 128, 4096, 500, [500, 3, 77, 256, 31, 32, 33, 64]),
    (32, 32, 128, 177, 301, [301, 0, 5, 300, 32]), (64, 8, 128, 900, 65, [1, 2, 3]), (12, 12, 64, 31, 40, [40] * 9),
    (8, 4, 128, 33, 90, [90, 1, 0]), (16, 8, 256, 700, 129, [128, 129, 5]), (8, 1, 256, 64, 33, [33, 32]),
    (32, 8, 128, 5000, 1, [1] * 40), (8, 8, 128, 257, 20, list(range(21)) * 4), (32, 4, 64, 1023, 600, [600, 599, 1]),
    (8, 1, 128, 300, 3000, [3000, 2999, 0, 33]), (16, 2, 128, 2000, 5, [5, 4, 3, 2, 1, 0] * 22),
    # short caches of which one could grow: tiles and shares; at most 16 blocks (32 at head_dim 64): one workgroup for both
    (32, 8, 128, 31, 700, [700, 5, 0]), (4, 4, 64, 1, 1100, [1, 1100]), (8, 2, 128, 33, 600, [0, 1, 32]),
    (4, 4, 64, 33, 1500, [40] * 9), (32, 8, 128, 64, 448, [448, 0, 31, 32, 33]), (32, 4, 64, 900, 96, [96, 95, 0, 1]),
    (8, 8, 128, 1, 30, [0, 1, 30]), (16, 2, 64, 32, 32, [32] * 100), (8, 8, 128, 65, 60, [60, 1] * 32),
]


def _case(kv, H, KVH, hd, p, own_max, lens):
    rng = np.random.default_rng([H, KVH, hd, p, own_max, len(lens), kv])
    prefix = cache(rng, kv, KVH, p + 5, hd)
    spoil(prefix, np.arange(p + 5) >= p)
    own = cache(rng, kv, KVH, own_max, hd, (len(lens),))
    for b, n in enumerate(lens):
        spoil(own, np.arange(own_max) >= n, (b,))
    return rng.standard_normal((len(lens), H, hd)).astype(np.float32), prefix, own


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:5])) + "-x%d" % len(s[5]))
def test_shared_against_64_bits(hip, shape, kv):
    print("shared", shape[:5], len(shape[5]), "kv", kv, flush=True)
    p, lens = shape[3], shape[5]
    q, prefix, own = _case(kv, *shape)
    for cap in (0.0, 30.0):
        err = row_err(shared_call(hip, q, prefix, p, own, lens, cap), shared_exact(q, prefix, p, own, lens, cap))
        print("cap %g worst row %.2e" % (cap, err.max()), flush=True)
        assert err.max() <= TOL


@pytest.mark.parametrize("kv", [0, 1])
def test_lengths_outside_the_cache(hip, kv):
    """Below 0 as 0, above own_max as own_max; nothing seen: zeros; no prefix pointers."""
    print("shared, odd lengths, kv", kv, flush=True)
    q, _, own = _case(kv, 32, 8, 128, 0, 40, [40] * 5)
    lens = [-3, 41, 2 ** 31 - 1, -2 ** 31, 7]
    got, want = shared_call(hip, q, None, 0, own, lens, 0.0), shared_exact(q, None, 0, own, lens, 0.0)
    assert np.all(got[[0, 3]] == 0)
    assert row_err(got, want).max() <= TOL


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("own_max", [40, 700])
def test_a_value_that_is_not_finite_reaches_those_that_see_it(hip, where, bad, own_max):
    print("shared, V not finite", where, bad, own_max, flush=True)
    lens = [20, 40, 3, 17]
    q, prefix, own = _case(0, 32, 8, 128, 50, own_max, lens)
    want = shared_exact(q, prefix, 50, own, lens, 0.0)
    if where == "own":
        own[1][1, :, 39] = bad
        got = shared_call(hip, q, prefix, 50, own, lens, 0.0)
        assert not np.isfinite(got[1]).any()
        assert row_err(got[[0, 2, 3]], want[[0, 2, 3]]).max() <= TOL
    else:
        prefix[1][:, 49, 5] = bad
        got = shared_call(hip, q, prefix, 50, own, lens, 0.0)
        assert not np.isfinite(got[:, :, 5]).any()
        keep = np.arange(128) != 5
        assert row_err(got[:, :, keep], want[:, :, keep]).max() <= TOL


@pytest.mark.parametrize("own_max", [60, 700])
def test_wide_int8_scales(hip, own_max):
    print("shared, wide scales", own_max, flush=True)
    lens = [1, 60, 33, 2]
    q, prefix, own = _case(1, 32, 8, 128, 300, own_max, lens)
    rng = np.random.default_rng(5)
    prefix[3] *= 10.0 ** rng.uniform(-8, 0, prefix[3].shape).astype(np.float32)
    own[3] *= 10.0 ** rng.uniform(-8, 3, own[3].shape).astype(np.float32)
    err = row_err(shared_call(hip, q, prefix, 300, own, lens, 0.0), shared_exact(q, prefix, 300, own, lens, 0.0))
    assert err.max() <= TOL
