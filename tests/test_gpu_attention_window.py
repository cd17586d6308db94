"""ss_hip_attention_window (sliding window, first tokens that stay visible)
against 64 bits, over both caches; tolerance in tests/serving.py. Positions that
no token of the call sees hold NaN."""
import numpy as np
import pytest

from tests.serving import TOL, cache, row_err, spoil, window_call, window_exact, window_seen

pytestmark = pytest.mark.gpu

# H, KVH, hd, pos0, tokens, window, sinks
SHAPES = [
    (4, 4, 64, 0, 1, 1, 0), (4, 2, 128, 0, 1, 100, 4), (8, 1, 256, 1, 1, 1, 1), (32, 8, 128, 2, 1, 1, 1),   # a few positions
    (32, 4, 64, 99, 1, 2048, 4), (32, 8, 128, 4096, 1, 1024, 4), (16, 8, 256, 700, 1, 333, 37),             # decode
    (32, 32, 128, 9000, 1, 8192, 64), (12, 12, 64, 5000, 1, 31, 33), (64, 8, 128, 3000, 1, 2999, 5),
    (32, 8, 128, 40, 1, 32, 10), (32, 8, 128, 40, 1, 31, 9), (32, 8, 128, 40, 1, 30, 8),                    # sinks meet the window
    (8, 8, 64, 300, 2, 17, 3), (32, 8, 128, 500, 3, 64, 4), (8, 4, 128, 100, 4, 1, 0), (32, 4, 64, 77, 5, 200, 4),
    (8, 1, 256, 333, 7, 100, 33), (32, 8, 128, 2047, 8, 1000, 4), (64, 8, 128, 900, 2, 300, 1),             # a few tokens
    (4, 4, 128, 0, 33, 8, 2), (32, 8, 128, 300, 40, 100, 4), (32, 4, 64, 31, 34, 500, 100), (8, 2, 128, 57, 70, 33, 1),
    (16, 8, 256, 500, 45, 129, 5), (12, 12, 64, 1000, 65, 1, 0), (32, 8, 128, 5, 130, 31, 200),             # prompts
    (128, 32, 128, 3, 79, 40, 4), (8, 1, 256, 126, 129, 64, 0), (32, 32, 64, 64, 257, 96, 32),
]


def _case(kv, H, KVH, hd, pos0, n, window, sinks, seed=0):
    rng = np.random.default_rng([H, KVH, hd, pos0, n, window, sinks, kv, seed])
    c = cache(rng, kv, KVH, pos0 + n + 5, hd)
    hidden = np.ones(pos0 + n + 5, bool)
    hidden[:pos0 + n] = ~window_seen(pos0, n, window, sinks).any(0)
    spoil(c, hidden)
    return rng.standard_normal((n, H, hd)).astype(np.float32), c


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_window_against_64_bits(hip, shape, kv):
    print("window", shape, "kv", kv, flush=True)
    H, KVH, hd, pos0, n, window, sinks = shape
    q, c = _case(kv, *shape)
    for cap in (0.0, 30.0):
        err = row_err(window_call(hip, q, c, pos0, window, sinks, cap), window_exact(q, c, pos0, window, sinks, cap))
        print("cap %g worst row %.2e" % (cap, err.max()), flush=True)
        assert err.max() <= TOL


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("shape", [(32, 8, 128, 200, 1), (32, 4, 64, 90, 6), (16, 8, 256, 60, 40)])
def test_wide_window_is_plain_attention(hip, shape, kv):
    """A window past the sequence, up to the largest number, and sinks past it: every earlier position."""
    print("wide window", shape, "kv", kv, flush=True)
    H, KVH, hd, pos0, n = shape
    q, c = _case(kv, H, KVH, hd, pos0, n, pos0 + n, 0)
    want = window_exact(q, c, pos0, pos0 + n, 0, 0.0)
    for window, sinks in ((pos0 + n, 0), (2 ** 31 - 1, 0), (1, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert row_err(window_call(hip, q, c, pos0, window, sinks, 0.0), want).max() <= TOL


@pytest.mark.parametrize("shape", [(32, 8, 128, 300, 5, 40, 4), (32, 8, 128, 300, 45, 40, 4), (8, 4, 64, 100, 40, 20, 0),
                                   (16, 8, 256, 100, 3, 20, 1), (16, 8, 256, 100, 33, 20, 1)])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_a_value_that_is_not_finite_stays_with_the_rows_that_see_it(hip, shape, bad):
    print("window, V not finite", shape, bad, flush=True)
    H, KVH, hd, pos0, n, window, sinks = shape
    q, c = _case(0, *shape)
    want = window_exact(q, c, pos0, window, sinks, 0.0)
    first, last = pos0 - window + 1, pos0 + n - 1   # the first row's oldest position, the last row's own
    c[1][:, first] = bad
    c[1][:, last] = bad
    seen = window_seen(pos0, n, window, sinks)[:, [first, last]].any(1)
    assert seen.any() and not seen.all()
    got = window_call(hip, q, c, pos0, window, sinks, 0.0)
    assert not np.isfinite(got[seen]).any()
    assert row_err(got[~seen], want[~seen]).max() <= TOL


@pytest.mark.parametrize("tokens", [1, 4, 40])
def test_wide_int8_scales(hip, tokens):
    """V scales spread over 8 decades: a row's precision goes by what it sees."""
    print("window, wide scales", tokens, flush=True)
    shape = (32, 8, 128, 500, tokens, 100, 4)
    q, c = _case(1, *shape)
    c[3] *= 10.0 ** np.random.default_rng(tokens).uniform(-8, 0, c[3].size).astype(np.float32)
    if tokens > 1:
        c[3][500 + tokens - 1] = 1e6   # the last row's alone
    got, want = window_call(hip, q, c, 500, 100, 4, 0.0), window_exact(q, c, 500, 100, 4, 0.0)
    assert row_err(got, want).max() <= TOL


def test_offsets_past_32_bits(hip):
    """A cache of 9 million positions: 2.3 GB of one head's K, the tokens at its end."""
    print("window, long cache", flush=True)
    max_seq, hd, window, sinks = 9_000_000, 128, 45, 4
    rng = np.random.default_rng(3)
    for n in (1, 12):
        pos0 = max_seq - n
        at = np.r_[0:sinks, pos0 - window + 1:max_seq]
        q = rng.standard_normal((n, 4, hd)).astype(np.float32)
        small = cache(rng, 0, 1, at.size, hd)
        big = [hip.buf(2 * hd * max_seq) for _ in "kv"]
        for b, z in zip(big, small[:2]):
            for lo, part in ((0, z[0, :sinks]), (pos0 - window + 1, z[0, sinks:])):
                part = np.ascontiguousarray(part)
                assert hip.L.ss_hip_memcpy_h2d(hip.ctx, b.ptr + 2 * hd * lo, part.ctypes.data, part.nbytes) == 0
        out, qd = hip.buf(q.nbytes), hip.upload(q)
        nb = hip.L.ss_hip_attention_window_workspace(hip.ctx, 4, 1, hd, n, window, sinks)
        ws = hip.buf(nb + 16)
        rc = hip.L.ss_hip_attention_window(hip.ctx, out.ptr, qd.ptr, big[0].ptr, big[1].ptr, None, None, 4, 1, hd, max_seq, pos0,
                                           n, window, sinks, 0.0, 0, ws.ptr, nb, None)
        assert rc == 0, hip.err()
        got = out.read(np.float32, q.size).reshape(q.shape)
        for b in big + [out, qd, ws]:
            b.free()
        # the same rows over the positions alone, moved together
        i, j = np.arange(pos0, max_seq)[:, None], at[None, :]
        seen = (j <= i) & ((i - j < window) | (j < sinks))
        from tests.serving import attend, values
        k, v = values(small, 0, slice(None))
        want = np.stack([attend(q[:, h], k, v, seen, 0.0) for h in range(4)], 1)
        assert row_err(got, want).max() <= TOL
