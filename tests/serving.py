"""Shared by the tests of the serving calls: caches with garbage where nothing
may be read, and the operators in 64 bits.

Tolerance of an attention row (2-norm of its difference over 2-norm of its exact
output, per query head), TOL = 4e-6: a score, up to 16 here, is a sum of up to
256 products in fp32, whose roundings, 2^-24 of partial sums below 16, add up
like a random walk to about 16 * 2^-24 * 2 = 2e-6, which the weight has as a
relative error; q and the weights held to 2^-22 and the exponential's 2^-22 add
0.7e-6, the sums over keys and their merges as much. One key's weight rounded to
11 bits gives 1e-5 to 2e-4 of a row, one key left out or taken twice 1e-4 and
more at these lengths.
"""
import ctypes as C

import numpy as np

TOL = 4e-6


def cache(rng, kv, heads, length, hd, lead=()):
    """K, V [*lead][heads][length][hd] and their scales [*lead][length] (None: fp16)."""
    shape = tuple(lead) + (heads, length, hd)
    if kv:
        k, v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in "kv")
        ks, vs = (rng.uniform(0.01, 0.03, tuple(lead) + (length,)).astype(np.float32) for _ in "kv")
        return [k, v, ks, vs]
    return [rng.standard_normal(shape).astype(np.float16) for _ in "kv"] + [None, None]


def spoil(c, at, lead=()):
    """NaN in the positions `at` (a mask) of a cache: of fp16 values, or of the scales."""
    for z in c[2:] if c[2] is not None else c[:2]:
        if c[2] is not None:
            z[lead + (at,)] = np.nan
        else:
            z[lead + (slice(None), at)] = np.nan


def values(c, head, at):
    k, v = (z[head, at].astype(np.float64) for z in c[:2])
    if c[2] is not None:
        k, v = (z * s[at].astype(np.float64)[:, None] for z, s in zip((k, v), c[2:]))
    return k, v


def attend(q, k, v, seen, cap):
    """q [rows][hd] over k, v [positions][hd] with seen [rows][positions]; 0 where nothing is seen."""
    s = q.astype(np.float64) @ k.T / np.sqrt(q.shape[1])
    if cap > 0:
        s = cap * np.tanh(s / cap)
    s = np.where(seen, s, -np.inf)
    m = s.max(1, keepdims=True, initial=-np.inf)
    e = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0.0)
    t = e.sum(1, keepdims=True)
    return np.where(t > 0, e @ v / np.where(t > 0, t, 1), 0.0)


def window_seen(pos0, n, window, sinks):
    i, j = np.arange(pos0, pos0 + n)[:, None], np.arange(pos0 + n)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def window_exact(q, c, pos0, window, sinks, cap):
    n, H, hd = q.shape
    G = H // c[0].shape[0]
    seen = window_seen(pos0, n, window, sinks)
    at = np.flatnonzero(seen.any(0))
    out = np.zeros((n, H, hd))
    for h in range(H):
        k, v = values(c, h // G, at)
        out[:, h] = attend(q[:, h], k, v, seen[:, at], cap)
    return out


def shared_exact(q, prefix, p, own, lens, cap):
    n, H, hd = q.shape
    G = H // own[0].shape[1]
    out = np.zeros((n, H, hd))
    for h in range(H):
        kp, vp = values(prefix, h // G, slice(0, p)) if p else (np.zeros((0, hd)),) * 2
        for b in range(n):
            one = [z if z is None else z[b] for z in own]
            ko, vo = values(one, h // G, slice(0, min(max(int(lens[b]), 0), own[0].shape[2])))
            k, v = np.concatenate([kp, ko]), np.concatenate([vp, vo])
            out[b, h] = attend(q[b, h][None], k, v, np.ones((1, len(k)), bool), cap)[0]
    return out


def row_err(got, want):
    """Per row and head; a row of zeros has to be zeros."""
    d, w = np.linalg.norm(got - want, axis=2), np.linalg.norm(want, axis=2)
    return np.where(w > 0, d / np.where(w > 0, w, 1), np.where(d > 0, np.inf, 0.0))


class Call:
    """Device copies of a call's arrays, its output with a guard behind it, and its
    workspace, of the size asked for and filled with NaN."""

    def __init__(self, hip):
        self.hip, self.bufs = hip, []

    def up(self, x):
        if x is None:
            return None
        self.bufs.append(self.hip.upload(x))
        return self.bufs[-1].ptr

    def ws(self, nbytes):
        if not nbytes:
            return None
        self.bufs.append(self.hip.buf(nbytes).write(np.full(nbytes // 4, np.nan, np.float32)))
        return self.bufs[-1].ptr

    def out(self, n, dtype=np.float32):
        self.n, self.dtype = n, dtype
        self.o = self.hip.buf(4 * (n + 64)).write(np.full(n + 64, 7, dtype))
        self.bufs.append(self.o)
        return self.o.ptr

    def result(self):
        got = self.o.read(self.dtype, self.n + 64)
        assert np.all(got[self.n:] == 7)   # nothing past the last row
        return got[:self.n]

    def free(self):
        for b in self.bufs:
            b.free()


def window_call(hip, q, c, pos0, window, sinks, cap, stream=None):
    n, H, hd = q.shape
    KVH, max_seq = c[0].shape[:2]
    x = Call(hip)
    nb = hip.L.ss_hip_attention_window_workspace(hip.ctx, H, KVH, hd, n, window, sinks)
    rc = hip.L.ss_hip_attention_window(hip.ctx, x.out(q.size), x.up(q), *map(x.up, c), H, KVH, hd, max_seq, pos0, n, window,
                                       sinks, cap, int(c[2] is not None), x.ws(nb), nb, stream)
    assert rc == 0, hip.err()
    got = x.result().reshape(q.shape)
    x.free()
    return got


def shared_call(hip, q, prefix, p, own, lens, cap, stream=None):
    n, H, hd = q.shape
    KVH, own_max = own[0].shape[1:3]
    x = Call(hip)
    nb = hip.L.ss_hip_attention_shared_workspace(hip.ctx, H, KVH, hd, n, p, own_max)
    pre = list(map(x.up, prefix)) if prefix else [None] * 4
    rc = hip.L.ss_hip_attention_shared(hip.ctx, x.out(q.size), x.up(q), *pre, prefix[0].shape[1] if prefix else 0, p,
                                       *map(x.up, own), own_max, x.up(np.asarray(lens, np.int32)), n, H, KVH, hd, cap,
                                       int(own[2] is not None), x.ws(nb), nb, stream)
    assert rc == 0, hip.err()
    got = x.result().reshape(q.shape)
    x.free()
    return got


# ---- sampling ----------------------------------------------------------------
def sample_exact(x, T, top_k, top_p, min_p, u):
    """(token, distance of the draw and of the cutoffs from a border) of one row in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    T, top_p, min_p, u = (float(np.float32(z)) for z in (T, top_p, min_p, u))
    m = x.max()
    if m == -np.inf:
        return -1, 1.0
    if T <= 0:
        return int(np.argmax(x)), 1.0
    w = np.exp(np.where(x == m, 0.0, x - m) / T)
    keep, near = np.ones(x.size, bool), 1.0
    down = np.sort(x)[::-1]
    if 0 < top_k < x.size:
        keep &= x >= down[top_k - 1]
    if 0 < top_p < 1:
        sums = np.cumsum(np.sort(w)[::-1])
        goal = top_p * sums[-1]
        keep &= x >= down[min(int((sums < goal).sum()), x.size - 1)]
        near = min(near, float(np.abs(sums / goal - 1).min()))
    if min_p > 0:
        keep &= w >= min_p
        near = min(near, float(np.abs(w / min_p - 1)[x < m].min(initial=1.0)))
    u = 0.0 if not u > 0 else min(u, np.nextafter(1.0, 0.0))
    c = np.cumsum(w * keep)
    near = min(near, float(np.abs(c[w * keep > 0] / c[-1] - u)[:-1].min(initial=1.0)))
    return int((c <= u * c[-1]).sum()), near


def sample_call(hip, x, T, top_k, top_p, min_p, u, ld=None, stream=None):
    n_rows, V = x.shape
    ld = ld or V
    wide = np.full((n_rows, ld), 1e9, np.float32)
    wide[:, :V] = x
    c = Call(hip)
    nb = hip.L.ss_hip_sample_rows_workspace(hip.ctx, n_rows, V)
    rc = hip.L.ss_hip_sample_rows(hip.ctx, c.out(n_rows, np.int32), c.up(wide), V, n_rows, ld, T, top_k, top_p, min_p,
                                  c.up(np.asarray(u, np.float32)), c.ws(nb), nb, stream)
    assert rc == 0, hip.err()
    got = c.result()
    c.free()
    return got


# ---- streams and graphs --------------------------------------------------------
class Stream:
    """A HIP stream, and captures of calls made on it; the runtime is the library's."""

    def __init__(self, hip):
        self.L, self.s = hip.L, C.c_void_p()
        self.made = []
        self.ok(self.L.hipStreamCreate(C.byref(self.s)))

    @staticmethod
    def ok(rc):
        assert rc == 0, rc

    @property
    def ptr(self):
        return self.s.value

    def wait(self):
        self.ok(self.L.hipStreamSynchronize(self.s))

    def capture(self, calls):
        """Records what calls() launches; returns what launches the graph."""
        graph, run = C.c_void_p(), C.c_void_p()
        self.ok(self.L.hipStreamBeginCapture(self.s, 1))   # hipStreamCaptureModeThreadLocal
        try:
            calls()
        finally:
            rc = self.L.hipStreamEndCapture(self.s, C.byref(graph))
        self.ok(rc)
        self.ok(self.L.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
        self.ok(self.L.hipGraphDestroy(graph))
        self.made.append(run)
        return lambda: self.ok(self.L.hipGraphLaunch(run, self.s))

    def free(self):
        self.wait()
        for run in self.made:
            self.ok(self.L.hipGraphExecDestroy(run))
        self.ok(self.L.hipStreamDestroy(self.s))
