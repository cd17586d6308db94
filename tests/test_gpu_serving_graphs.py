"""The serving calls as a serving program makes them: captured in HIP graphs and
replayed with other inputs and lengths, on streams other than the context's, two
at a time with a workspace each, and beside the calls for one sequence."""
import numpy as np
import pytest

from tests.serving import TOL, Stream, cache, row_err, sample_exact, shared_call, shared_exact, window_call, window_exact

pytestmark = pytest.mark.gpu
H, KVH, HD = 32, 8, 128


def _up(hip, c):
    return [None if z is None else hip.upload(z) for z in c]


def _ptrs(bufs):
    return [b and b.ptr for b in bufs]


def _nan(buf):
    return buf.write(np.full(buf.nbytes // 4, np.nan, np.float32))


class Shared:
    """A call's buffers: prefix and own caches, queries, lengths, workspace, output."""

    def __init__(self, hip, kv, seqs, prefix, own_max, seed):
        rng = np.random.default_rng(seed)
        self.hip, self.kv, self.seqs, self.p, self.own_max = hip, kv, seqs, prefix, own_max
        self.host = cache(rng, kv, KVH, prefix, HD), cache(rng, kv, KVH, own_max, HD, (seqs,))
        self.pre, self.own = (_up(hip, c) for c in self.host)
        self.q, self.out, self.lens = (hip.buf(n) for n in (4 * seqs * H * HD, 4 * seqs * H * HD, 4 * seqs))
        self.ws = hip.buf(max(hip.L.ss_hip_attention_shared_workspace(hip.ctx, H, KVH, HD, seqs, prefix, own_max), 16))

    def call(self, stream):
        rc = self.hip.L.ss_hip_attention_shared(
            self.hip.ctx, self.out.ptr, self.q.ptr, *_ptrs(self.pre), self.p, self.p, *_ptrs(self.own), self.own_max, self.lens.ptr,
            self.seqs, H, KVH, HD, 0.0, self.kv, self.ws.ptr, self.ws.nbytes, stream)
        assert rc == 0, self.hip.err()

    def set(self, seed, q=None):
        """Other queries and lengths, nothing left in workspace and output; the exact output."""
        rng = np.random.default_rng(seed)
        lens = rng.integers(0, self.own_max + 1, self.seqs).astype(np.int32)
        if q is None:
            q = rng.standard_normal((self.seqs, H, HD)).astype(np.float32)
            self.q.write(q)
        self.lens.write(lens)
        self.clear()
        return shared_exact(q, self.host[0], self.p, self.host[1], lens, 0.0)

    def clear(self):
        _nan(self.ws), _nan(self.out)

    def got(self):
        return self.out.read(np.float32, self.seqs * H * HD).reshape(self.seqs, H, HD)

    def free(self):
        for b in [*self.pre, *self.own, self.q, self.out, self.lens, self.ws]:
            if b:
                b.free()


@pytest.fixture
def streams(hip):
    made = []

    def make():
        made.append(Stream(hip))
        return made[-1]
    yield make
    for s in made:
        s.free()


@pytest.mark.parametrize("kv,prefix", [(0, 700), (1, 700), (0, 3000), (1, 3000)])
def test_shared_replayed_with_other_lengths(hip, streams, kv, prefix):
    """One capture serves every step: queries and lengths are read when it runs."""
    print("graph, shared, kv", kv, prefix, flush=True)
    c, st = Shared(hip, kv, 5, prefix, 90, 1), streams()
    run = st.capture(lambda: c.call(st.ptr))
    for step in range(6):
        want = c.set(10 + step)
        run()
        st.wait()
        once = c.got()
        assert row_err(once, want).max() <= TOL
        c.clear()
        c.call(st.ptr)
        st.wait()
        assert np.array_equal(once, c.got())   # the same sums in the same order
    c.free()


def test_two_graphs_at_a_time(hip, streams):
    """Two captures with a workspace each, launched on two streams without waiting between."""
    print("graph, two at a time", flush=True)
    calls, sts = [Shared(hip, 0, 7, 2500, 300, s) for s in (3, 4)], [streams(), streams()]
    wants = [c.set(20 + i) for i, c in enumerate(calls)]
    runs = [st.capture(lambda c=c, st=st: [c.call(st.ptr) for _ in range(4)]) for c, st in zip(calls, sts)]
    for _ in range(5):
        for c in calls:
            c.clear()
        for run in runs:
            run()
        for st in sts:
            st.wait()
        for c, want in zip(calls, wants):
            assert row_err(c.got(), want).max() <= TOL
    for c in calls:
        c.free()


@pytest.mark.parametrize("tokens", [1, 5, 60])
def test_window_replayed(hip, streams, tokens):
    print("graph, window", tokens, flush=True)
    rng, st = np.random.default_rng(tokens), streams()
    pos0, window, sinks = 900, 600, 4
    c = cache(rng, 0, KVH, pos0 + tokens, HD)
    k, v = _up(hip, c[:2])
    q, out = hip.buf(4 * tokens * H * HD), hip.buf(4 * tokens * H * HD)
    n = hip.L.ss_hip_attention_window_workspace(hip.ctx, H, KVH, HD, tokens, window, sinks)
    ws = hip.buf(max(n, 16))

    def call():
        assert hip.L.ss_hip_attention_window(hip.ctx, out.ptr, q.ptr, k.ptr, v.ptr, None, None, H, KVH, HD, pos0 + tokens, pos0,
                                             tokens, window, sinks, 0.0, 0, ws.ptr, n, st.ptr) == 0, hip.err()
    run = st.capture(call)
    for step in range(4):
        x = rng.standard_normal((tokens, H, HD)).astype(np.float32)
        q.write(x)
        _nan(ws), _nan(out)
        run()
        st.wait()
        assert row_err(out.read(np.float32, x.size).reshape(x.shape), window_exact(x, c, pos0, window, sinks, 0.0)).max() <= TOL
    for b in (k, v, q, out, ws):
        b.free()


@pytest.mark.parametrize("V", [3000, 9000, 128256])
def test_sampling_replayed(hip, streams, V):
    """Rows in one launch, in two, and in two with several workgroups to a row: the
    same tokens from a replay as from a call, each time."""
    print("graph, sample", V, flush=True)
    rows, rng, st = 3, np.random.default_rng(V), streams()
    x, u, out = hip.buf(4 * rows * V), hip.buf(4 * rows), hip.buf(4 * rows)
    n = hip.L.ss_hip_sample_rows_workspace(hip.ctx, rows, V)
    ws = hip.buf(max(n, 16))
    setting = (1.0, 200, 0.95, 0.001)

    def call():
        assert hip.L.ss_hip_sample_rows(hip.ctx, out.ptr, x.ptr, V, rows, V, *setting, u.ptr, ws.ptr, n, st.ptr) == 0, hip.err()
    run = st.capture(call)
    for step in range(6):
        xs, us = (2.5 * rng.standard_normal((rows, V))).astype(np.float32), rng.random(rows, np.float32)
        x.write(xs), u.write(us), out.write(np.full(rows, -7, np.int32))
        _nan(ws)
        run()
        st.wait()
        got = out.read(np.int32, rows)
        for r in range(rows):
            want, near = sample_exact(xs[r], *setting, us[r])
            assert got[r] == want or near <= 1e-9
        call()
        st.wait()
        assert np.array_equal(out.read(np.int32, rows), got)
    for b in (x, u, out, ws):
        b.free()


@pytest.mark.parametrize("kv", [0, 1])
def test_beside_the_calls_for_one_sequence(hip, kv):
    """A window past the sequence, and one sequence behind a prefix, are ss_hip_attention
    over the positions put together; prompt rows are ss_hip_attention_rows."""
    print("serving calls beside the plain ones, kv", kv, flush=True)
    rng = np.random.default_rng(kv)
    n, p = 333, 200
    c = cache(rng, kv, KVH, n, HD)
    q = rng.standard_normal((1, H, HD)).astype(np.float32)
    bufs = _up(hip, [q] + c)
    out = hip.buf(q.nbytes)
    assert hip.L.ss_hip_attention(hip.ctx, out.ptr, *_ptrs(bufs), H, KVH, HD, n, n, kv, None) == 0, hip.err()
    plain = out.read(np.float32, q.size).reshape(q.shape).astype(np.float64)
    assert row_err(window_call(hip, q, c, n - 1, n, 0, 0.0), plain).max() <= 2 * TOL

    def part(z, a, b):   # scales [positions], values [heads][positions][hd]
        return z if z is None else np.ascontiguousarray(z[a:b] if z.ndim == 1 else z[:, a:b])
    own = [z if z is None else part(z, p, n)[None] for z in c]
    assert row_err(shared_call(hip, q, [part(z, 0, p) for z in c], p, own, [n - p], 0.0), plain).max() <= 2 * TOL
    if not kv:
        t = 40
        qs = rng.standard_normal((t, H, HD)).astype(np.float32)
        a, o = hip.upload(qs), hip.buf(qs.nbytes)
        assert hip.L.ss_hip_attention_rows(hip.ctx, o.ptr, a.ptr, bufs[1].ptr, bufs[2].ptr, H, KVH, HD, n, n - t, t, None) == 0
        rows = o.read(np.float32, qs.size).reshape(qs.shape).astype(np.float64)
        assert row_err(window_call(hip, qs, c, n - t, n, 0, 0.0), rows).max() <= 2 * TOL


def test_on_another_stream(hip, streams):
    """A stream of the caller's: the call follows that stream's work, here what
    writes its queries, with no wait between."""
    print("serving calls on a stream", flush=True)
    c, st, rng = Shared(hip, 0, 4, 300, 40, 9), streams(), np.random.default_rng(8)
    n = c.seqs * H * HD
    for step in range(3):
        g, u = hip.upload(3 * rng.standard_normal(n).astype(np.float32)), hip.upload(rng.standard_normal(n).astype(np.float32))
        _nan(c.q)
        c.set(50 + step, q=np.zeros((c.seqs, H, HD), np.float32))
        for _ in range(20):
            assert hip.L.ss_hip_swiglu(hip.ctx, c.q.ptr, g.ptr, u.ptr, n, st.ptr) == 0, hip.err()
        c.call(st.ptr)
        st.wait()
        got = c.got()
        q = c.q.read(np.float32, n).reshape(c.seqs, H, HD)
        assert row_err(got, shared_exact(q, c.host[0], c.p, c.host[1], c.lens.read(np.int32, c.seqs), 0.0)).max() <= TOL
        g.free(), u.free()
    c.free()


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("heads,kv_heads,hd,n,pos0,window", [
    (32, 4, 64, 200, 600, 1900),   # the few rows' kernel, in slots, where the whole window is the prompt rows'
    (32, 4, 64, 200, 1000, 1900), (16, 2, 128, 120, 500, 9000), (8, 8, 64, 150, 2000, 2 ** 31 - 1)])
def test_workspace_at_every_start(hip, heads, kv_heads, hd, n, pos0, window, kv):
    print("window", heads, kv_heads, hd, n, pos0, window, kv, flush=True)
    rng = np.random.default_rng(pos0)
    c = cache(rng, kv, kv_heads, pos0 + n + 1, hd)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    assert row_err(window_call(hip, q, c, pos0, window, 4, 0.0), window_exact(q, c, pos0, window, 4, 0.0)).max() <= TOL
