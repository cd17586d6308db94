"""The serving calls together with the framework's others, as a program that
writes several answers to one prompt and one that goes on for long would call
them: a layer of attention between an embedding and a head, Q8_0 weights.

Bar: each step's logits within 1e-3 of 64 bits given the same tokens (the
framework's bar for its products), and each token the one that the logits of that
step give in 64 bits."""
import numpy as np
import pytest

from tests.serving import sample_exact
from tests.util import Q8_0, dequant_np, make_blocks, rel_err

pytestmark = pytest.mark.gpu
HIDDEN, H, KVH, HD, VOCAB, THETA = 512, 8, 2, 64, 2048, 10000.0
QD, KD = H * HD, KVH * HD


class Layer:
    def __init__(self, hip, seed):
        rng = np.random.default_rng(seed)
        self.hip, self.L = hip, hip.L
        shapes = dict(emb=(VOCAB, HIDDEN), wq=(QD, HIDDEN), wk=(KD, HIDDEN), wv=(KD, HIDDEN), wo=(HIDDEN, QD), head=(VOCAB, HIDDEN))
        blocks = {k: make_blocks(Q8_0, r, c, rng, 0.02 if k == "emb" else 0.001) for k, (r, c) in shapes.items()}
        self.dev = {k: hip.packed(blocks[k], Q8_0, *s) for k, s in shapes.items()}
        self.w = {k: dequant_np(blocks[k], *s, Q8_0).reshape(s) for k, s in shapes.items()}
        self.x, self.q, self.att = hip.buf(4 * 4 * HIDDEN), hip.buf(4 * 4 * QD), hip.buf(4 * 4 * QD)
        self.kv = hip.buf(4 * 2 * KD)

    def ok(self, rc):
        assert rc == 0, self.hip.err()

    # ---- on the device
    def token(self, row, tok, pos, kc, vc, max_seq, index):
        """Embedding, q, k, v, RoPE and append of one token, as row `row` of the batch."""
        L, c, d = self.L, self.hip.ctx, self.dev
        x, q, k, v = self.x.ptr + 4 * HIDDEN * row, self.q.ptr + 4 * QD * row, self.kv.ptr, self.kv.ptr + 4 * KD
        self.ok(L.ss_hip_embed_row(c, x, d["emb"].ptr, Q8_0, VOCAB, HIDDEN, tok, None))
        for y, m, rows in ((q, "wq", QD), (k, "wk", KD), (v, "wv", KD)):
            self.ok(L.ss_hip_matvec(c, y, d[m].ptr, x, rows, HIDDEN, Q8_0, None))
        self.ok(L.ss_hip_rope(c, q, k, H, KVH, HD, HD, pos, THETA, 0, None))
        self.ok(L.ss_hip_kv_append(c, kc, vc, None, None, k, v, KVH, HD, max_seq, index, 0, None))

    def logits(self, n, out):
        """x += Wo attention, then the head, for n rows."""
        L, c, d = self.L, self.hip.ctx, self.dev
        self.ok(L.ss_hip_gemm(c, self.x.ptr, d["wo"].ptr, self.att.ptr, None, 0.0, 1, HIDDEN, QD, n, Q8_0, None))
        self.ok(L.ss_hip_gemm(c, out.ptr, d["head"].ptr, self.x.ptr, None, 0.0, 0, VOCAB, HIDDEN, n, Q8_0, None))

    # ---- in 64 bits
    def rope(self, z, pos):
        f = THETA ** (-np.arange(0, HD, 2) / HD) * pos
        z = z.reshape(-1, HD // 2, 2)
        return np.stack([z[..., 0] * np.cos(f) - z[..., 1] * np.sin(f), z[..., 0] * np.sin(f) + z[..., 1] * np.cos(f)], -1).reshape(-1, HD)

    def kv64(self, tok, pos):
        x = self.w["emb"][tok]
        return (self.rope(self.w["wk"] @ x, pos).astype(np.float16).astype(np.float64),
                (self.w["wv"] @ x).reshape(KVH, HD).astype(np.float16).astype(np.float64))

    def logits64(self, tok, pos, ks, vs):
        x = self.w["emb"][tok]
        q, out = self.rope(self.w["wq"] @ x, pos), np.zeros((H, HD))
        for h in range(H):
            s = np.array([k[h // (H // KVH)] for k in ks]) @ q[h] / np.sqrt(HD)
            e = np.exp(s - s.max())
            out[h] = (e / e.sum()) @ np.array([v[h // (H // KVH)] for v in vs])
        return self.w["head"] @ (x + self.w["wo"] @ out.reshape(-1))


def _prompt_cache(m, tokens, max_seq):
    kc, vc = (m.hip.buf(2 * KVH * max_seq * HD) for _ in "kv")
    for i, t in enumerate(tokens):
        m.token(0, t, i, kc.ptr, vc.ptr, max_seq, i)
    return kc, vc, [m.kv64(t, i) for i, t in enumerate(tokens)]


def test_several_answers_to_one_prompt(hip):
    m, n, p, own_max, steps = Layer(hip, 1), 3, 40, 6, 5
    L, rng = hip.L, np.random.default_rng(2)
    prompt = rng.integers(0, VOCAB, p).tolist()
    kc, vc, past = _prompt_cache(m, prompt[:-1], p)
    block = KVH * own_max * HD
    ko, vo = (hip.buf(2 * n * block) for _ in "kv")
    lens, out, logits = hip.buf(4 * n), hip.buf(4 * n), hip.buf(4 * n * VOCAB)
    ws = hip.buf(max(L.ss_hip_attention_shared_workspace(hip.ctx, H, KVH, HD, n, p - 1, own_max),
                     L.ss_hip_sample_rows_workspace(hip.ctx, n, VOCAB), 16))
    toks, mine, spread = [prompt[-1]] * n, [[] for _ in range(n)], set()
    setting = (0.9, 50, 0.95, 0.01)
    for step in range(steps):
        print("answers, step", step, flush=True)
        for b in range(n):
            m.token(b, toks[b], p - 1 + step, ko.ptr + 2 * b * block, vo.ptr + 2 * b * block, own_max, step)
            mine[b].append(m.kv64(toks[b], p - 1 + step))
        lens.write(np.full(n, step + 1, np.int32))
        m.ok(L.ss_hip_attention_shared(hip.ctx, m.att.ptr, m.q.ptr, kc.ptr, vc.ptr, None, None, p, p - 1, ko.ptr, vo.ptr, None, None,
                                       own_max, lens.ptr, n, H, KVH, HD, 0.0, 0, ws.ptr, ws.nbytes, None))
        m.logits(n, logits)
        us = rng.random(n, np.float32)
        u = hip.upload(us)
        m.ok(L.ss_hip_sample_rows(hip.ctx, out.ptr, logits.ptr, VOCAB, n, VOCAB, *setting, u.ptr, ws.ptr, ws.nbytes, None))
        got, lg = out.read(np.int32, n).tolist(), logits.read(np.float32, n * VOCAB).reshape(n, VOCAB)
        for b in range(n):
            seen = past + mine[b]
            assert rel_err(lg[b], m.logits64(toks[b], p - 1 + step, [k for k, _ in seen], [v for _, v in seen])) <= 1e-3
            want, near = sample_exact(lg[b], setting[0], *setting[1:], us[b])
            assert got[b] == want or near <= 1e-9
        toks = got
        spread.add(tuple(got))
    assert any(len(set(s)) > 1 for s in spread)   # the answers differ


def test_a_long_conversation_in_a_window(hip):
    m, steps, window, sinks, max_seq = Layer(hip, 3), 60, 16, 3, 64
    L, rng = hip.L, np.random.default_rng(4)
    kc, vc = (hip.buf(2 * KVH * max_seq * HD) for _ in "kv")
    out, logits = hip.buf(4), hip.buf(4 * VOCAB)
    ws = hip.buf(max(L.ss_hip_attention_window_workspace(hip.ctx, H, KVH, HD, 1, window, sinks), 16))
    tok, past = 5, []
    for i in range(steps):
        print("conversation, step", i, flush=True)
        m.token(0, tok, i, kc.ptr, vc.ptr, max_seq, i)
        past.append(m.kv64(tok, i))
        m.ok(L.ss_hip_attention_window(hip.ctx, m.att.ptr, m.q.ptr, kc.ptr, vc.ptr, None, None, H, KVH, HD, max_seq, i, 1, window,
                                       sinks, 0.0, 0, ws.ptr, ws.nbytes, None))
        m.logits(1, logits)
        us = rng.random(1, np.float32)
        u = hip.upload(us)
        m.ok(L.ss_hip_sample_rows(hip.ctx, out.ptr, logits.ptr, VOCAB, 1, VOCAB, 1.0, 0, 0.9, 0.0, u.ptr, ws.ptr, ws.nbytes, None))
        got, lg = int(out.read(np.int32, 1)[0]), logits.read(np.float32, VOCAB)
        seen = [past[j] for j in range(i + 1) if i - j < window or j < sinks]
        assert rel_err(lg, m.logits64(tok, i, [k for k, _ in seen], [v for _, v in seen])) <= 1e-3
        want, near = sample_exact(lg, 1.0, 0, 0.9, 0.0, us[0])
        assert got == want or near <= 1e-9
        u.free()
        tok = got
