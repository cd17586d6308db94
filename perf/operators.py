"""The serving operators that performance is measured on, with their plain forms.

A case is a dict of plain values with a "kind":

  window  attention of a sequence's newest tokens, each over a sliding window
          and the first tokens of the sequence (ss_hip_attention_window)
  shared  one decode step's attention of several sequences that continue the
          same prompt (ss_hip_attention_shared)
  sample  the next token of each row of logits with temperature, top-k, top-p
          and min-p, from given random numbers (ss_hip_sample_rows)

Queries are N(0, 1), cached K and V N(0, 1) (int8: uniform codes, scales 0.01 to
0.03), logits N(0, 2.5^2). The caches are longer than what they hold.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # one token of a long chat through an 8B shape: the newest 1024 tokens and four first ones
        dict(name="window-token-8b", kind="window", heads=32, kv_heads=8, hd=128, pos0=4096, tokens=1, window=1024,
             sinks=4, softcap=0.0, kv=0),
        # the smallest call: TinyLlama, int8 cache, a conversation shorter than its window
        dict(name="window-token-tinyllama-int8", kind="window", heads=32, kv_heads=4, hd=64, pos0=99, tokens=1, window=2048,
             sinks=4, softcap=0.0, kv=1),
        # one token of a 7B shape, all heads with K and V of their own, far into a long document
        dict(name="window-token-7b-long", kind="window", heads=32, kv_heads=32, hd=128, pos0=100000, tokens=1, window=8192,
             sinks=64, softcap=0.0, kv=0),
        # a full prompt chunk in the middle of a long document, 8B shape
        dict(name="window-chunk-512", kind="window", heads=32, kv_heads=8, hd=128, pos0=7000, tokens=512, window=4096,
             sinks=4, softcap=0.0, kv=0),
        # a chat turn of odd length through a Gemma shape: head_dim 256, capped scores, int8 cache
        dict(name="window-turn-gemma-77", kind="window", heads=16, kv_heads=8, hd=256, pos0=2500, tokens=77, window=1000,
             sinks=0, softcap=50.0, kv=1),
        # four short answers to a short question: TinyLlama
        dict(name="shared-4-tinyllama", kind="shared", heads=32, kv_heads=4, hd=64, seqs=4, prefix=200, own=32, softcap=0.0, kv=0),
        # sixteen answers to one long prompt: 8B shape
        dict(name="shared-16-8b", kind="shared", heads=32, kv_heads=8, hd=128, seqs=16, prefix=4096, own=500, softcap=0.0, kv=0),
        # a system prompt of odd length shared by 37 chats over the int8 cache: 7B shape
        dict(name="shared-37-7b-int8", kind="shared", heads=32, kv_heads=32, hd=128, seqs=37, prefix=1777, own=301, softcap=0.0, kv=1),
        # the largest: 64 chats about one long document, 8B shape
        dict(name="shared-64-8b-long", kind="shared", heads=32, kv_heads=8, hd=128, seqs=64, prefix=32000, own=1024, softcap=0.0, kv=0),
        # one token of one answer with the settings of a chat program
        dict(name="sample-1-32k", kind="sample", rows=1, vocab=32000, temperature=0.8, top_k=40, top_p=0.95, min_p=0.05),
        # a batch of answers, min-p alone
        dict(name="sample-16-min-p", kind="sample", rows=16, vocab=32000, temperature=1.1, top_k=0, top_p=1.0, min_p=0.02),
        # the largest batch over the 128k vocabulary, top-p alone
        dict(name="sample-64-128k-top-p", kind="sample", rows=64, vocab=128256, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "shared", "shared", "sample"])
    if kind == "sample":
        c = dict(kind=kind, rows=_log(rng, 1, 64), vocab=_log(rng, 500, 128256), temperature=round(rng.uniform(0.5, 1.5), 2),
                 top_k=rng.choice([0, 0, 1, 20, 40, 100, 1500]), top_p=rng.choice([0.5, 0.9, 0.95, 1.0]),
                 min_p=rng.choice([0.0, 0.02, 0.1]))
        return c
    kvh, group, hd = rng.choice([(4, 8, 64), (8, 4, 128), (8, 8, 128), (32, 1, 128), (12, 1, 64), (4, 2, 128), (8, 2, 256), (1, 8, 256)])
    c = dict(kind=kind, heads=kvh * group, kv_heads=kvh, hd=hd, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), kv=int(rng.random() < 0.4))
    if kind == "window":
        n = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, 500)])
        c.update(pos0=_log(rng, 1, 40000) - 1, tokens=n, window=_log(rng, 16, 8192 if n == 1 else 1900), sinks=rng.choice([0, 1, 4, 4, 37, 100]))
    else:
        c.update(seqs=_log(rng, 1, 48), prefix=rng.choice([0, 1, _log(rng, 16, 16000), _log(rng, 16, 16000)]), own=_log(rng, 1, 700))
    return c


def _own_lengths(case):
    """Positions of each sequence's own cache: ragged, the longest in full."""
    return [1 + (case["own"] - 1) * ((37 * b + 100) % 101) // 100 for b in range(case["seqs"])]


# ---- inputs ------------------------------------------------------------------
class State:
    pass


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _cache(g, kv, shape, scales):
    """K and V with their scales: fp16, or int8 codes and one scale per position."""
    if kv:
        k, v = (torch.randint(-127, 128, shape, generator=g, device=DEVICE, dtype=torch.int8) for _ in "kv")
        ks, vs = (0.01 + 0.02 * torch.rand(*scales, generator=g, device=DEVICE) for _ in "kv")
        return k, v, ks, vs
    return _normal(g, *shape).half(), _normal(g, *shape).half(), None, None


def _inputs(case, seed):
    c, s = case, State()
    s.case = c
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    if c["kind"] == "window":
        s.max_seq = c["pos0"] + c["tokens"] + 7
        s.q = _normal(g, c["tokens"], c["heads"] * c["hd"])
        s.cache = _cache(g, c["kv"], (c["kv_heads"], s.max_seq, c["hd"]), (s.max_seq,))
    elif c["kind"] == "shared":
        s.prefix_max, s.own_max = c["prefix"] + 5, c["own"] + 3
        s.q = _normal(g, c["seqs"], c["heads"] * c["hd"])
        s.prefix = _cache(g, c["kv"], (c["kv_heads"], s.prefix_max, c["hd"]), (s.prefix_max,))
        s.cache = _cache(g, c["kv"], (c["seqs"], c["kv_heads"], s.own_max, c["hd"]), (c["seqs"], s.own_max))
        s.lens = torch.tensor(_own_lengths(c), dtype=torch.int32, device=DEVICE)
    else:
        s.logits = 2.5 * _normal(g, c["rows"], c["vocab"])
        s.u = torch.rand(c["rows"], generator=g, device=DEVICE)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s.out = torch.empty(case["rows"], dtype=torch.int32, device=DEVICE) if case["kind"] == "sample" else torch.empty_like(s.q)
    s.ws = None
    torch.cuda.synchronize()   # the framework's calls run on a stream of their own
    return s


# ---- one pass ----------------------------------------------------------------
_ctx = None


def _library():
    """The framework's library and a context, made once."""
    global _ctx
    import phonemap_amd as pm
    if _ctx is None:
        _ctx = pm.lib().ss_hip_init(0)
        if not _ctx:
            raise RuntimeError(pm.lib().ss_hip_last_error().decode())
    return pm, pm.lib(), _ctx


def _workspace(c, L, x):
    """What a program allocates once for its calls of this shape."""
    if c["kind"] == "window":
        n = L.ss_hip_attention_window_workspace(x, c["heads"], c["kv_heads"], c["hd"], c["tokens"], c["window"], c["sinks"])
    elif c["kind"] == "shared":
        n = L.ss_hip_attention_shared_workspace(x, c["heads"], c["kv_heads"], c["hd"], c["seqs"], c["prefix"], c["own"] + 3)
    else:
        n = L.ss_hip_sample_rows_workspace(x, c["rows"], c["vocab"])
    return torch.empty(max(n, 1), dtype=torch.uint8, device=DEVICE)


def _p(t):
    return t.data_ptr() if t is not None else None


def _run_own(s):
    c, (pm, L, x) = s.case, _library()
    if s.ws is None:
        s.ws = _workspace(c, L, x)
    if c["kind"] == "window":
        pm.check(L.ss_hip_attention_window(x, _p(s.out), _p(s.q), *map(_p, s.cache), c["heads"], c["kv_heads"], c["hd"], s.max_seq,
                                           c["pos0"], c["tokens"], c["window"], c["sinks"], c["softcap"], c["kv"], _p(s.ws),
                                           s.ws.numel(), None))
    elif c["kind"] == "shared":
        pm.check(L.ss_hip_attention_shared(x, _p(s.out), _p(s.q), *map(_p, s.prefix), s.prefix_max, c["prefix"], *map(_p, s.cache),
                                           s.own_max, _p(s.lens), c["seqs"], c["heads"], c["kv_heads"], c["hd"], c["softcap"],
                                           c["kv"], _p(s.ws), s.ws.numel(), None))
    else:
        pm.check(L.ss_hip_sample_rows(x, _p(s.out), _p(s.logits), c["vocab"], c["rows"], c["vocab"], c["temperature"], c["top_k"],
                                      c["top_p"], c["min_p"], _p(s.u), _p(s.ws), s.ws.numel(), None))
    return s.out


def _values(x, scale):
    """Cached K or V [..., positions, hd] in 32 bits."""
    return x.float() if scale is None else x.float() * scale.unsqueeze(-1)


def _capped(s, cap):
    return cap * torch.tanh(s / cap) if cap > 0 else s


def _window_plain(s):
    c = s.case
    n, hd, h, kvh, pos0 = c["tokens"], c["hd"], c["heads"], c["kv_heads"], c["pos0"]
    g, end = h // kvh, pos0 + n
    low = max(pos0 - c["window"] + 1, min(c["sinks"], end))   # the first position after the sinks that a token sees
    at = torch.cat([torch.arange(min(c["sinks"], end), device=DEVICE), torch.arange(low, end, device=DEVICE)])
    ks, vs = (z[at] if z is not None else None for z in s.cache[2:])
    k, v = _values(s.cache[0][:, at], ks), _values(s.cache[1][:, at], vs)
    q = s.q.reshape(n, kvh, g, hd).permute(1, 0, 2, 3).reshape(kvh, n * g, hd) / math.sqrt(hd)
    x = _capped(torch.matmul(q, k.transpose(1, 2)), c["softcap"]).reshape(kvh, n, g, -1)
    last = pos0 + torch.arange(n, device=DEVICE).reshape(1, n, 1, 1)
    x = x.masked_fill((at > last) | ((at <= last - c["window"]) & (at >= c["sinks"])), -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    e = (e / e.sum(-1, keepdim=True)).reshape(kvh, n * g, -1)
    return torch.matmul(e, v).reshape(kvh, n, g, hd).permute(1, 0, 2, 3).reshape(n, h * hd)


def _shared_plain(s):
    c = s.case
    b, hd, h, kvh, p = c["seqs"], c["hd"], c["heads"], c["kv_heads"], c["prefix"]
    g = h // kvh
    kp, vp = (_values(z[:, :p], sc[:p] if sc is not None else None) for z, sc in zip(s.prefix[:2], s.prefix[2:]))
    ko, vo = (_values(z, sc.unsqueeze(1) if sc is not None else None) for z, sc in zip(s.cache[:2], s.cache[2:]))
    q = s.q.reshape(b, kvh, g, hd) / math.sqrt(hd)
    xp = torch.matmul(q.transpose(0, 1).reshape(kvh, b * g, hd), kp.transpose(1, 2)).reshape(kvh, b, g, p).transpose(0, 1)
    xo = torch.matmul(q, ko.transpose(2, 3))
    xo = _capped(xo, c["softcap"]).masked_fill(torch.arange(s.own_max, device=DEVICE) >= s.lens.reshape(b, 1, 1, 1), -math.inf)
    x = torch.cat([_capped(xp, c["softcap"]), xo], -1)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    ep = e[..., :p].transpose(0, 1).reshape(kvh, b * g, p)
    out = torch.matmul(ep, vp).reshape(kvh, b, g, hd).transpose(0, 1) + torch.matmul(e[..., p:], vo)
    return out.reshape(b, h * hd)


def _sample_plain(s):
    """In 64 bits, with the settings as the 32-bit numbers that the call takes: a
    draw falls between two sums. Equal logits are kept or dropped together."""
    c = {k: float(np.float32(v)) if k in ("temperature", "top_p", "min_p") else v for k, v in s.case.items()}
    x = s.logits.double() / c["temperature"]
    e = torch.exp(x - x.amax(-1, keepdim=True))
    keep = torch.ones_like(e, dtype=torch.bool)
    if 0 < c["top_k"] < c["vocab"] or 0 < c["top_p"] < 1:
        down = torch.sort(e, -1, descending=True).values
        if 0 < c["top_k"] < c["vocab"]:
            keep &= e >= down[:, c["top_k"] - 1:c["top_k"]]
        if 0 < c["top_p"] < 1:   # down to the entry at which the running sum reaches top_p of the whole
            reached = (torch.cumsum(down, -1) < c["top_p"] * e.sum(-1, keepdim=True)).sum(-1, keepdim=True)
            keep &= e >= torch.gather(down, -1, reached.clamp(max=c["vocab"] - 1))
    if c["min_p"] > 0:
        keep &= e >= c["min_p"]
    total = torch.cumsum(e * keep, -1)
    return (total <= s.u.double().unsqueeze(-1) * total[:, -1:]).sum(-1).to(torch.int32)


def run(state):
    if own:
        return _run_own(state)
    return {"window": _window_plain, "shared": _shared_plain, "sample": _sample_plain}[state.case["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------
def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return dict(bytes=4 * n + 8 * c["rows"], flops=4 * n)
    kd, qd = c["kv_heads"] * c["hd"], c["heads"] * c["hd"]
    row = 2 * kd + 8 if c["kv"] else 4 * kd   # K and V of a position, and their scales
    if c["kind"] == "window":
        n, end = c["tokens"], c["pos0"] + c["tokens"]
        sinks = min(c["sinks"], end)
        read = sinks + max(0, end - max(c["pos0"] - c["window"] + 1, sinks))
        seen = sum(min(p + 1, c["sinks"]) + max(0, p + 1 - max(p - c["window"] + 1, min(c["sinks"], p + 1)))
                   for p in range(c["pos0"], end))
        return dict(bytes=read * row + 8 * n * qd, flops=4 * seen * qd)
    held = sum(_own_lengths(c))
    return dict(bytes=(c["prefix"] + held) * row + 8 * c["seqs"] * qd + 4 * c["seqs"],
                flops=4 * (c["seqs"] * c["prefix"] + held) * qd)


# ---- the same in 64 bits -----------------------------------------------------
def _head64(q, k, v, seen, cap):
    """q [rows][hd] over k, v [positions][hd], seen [rows][positions]."""
    s = (q @ k.T) / math.sqrt(q.shape[1])
    if cap > 0:
        s = cap * torch.tanh(s / cap)
    return torch.softmax(torch.where(seen, s, -math.inf), 1) @ v


def exact(case, seed):
    c = case
    if c["kind"] == "sample":
        return None   # whole numbers
    s = _inputs(case, seed)
    hd, kvh = c["hd"], c["kv_heads"]
    g = c["heads"] // kvh
    q = s.q.double().reshape(s.q.shape[0], kvh, g, hd)
    out = torch.zeros_like(q)

    def wide(z, scale):
        return z.double() * (1.0 if scale is None else scale.double().reshape(-1, 1))
    if c["kind"] == "window":
        end = c["pos0"] + c["tokens"]
        first = max(0, c["pos0"] + 1 - c["window"])
        sinks = min(c["sinks"], first)   # those before the window's first position
        at = torch.arange(first, end, device=DEVICE)
        at = torch.cat([torch.arange(sinks, device=DEVICE), at])
        me = torch.arange(c["pos0"], end, device=DEVICE).repeat_interleave(g).reshape(-1, 1)
        back = me - at
        seen = (back >= 0) & ((back < c["window"]) | (at < c["sinks"]))
        ks, vs = (z if z is None else z[at] for z in s.cache[2:])
        for j in range(kvh):
            o = _head64(q[:, j].reshape(-1, hd), wide(s.cache[0][j, at], ks), wide(s.cache[1][j, at], vs), seen, c["softcap"])
            out[:, j] = o.reshape(-1, g, hd)
        return out.reshape(s.q.shape)
    lens, p = _own_lengths(c), c["prefix"]
    none = [None] * c["seqs"]
    cut = lambda z: z if z is None else z[:p]  # noqa: E731
    for j in range(kvh):
        kp, vp = (wide(z[j, :p], cut(sc)) for z, sc in zip(s.prefix[:2], s.prefix[2:]))
        for b, n in enumerate(lens):
            ks, vs = (none if z is None else z for z in s.cache[2:])
            k = torch.cat([kp, wide(s.cache[0][b, j, :n], ks[b] if ks[b] is None else ks[b][:n])])
            v = torch.cat([vp, wide(s.cache[1][b, j, :n], vs[b] if vs[b] is None else vs[b][:n])])
            out[b, j] = _head64(q[b, j], k, v, torch.ones(g, p + n, dtype=torch.bool, device=DEVICE), c["softcap"])
    return out.reshape(s.q.shape)
