"""The serving calls refuse what they cannot compute, before any work on a
device: the checks read the context's fields alone, so a block of zeros stands
in for one. Every call here is refused."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import phonemap_amd as pm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CTX = (C.c_uint8 * 4096)()
P = 1 << 20   # an aligned address; nothing is read there

WINDOW = dict(ctx=C.addressof(CTX), out=P, q=P, k=P, v=P, ks=None, vs=None, heads=8, kv_heads=2, hd=64, max_seq=100, pos0=10,
              tokens=2, window=5, sinks=1, cap=0.0, kv=0, ws=P, ws_bytes=1 << 30, stream=None)
SHARED = dict(ctx=C.addressof(CTX), out=P, q=P, kp=P, vp=P, ksp=None, vsp=None, prefix_max=50, prefix=20, ko=P, vo=P, kso=None,
              vso=None, own_max=10, lens=P, seqs=2, heads=8, kv_heads=2, hd=64, cap=0.0, kv=0, ws=P, ws_bytes=1 << 30, stream=None)
SAMPLE = dict(ctx=C.addressof(CTX), out=P, logits=P, n=100, rows=2, ld=100, temperature=1.0, top_k=5, top_p=0.9, min_p=0.1, u=P,
              ws=P, ws_bytes=1 << 30, stream=None)


def _refused(name, good, **bad):
    L = pm.lib()
    assert getattr(L, name)(*{**good, **bad}.values()) == -5, bad
    assert L.ss_hip_last_error().decode().startswith(name[len("ss_hip_"):] + ":"), L.ss_hip_last_error()


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(out=None), dict(q=None), dict(k=None), dict(v=None), dict(heads=0), dict(heads=7), dict(heads=-8),
    dict(kv_heads=0), dict(kv_heads=-2), dict(heads=6), dict(hd=96), dict(hd=0), dict(heads=32), dict(pos0=-1), dict(tokens=0),
    dict(tokens=-1), dict(pos0=99), dict(pos0=2 ** 31 - 1), dict(tokens=2 ** 31 - 1), dict(window=0), dict(window=-1),
    dict(sinks=-1), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(kv=2), dict(kv=-1), dict(kv=1),
    dict(kv=1, ks=P), dict(kv=1, vs=P), dict(q=P + 4), dict(out=P + 8), dict(k=P + 2), dict(v=P + 1), dict(kv=1, ks=P + 2, vs=P),
], ids=str)
def test_window(bad):
    _refused("ss_hip_attention_window", WINDOW, **bad)


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(out=None), dict(q=None), dict(kp=None), dict(vp=None), dict(ko=None), dict(vo=None), dict(lens=None),
    dict(prefix=-1), dict(prefix=51), dict(own_max=0), dict(own_max=-1), dict(seqs=0), dict(seqs=-1), dict(heads=7), dict(hd=32),
    dict(heads=32), dict(cap=float("nan")), dict(kv=3), dict(kv=1), dict(kv=1, ksp=P, vsp=P), dict(kv=1, kso=P, vso=P),
    dict(kv=1, ksp=P, vsp=P, kso=P), dict(ko=P + 8), dict(vo=P + 2), dict(kp=P + 2), dict(lens=P + 2),
    dict(kv=1, ksp=P, vsp=P, kso=P, vso=P + 1),
], ids=str)
def test_shared(bad):
    _refused("ss_hip_attention_shared", SHARED, **bad)


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(out=None), dict(logits=None), dict(u=None), dict(n=0), dict(n=-1), dict(n=1 << 19, ld=1 << 19),
    dict(rows=0), dict(rows=-1), dict(rows=65536), dict(ld=99), dict(temperature=float("nan")), dict(temperature=float("inf")),
    dict(top_p=float("nan")), dict(min_p=float("nan")), dict(min_p=1.5), dict(logits=P + 2), dict(u=P + 1), dict(out=P + 2),
], ids=str)
def test_sample(bad):
    _refused("ss_hip_sample_rows", SAMPLE, **bad)


def _context(n_cu=256):
    """A context's fields as the checks read them: the number of compute units behind device and stream."""
    ctx = (C.c_uint8 * 4096)()
    np.frombuffer(ctx, np.int32)[4] = n_cu
    return ctx


@pytest.mark.parametrize("bad", [dict(ws=None), dict(ws=P + 8), dict(ws_bytes=-1)], ids=str)
def test_workspaces(bad):
    """None, one that is not aligned, one byte too few."""
    L, ctx = pm.lib(), _context()
    x = C.addressof(ctx)
    needs = [("ss_hip_attention_window", dict(WINDOW, max_seq=5000, pos0=4000, window=3000),
              L.ss_hip_attention_window_workspace(x, 8, 2, 64, 2, 3000, 1)),
             ("ss_hip_attention_shared", dict(SHARED, prefix_max=5000, prefix=4000), L.ss_hip_attention_shared_workspace(x, 8, 2, 64, 2, 4000, 10)),
             ("ss_hip_sample_rows", dict(SAMPLE, n=100000, ld=100000), L.ss_hip_sample_rows_workspace(x, 2, 100000))]
    for name, good, need in needs:
        assert need > 0, name
        _refused(name, good, **dict(dict(ctx=x, ws_bytes=need), **(dict(ws_bytes=need - 1) if "ws_bytes" in bad else bad)))
        assert str(need) in L.ss_hip_last_error().decode()


def test_workspaces_of_refused_shapes():
    L, ctx = pm.lib(), _context()
    x = C.addressof(ctx)
    assert L.ss_hip_attention_window_workspace(None, 8, 2, 64, 2, 3000, 1) == 0
    assert L.ss_hip_attention_window_workspace(x, 7, 2, 64, 2, 3000, 1) == 0
    assert L.ss_hip_attention_window_workspace(x, 8, 2, 64, 2 ** 31 - 1, 3000, 1) == 0
    assert L.ss_hip_attention_shared_workspace(x, 8, 2, 64, 2, -1, 10) == 0
    assert L.ss_hip_attention_shared_workspace(x, 8, 2, 64, 2 ** 31 - 1, 10, 10) == 0
    assert L.ss_hip_attention_shared_workspace(x, 8, 2, 64, 2 ** 19, 10, 10) > 0
    assert L.ss_hip_attention_shared_workspace(x, 8, 2, 64, 2 ** 19 + 1, 10, 10) == 0
    assert L.ss_hip_attention_shared_workspace(x, 8, 2, 64, 2, 2 ** 30 + 1, 10) == 0
    assert L.ss_hip_sample_rows_workspace(x, 65536, 100000) == 0
    assert L.ss_hip_sample_rows_workspace(x, 2, 1 << 19) == 0


def test_workspaces_cover_every_position():
    """The window's workspace goes by the window alone: no position asks for more.
    (With the window behind them 200 tokens of 32 heads on 4, head_dim 64, are the
    prompt rows' kernel's, in one piece; at position 600 they are two slots.)"""
    L, ctx = pm.lib(), _context()
    x = C.addressof(ctx)
    assert L.ss_hip_attention_window_bytes(32, 4, 64, 600, 200, 1900, 4, 256) > 0
    for heads, kv_heads in ((32, 4), (32, 8), (8, 1), (8, 8), (1, 1), (64, 8)):
        for hd in (64, 128, 256):
            for n in (1, 2, 3, 9, 17, 33, 40, 64, 100, 150, 200, 257, 400, 700, 1000, 3000):
                for w, sinks in ((1, 0), (100, 4), (1900, 4), (5000, 0), (300, 900), (20000, 0), (2 ** 30, 0), (2 ** 31 - 1, 2 ** 31 - 1)):
                    have = L.ss_hip_attention_window_workspace(x, heads, kv_heads, hd, n, w, sinks)
                    for pos0 in (0, 1, 31, 64, 150, 300, 600, 777, 1500, 2500, 6000, 19999, 50000, 10 ** 6):
                        end = pos0 + n + 3
                        need = L.ss_hip_attention_window_bytes(heads, kv_heads, hd, pos0, n, min(w, end), min(sinks, end), 256)
                        assert need <= have, (heads, kv_heads, hd, n, w, sinks, pos0)
    for n in (1, 3, 40):
        sizes = [L.ss_hip_attention_window_workspace(x, 32, 8, 128, n, w, 4) for w in (1, 10, 100, 1000, 5000, 20000, 2 ** 31 - 1)]
        assert sizes == sorted(sizes)


@pytest.mark.parametrize("bad", [dict(max_seq=2 ** 30 + 1), dict(max_seq=2 ** 31 - 1), dict(cap=1e-40)], ids=str)
def test_window_limits(bad):
    _refused("ss_hip_attention_window", WINDOW, **bad)


@pytest.mark.parametrize("bad", [dict(prefix_max=2 ** 30 + 1), dict(prefix_max=2 ** 31 - 1, prefix=2 ** 31 - 1),
                                 dict(own_max=2 ** 30 + 1), dict(own_max=2 ** 31 - 1), dict(cap=1e-40),
                                 dict(seqs=2 ** 19 + 1), dict(seqs=2 ** 31 - 1)], ids=str)
def test_shared_limits(bad):
    _refused("ss_hip_attention_shared", SHARED, **bad)


def test_header(tmp_path):
    """ss_hip.h brings the serving calls with it, either header can come first, and each declared call is exported."""
    text = open(os.path.join(ROOT, "include", "ss_hip_serving.h")).read()
    names = set(re.findall(r"^(?:size_t|int32_t) (ss_hip_\w+)\(", text, flags=re.M))
    assert names == {"ss_hip_%s%s" % (n, w) for n in ("attention_window", "attention_shared", "sample_rows") for w in ("", "_workspace")}
    assert all(hasattr(pm.lib(), n) for n in names)
    for first in ("ss_hip.h", "ss_hip_serving.h"):
        src = tmp_path / "a.c"
        src.write_text('#include "%s"\nvoid *calls[] = {%s};\n' % (first, ", ".join("(void *)" + n for n in sorted(names))))
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(src)], check=True)
