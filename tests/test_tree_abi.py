"""The third C header, checked without a GPU: it and its binding agree, and bad
arguments are refused before any launch (there is no device here, and a launch would
report that instead)."""

from __future__ import annotations

import ctypes
import hashlib
import os
import re

import pytest
import torch

from latentserve_amd import _lib, _tree
from latentserve_amd.kernels.hip import cache_eviction as ce
from latentserve_amd.kernels.hip import tree_attention as ta

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "latentserve_amd_tree.h")
DECLARATIONS = (1, "ad258b6f9807be13")


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


@pytest.fixture(scope="module")
def lib():
    return _tree.lib()


def test_header_binding_and_library_agree(lib):
    names = sorted(set(re.findall(r"\b(ls_[a-z0-9_]+)\s*\(", _text())))
    assert names == _tree.exported_symbols()
    assert lib.ls_tree_abi_version() == _tree.ABI_VERSION
    for n in names:
        decl = re.search(r"\b%s\s*\(([^)]*)\)" % n, _text()).group(1)
        args = 0 if decl.strip() == "void" else decl.count(",") + 1
        assert args == len(_tree._SIGNATURES[n]), n


def test_a_changed_declaration_is_a_new_version():
    digest = hashlib.sha256(" ".join(_text().split()).encode()).hexdigest()[:16]
    assert (_tree.ABI_VERSION, digest) == DECLARATIONS


def _st(*v):
    return (ctypes.c_int64 * len(v))(*v)


BASE = dict(q=1 << 12, qs=_st(4096, 1024, 512, 128), k=1 << 20, v=1 << 21, ps=_st(4096, 256, 128), nb=10,
            t=64, ts=4, mp=4, l=64, b=2, h=2, n=8, r=6, d=128, page=16, m=0, scale=0.088, w=1 << 14, wb=1 << 40,
            o=1 << 13, os=_st(4096, 1024, 512, 128), s=1 << 22, ss=_st(200, 100), sl=64, sr=None, ns=4)


def _tree_call(lib, **over):
    a = dict(BASE, **over)
    return lib.ls_tree_attention(a["q"], a["qs"], a["k"], a["v"], a["ps"], a["nb"], a["t"], a["ts"], a["mp"], a["l"],
                                 None, None, a["o"], a["os"], None, a["w"], a["wb"], a["b"], a["h"], a["n"], a["r"],
                                 a["d"], a["page"], a["m"], a["scale"], None)


def _decode(lib, **over):
    a = dict(BASE, qs=_st(1536, 768, 128), os=_st(1536, 768, 128))
    a.update(over)
    return lib.ls_paged_decode_weights(a["q"], a["qs"], a["k"], a["v"], a["ps"], a["nb"], a["t"], a["ts"], a["mp"],
                                       a["l"], a["o"], a["os"], a["s"], a["ss"], a["sl"], a["sr"], a["ns"], a["w"],
                                       a["wb"], a["b"], a["h"], a["r"], a["d"], a["page"], a["m"], a["scale"], None)


def _add(lib, **over):
    a = dict(BASE, e=1 << 15, p=64, pl=3)
    a.update(over)
    return lib.ls_add_weights(a["q"], a["qs"], a["e"], a["k"], a["ps"], a["nb"], a["t"], a["ts"], a["mp"], a["l"],
                              a["s"], a["ss"], a["sl"], a["sr"], a["ns"], a["p"], None, a["b"], a["h"], a["n"],
                              a["pl"], a["r"], a["d"], a["page"], a["m"], a["scale"], None)


def _accept(lib, **over):
    a = dict(BASE, np=1, tok=64, par=64, ch=64, path=64, len=64, nx=64)
    a.update(over)
    one = lambda x: ctypes.cast((ctypes.c_void_p * 1)(x), ctypes.c_void_p)  # noqa: E731
    return lib.ls_accept_tokens(a["tok"], a["par"], a["ch"], None, a["path"], a["len"], a["nx"], one(a["k"]),
                                one(a["v"]), a["np"], a["ps"], a["nb"], a["t"], a["ts"], a["mp"], a["l"], a["b"],
                                a["h"], a["n"], a["d"], a["page"], None)


def _move(lib, **over):
    a = dict(BASE, keep=64, budget=8, layers=1)
    a.update(over)
    one = lambda x: ctypes.cast((ctypes.c_void_p * 1)(x), ctypes.c_void_p)  # noqa: E731
    return lib.ls_move_tokens(one(a["k"]), one(a["v"]), a["layers"], a["ps"], a["nb"], a["t"], a["ts"], a["mp"],
                              a["l"], a["keep"], a["b"], a["h"], a["budget"], a["d"], a["page"], None)


def _select(lib, **over):
    a = dict(BASE, ss=_st(400, 200, 100), keep=64, kept=64, layers=2, budget=8, sinks=2, recent=3)
    a.update(over)
    return lib.ls_select_tokens(a["s"], a["ss"], a["sl"], a["l"], a["keep"], a["kept"], a["layers"], a["b"], a["h"],
                                a["budget"], a["sinks"], a["recent"], None)


POOL = [(dict(ps=None), "null"), (dict(d=64), "head_dim"), (dict(page=32), "page"), (dict(nb=0), "num_blocks"),
        (dict(nb=1 << 31), "num_blocks"), (dict(ps=_st(4096, 252, 128)), "16 bytes"),
        (dict(ps=_st(4096, -256, 128)), "backwards"), (dict(ps=_st(1 << 40, 1 << 25, 128)), "2^24"),
        (dict(b=-1), "batch"), (dict(b=65536), "batch"), (dict(h=0), "kv_heads"), (dict(h=65536), "kv_heads")]
TABLES = [(dict(t=None), "null"), (dict(l=None), "null"), (dict(mp=0), "max_pages"),
          (dict(mp=(1 << 24) + 1), "max_pages"), (dict(ts=-1), "backwards")]
SUMS = [(dict(s=None), "null"), (dict(ss=None), "null"), (dict(s=2), "aligned"), (dict(sl=-1), "sum_len"),
        (dict(ns=-1), "num_sum_rows"), (dict(ss=_st(-1, 100)), "strides")]
SCALES = [(dict(scale=x), "softmax_scale") for x in (0.0, -1.0, float("nan"), float("inf"))]


@pytest.mark.parametrize("over,needle", POOL + TABLES + SCALES + [
    (dict(q=None), "null"), (dict(o=None), "null"), (dict(w=None), "null"), (dict(n=0), "nodes"),
    (dict(n=257), "nodes"), (dict(r=0), "n_rep"), (dict(r=17), "n_rep"), (dict(q=(1 << 12) + 2), "aligned"),
    (dict(os=_st(4096, 1024, 512, 129)), "aligned"), (dict(k=(1 << 20) + 8), "aligned"), (dict(wb=100), "workspace"),
    (dict(w=(1 << 14) + 4), "workspace"), (dict(b=65535, h=100), "too large"),
    (dict(b=4096, h=8, mp=1 << 24), "too large")])
def test_tree_attention_refuses(lib, over, needle):
    assert _tree_call(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("over,needle", POOL + TABLES + SCALES + SUMS + [
    (dict(q=None), "null"), (dict(r=17), "n_rep"), (dict(qs=_st(1536, 768, 129)), "aligned"),
    (dict(wb=100), "workspace"), (dict(b=65535, h=100), "too large")])
def test_decode_weights_refuses(lib, over, needle):
    assert _decode(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("over,needle", POOL + TABLES + SCALES + SUMS + [
    (dict(q=None), "null"), (dict(e=None), "null"), (dict(pl=9), "path_len"), (dict(pl=-1), "path_len"),
    (dict(p=None), "path_len"), (dict(n=257), "nodes"), (dict(k=(1 << 20) + 8), "aligned")])
def test_add_weights_refuses(lib, over, needle):
    assert _add(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("over,needle", POOL + TABLES + [
    (dict(tok=None), "null"), (dict(path=None), "null"), (dict(n=257), "nodes"), (dict(np=-1), "pools"),
    (dict(k=None), "null"), (dict(v=(1 << 21) + 2), "aligned")])
def test_accept_refuses(lib, over, needle):
    assert _accept(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("over,needle", POOL + TABLES + [
    (dict(keep=None), "null"), (dict(budget=0), "budget"), (dict(layers=-1), "pools"), (dict(k=None), "null")])
def test_move_refuses(lib, over, needle):
    assert _move(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("over,needle", [
    (dict(s=None), "null"), (dict(l=None), "null"), (dict(keep=None), "null"), (dict(kept=None), "null"),
    (dict(budget=0), "budget"), (dict(sinks=6), "budget"), (dict(sinks=-1), "budget"), (dict(recent=-1), "budget"),
    (dict(sl=-1), "sum_len"), (dict(ss=_st(400, -200, 100)), "backwards"), (dict(layers=1 << 22), "layers"),
    (dict(b=-1), "batch")])
def test_select_refuses(lib, over, needle):
    assert _select(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


def test_nothing_to_do_is_no_launch(lib):
    assert _tree_call(lib, b=0) == _decode(lib, b=0) == _add(lib, b=0) == _add(lib, pl=0) == 0
    assert _accept(lib, b=0) == _move(lib, b=0) == _move(lib, layers=0) == _select(lib, layers=0) == 0


def test_workspaces_hold_every_group(lib):
    """Sizes grow with the call and are 0 for calls that are refused."""
    size = lib.ls_tree_attention_workspace_bytes
    assert size(0, 2, 8, 6, 10, 0) == size(1, 2, 257, 6, 10, 0) == size(1, 2, 8, 17, 10, 0) == 0
    for b in (1, 3, 16, 300):
        for n in (1, 5, 16, 64, 256):
            assert 0 < size(b, 2, n, 6, 64, 100) <= size(b, 2, n, 6, 64, 0) < 1 << 30
    assert lib.ls_decode_weights_workspace_bytes(2, 2, 6, 64, 0) >= 2 * 2 * 6 * 1024 * 4


# ---- the Python layer, with a recorder in the library's place -----------------------


class _Recorder:
    def __init__(self):
        self.launched = []

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *a: 64
        return lambda *a: self.launched.append(name) or 0


@pytest.fixture
def recorder(monkeypatch):
    rec = _Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: rec)
    return rec


def _case(b=2, n=3, h=2, r=6, nb=9):
    half = torch.float16
    return dict(q=torch.zeros(b, n, h, r, 128, dtype=half), k=torch.zeros(nb, 16, h, 128, dtype=half),
                v=torch.zeros(nb, 16, h, 128, dtype=half), t=torch.zeros(b, 4, dtype=torch.int32),
                l=torch.zeros(b, dtype=torch.int32), m=torch.zeros(b, n, 1, dtype=torch.int64),
                c=torch.zeros(b, dtype=torch.int32), lse=torch.zeros(b, n, h, r), sums=torch.zeros(b, h, 64),
                tok=torch.zeros(b, n, dtype=torch.int64), par=torch.zeros(b, n, dtype=torch.int32),
                keep=torch.zeros(1, b, h, 8, dtype=torch.int32), s4=torch.zeros(1, b, h, 64))


def test_cpu_tensors_reach_no_launch(recorder):
    c = _case()
    pools = ([c["k"]], [c["v"]])
    calls = [lambda: ta.tree_masks(c["par"]),
             lambda: ta.tree_attention(c["q"], c["k"], c["v"], c["t"], c["l"], c["m"], c["c"], lse=c["lse"]),
             lambda: ta.accept_tokens(c["tok"], c["par"], c["tok"], *pools, c["t"], c["l"]),
             lambda: ce.paged_decode_weights(c["q"][:, 0], c["k"], c["v"], c["t"], c["l"], c["sums"]),
             lambda: ce.add_weights(c["q"], c["lse"], c["k"], c["t"], c["l"], c["sums"]),
             lambda: ce.select_tokens(c["s4"], c["l"], 8), lambda: ce.move_tokens(c["keep"], *pools, c["t"], c["l"]),
             lambda: ce.evict_tokens(c["s4"], *pools, c["t"], c["l"], 8)]
    for call in calls:
        with pytest.raises(ValueError, match="cuda"):
            call()
    assert recorder.launched == []


def test_python_refusals(recorder):
    c = _case()
    half = torch.float16
    q, k, v, t, l, m, lse, sums = (c[x] for x in ("q", "k", "v", "t", "l", "m", "lse", "sums"))

    def no(fn, *a, **kw):
        with pytest.raises(ValueError) as e:
            fn(*a, **kw)
        assert "cuda device" not in str(e.value)           # refused for its own reason

    no(ta.tree_masks, c["par"].long())
    no(ta.tree_masks, torch.zeros(1, 257, dtype=torch.int32))
    no(ta.tree_masks, torch.zeros(1, 0, dtype=torch.int32))
    tree = ta.tree_attention
    no(tree, q[..., :64], k, v, t, l)
    no(tree, q[:, :, :1], k, v, t, l)
    no(tree, q.float(), k, v, t, l, m)
    no(tree, torch.zeros(2, 257, 2, 1, 128, dtype=half), k, v, t, l)
    no(tree, torch.zeros(2, 2, 2, 17, 128, dtype=half), k, v, t, l)
    no(tree, q, k, v[:5], t, l)
    no(tree, q, k.float(), v, t, l)
    no(tree, q, k[:, :8], v[:, :8], t, l)
    no(tree, q, k, v, t.long(), l)
    no(tree, q, k, v, t[:1], l)
    no(tree, q, k, v, t, l[:1])
    no(tree, q, k, v, t, l, m[:, :2])
    no(tree, q, k, v, t, l, m.int())
    no(tree, q, k, v, t, l, m, c["c"].long())
    no(tree, q, k, v, t, l, m, lse=lse[..., :3])
    no(tree, q, k, v, t, l, m, lse=lse.half())
    decode = ce.paged_decode_weights
    q1 = q[:, 0]
    no(decode, q, k, v, t, l, sums)
    no(decode, q1, k, v, t, l, sums.half())
    no(decode, q1, k, v, t, l, sums[:, :1])
    no(decode, q1, k, v, t, l, sums[:1])
    no(decode, q1, k, v, t, l, sums[:1].expand(2, -1, -1))
    no(decode, q1, k, v, t, l, sums[:, :1].expand(-1, 2, -1))
    no(decode, q1, k, v, t, l, torch.zeros(2, 2, 128)[..., ::2])
    no(decode, q1, k, v, t, l, sums, c["c"][:1])
    no(decode, q1, k, v, t, l, sums, c["c"].long())
    no(ce.add_weights, q, lse[:, :2], k, t, l, sums)
    no(ce.add_weights, q, lse, k, t, l, sums, path=torch.zeros(2, 4, dtype=torch.int32))
    no(ce.add_weights, q, lse, k, t, l, sums, path=torch.zeros(2, 3, dtype=torch.int64))
    no(ce.add_weights, q, lse, k, t, l, sums, lengths=c["c"][:1])
    pools = ([k], [v])
    no(ta.accept_tokens, c["tok"].int(), c["par"], c["tok"], *pools, t, l)
    no(ta.accept_tokens, c["tok"], c["par"][:, :2], c["tok"], *pools, t, l)
    no(ta.accept_tokens, c["tok"], c["par"], c["tok"], [k], [], t, l)
    no(ta.accept_tokens, c["tok"], c["par"], c["tok"], [], [], t, l)
    no(ta.accept_tokens, c["tok"], c["par"], c["tok"], [k], [v[:5]], t, l)
    no(ta.accept_tokens, c["tok"], c["par"], c["tok"], [k[:1].expand(9, -1, -1, -1)], [v[:1].expand(9, -1, -1, -1)], t, l)
    no(ce.select_tokens, c["s4"].half(), l, 8)
    no(ce.select_tokens, c["s4"], l[:1], 8)
    no(ce.select_tokens, c["s4"], l, 0)
    no(ce.select_tokens, c["s4"], l, 8, 5, 4)
    no(ce.select_tokens, c["s4"], l, 8, -1)
    no(ce.move_tokens, c["keep"].long(), *pools, t, l)
    no(ce.move_tokens, c["keep"], [k, k], [v, v], t, l)
    no(ce.move_tokens, c["keep"][:, :, :1], *pools, t, l)
    no(ce.evict_tokens, c["s4"], [k, k], [v, v], t, l, 8)
    no(ce.evict_tokens, c["s4"][:, :, :1], *pools, t, l, 8)
    assert recorder.launched == []
