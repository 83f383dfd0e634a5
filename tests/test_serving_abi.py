"""The second C header, checked without a GPU: it and its binding agree, and bad
arguments are refused before any launch (there is no device here, and a launch
would report that instead)."""

from __future__ import annotations

import ctypes
import hashlib
import os
import re

import numpy as np
import pytest
import torch

from latentserve_amd import _lib, _serving
from latentserve_amd.kernels import logprobs as lp
from latentserve_amd.kernels.hip import int4_cache as i4
from latentserve_amd.kernels.hip import page_copy as pc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "latentserve_amd_serving.h")
DECLARATIONS = (1, "7a1d70adfe011700")


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


@pytest.fixture(scope="module")
def lib():
    return _serving.lib()


def test_header_binding_and_library_agree(lib):
    names = sorted(set(re.findall(r"\b(ls_[a-z0-9_]+)\s*\(", _text())))
    assert names == _serving.exported_symbols()
    assert lib.ls_serving_abi_version() == _serving.ABI_VERSION
    for n in names:
        decl = re.search(r"\b%s\s*\(([^)]*)\)" % n, _text()).group(1)
        args = 0 if decl.strip() == "void" else decl.count(",") + 1
        assert args == len(_serving._SIGNATURES[n]), n


def test_a_changed_declaration_is_a_new_version():
    digest = hashlib.sha256(" ".join(_text().split()).encode()).hexdigest()[:16]
    assert (_serving.ABI_VERSION, digest) == DECLARATIONS


def _st(*v):
    return (ctypes.c_int64 * len(v))(*v)


POOL = dict(kc=1 << 20, ka=1 << 21, vc=1 << 22, va=1 << 23, ps=_st(2048, 512, 2048, 512), nb=10)


def _write(lib, **over):
    a = dict(POOL, k=1 << 12, ks=_st(512, 256, 128), v=1 << 13, vs=_st(512, 256, 128), sl=64, b=2,
             h=2, n=3, d=128, page=16)
    a.update(over)
    return lib.ls_int4_write(a["k"], a["ks"], a["v"], a["vs"], a["sl"], a["kc"], a["ka"], a["vc"],
                             a["va"], a["ps"], a["nb"], a["b"], a["h"], a["n"], a["d"], a["page"],
                             None)


def _read(lib, **over):
    a = dict(POOL, t=64, ts=4, mp=4, l=64, ko=1 << 12, vo=1 << 13, b=2, h=2, d=128, page=16, n=7)
    a.update(over)
    return lib.ls_int4_read(a["kc"], a["ka"], a["vc"], a["va"], a["ps"], a["nb"], a["t"], a["ts"],
                            a["mp"], a["l"], a["ko"], a["vo"], a["b"], a["h"], a["d"], a["page"],
                            a["n"], None)


def _decode(lib, **over):
    a = dict(POOL, q=1 << 12, qs=_st(1536, 768, 128), t=64, ts=4, mp=4, l=64, o=1 << 13,
             os=_st(1536, 768, 128), w=1 << 14, wb=1 << 30, c=64, b=2, h=2, r=6, d=128, page=16,
             g=4, scale=0.088)
    a.update(over)
    return lib.ls_paged_decode_int4(a["q"], a["qs"], a["kc"], a["ka"], a["vc"], a["va"], a["ps"],
                                    a["nb"], a["t"], a["ts"], a["mp"], a["l"], a["o"], a["os"],
                                    a["w"], a["wb"], a["c"], a["b"], a["h"], a["r"], a["d"],
                                    a["page"], a["g"], a["scale"], None)


BAD_POOLS = [(dict(kc=None), "null"), (dict(va=None), "null"), (dict(ps=None), "null"),
             (dict(kc=(1 << 20) + 8), "16 bytes"), (dict(ps=_st(2048, 512, 2040, 512)), "16 bytes"),
             (dict(d=64), "head_dim"), (dict(page=32), "page"), (dict(h=0), "kv_heads"),
             (dict(nb=0), "num_blocks"), (dict(nb=1 << 31), "num_blocks")]
BAD_TABLES = [(dict(t=None), "null"), (dict(l=None), "null"), (dict(b=-1), "batch"),
              (dict(b=65536), "batch"), (dict(mp=0), "max_pages"), (dict(mp=(1 << 24) + 1), "max_pages"),
              (dict(b=65535, mp=1 << 16), "2^31")]


@pytest.mark.parametrize("over,needle", BAD_POOLS + [
    (dict(k=None), "null"), (dict(sl=None), "null"), (dict(k=(1 << 12) + 2), "aligned"),
    (dict(vs=_st(512, 256, 129)), "aligned"), (dict(n=-1), "tokens"), (dict(n=1 << 26), "too large")])
def test_write_refuses(lib, over, needle):
    assert _write(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("over,needle", BAD_POOLS + BAD_TABLES + [
    (dict(ko=None), "null"), (dict(vo=(1 << 13) + 2), "aligned"), (dict(n=-1), "length")])
def test_read_refuses(lib, over, needle):
    assert _read(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("over,needle", BAD_POOLS + BAD_TABLES + [
    (dict(q=None), "null"), (dict(w=None), "null"), (dict(c=None), "null"), (dict(o=None), "null"),
    (dict(r=0), "n_rep"), (dict(r=17), "n_rep"), (dict(g=0), "groups"), (dict(g=1 << 20), "groups"),
    (dict(q=(1 << 12) + 2), "aligned"), (dict(os=_st(1536, 768, 129)), "aligned"),
    (dict(wb=100), "workspace"), (dict(w=(1 << 14) + 4), "workspace")])
def test_decode_refuses(lib, over, needle):
    assert _decode(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_decode_refuses_a_scale_that_is_not_finite(lib, scale):
    assert _decode(lib, scale=scale) == 1
    assert "finite" in lib.ls_last_error().decode()


def test_sizes_past_a_launch_are_refused(lib):
    assert _read(lib, b=4, h=64, n=1 << 20) == 1 and "too large" in lib.ls_last_error().decode()
    assert _score(lib, rows=1 << 24, n=1, top=0) == 1 and "too large" in lib.ls_last_error().decode()


def test_decode_refuses_more_pages_than_its_places(lib):
    assert _decode(lib, b=65535, mp=32767) == 1        # below 2^31 as a table
    assert "+ 16" in lib.ls_last_error().decode()


def test_nothing_to_do_is_no_launch(lib):
    assert _write(lib, b=0) == _write(lib, n=0) == _read(lib, b=0) == _read(lib, n=0) == 0
    assert _decode(lib, b=0) == 0
    assert _copy(lib, [], []) == 0
    assert _score(lib, rows=0) == 0


def _copy(lib, src, dst, pages=10, stride=4096, size=4096, base=1 << 20):
    n = len(src)
    one = lambda v: ctypes.cast(_st(v), ctypes.c_void_p)  # noqa: E731
    return lib.ls_page_copy(one(base), one(stride), one(size), 1, pages,
                            (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst), n, None)


@pytest.mark.parametrize("src,dst,needle", [
    ([0, 10], [1, 2], "outside"), ([0, 1], [2, -1], "outside"), ([0, 1], [2, 2], "twice"),
    ([0, 1], [1, 2], "both"), ([3], [3], "both"),
    (list(range(100)) + [150], list(range(100, 200)) + [200], "both"),
    (list(range(100)), [200] + list(range(200, 299)), "twice")])
def test_page_copy_refuses(lib, src, dst, needle):
    assert _copy(lib, src, dst, pages=10 if max(src + dst) <= 10 else 300) == 1
    assert needle in lib.ls_last_error().decode()


def test_page_copy_refuses_overlapping_pages_and_null(lib):
    assert _copy(lib, [0], [1], stride=2048) == 1 and "apart" in lib.ls_last_error().decode()
    assert _copy(lib, [0], [1], base=0) == 1 and "null" in lib.ls_last_error().decode()


def _score(lib, **over):
    a = dict(x=1 << 12, xs=1000, e=2, t=64, ts=1, lp=1 << 13, en=1 << 14, tv=1 << 15, ti=1 << 16,
             w=1 << 17, wb=1 << 30, c=64, rows=2, n=100000, top=5)
    a.update(over)
    return lib.ls_token_logprobs(a["x"], a["xs"], a["e"], a["t"], a["ts"], a["lp"], a["en"],
                                 a["tv"], a["ti"], a["w"], a["wb"], a["c"], a["rows"], a["n"],
                                 a["top"], None)


@pytest.mark.parametrize("over,needle", [
    (dict(x=None), "null"), (dict(t=None), "null"), (dict(lp=None), "null"), (dict(tv=None), "null"),
    (dict(e=1), "elem_bytes"), (dict(n=0), "n must"), (dict(n=1 << 29), "n must"),
    (dict(rows=-1), "rows"), (dict(top=33), "top"), (dict(top=-1), "top"), (dict(n=4, top=5), "top"),
    (dict(x=(1 << 12) + 1), "aligned"), (dict(w=None), "workspace"), (dict(wb=8), "workspace"),
    (dict(c=None), "counters"), (dict(rows=(1 << 31) - 1), "too large")])
def test_logprobs_refuses(lib, over, needle):
    assert _score(lib, **over) == 1
    assert needle in lib.ls_last_error().decode()


# ---- the Python layer, with a recorder in the library's place -----------------------


class _Recorder:
    def __init__(self):
        self.launched = []

    def __getattr__(self, name):
        if name.endswith("_bytes") or name.endswith("_ints") or name.endswith("_groups"):
            return lambda *a: 64
        return lambda *a: self.launched.append(name) or 0


@pytest.fixture
def recorder(monkeypatch):
    rec = _Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: rec)
    return rec


def _case(b=2, h=2, n=3, nb=9):
    pools = i4.empty_pools(nb, h, "cpu")
    k = torch.zeros(b, h, n, 128, dtype=torch.float16)
    t, l = torch.zeros(b, 4, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    q = torch.zeros(b, h, 6, 128, dtype=torch.float16)
    return pools, k, torch.arange(b * n), t, l, q


def test_cpu_tensors_reach_no_launch(recorder):
    pools, k, slots, t, l, q = _case()
    calls = [lambda: i4.write(k, k, slots, pools), lambda: i4.read(pools, t, l),
             lambda: i4.paged_decode_int4(q, pools, t, l),
             lambda: pc.copy_pages([k], [0], [1]),
             lambda: lp.token_logprobs(torch.zeros(2, 50), torch.zeros(2, dtype=torch.int64))]
    for call in calls:
        with pytest.raises(ValueError, match="cuda"):
            call()
    assert recorder.launched == []


def test_python_refusals(recorder):
    pools, k, slots, t, l, q = _case()
    half = torch.float16

    def no(fn, *a, **kw):
        with pytest.raises(ValueError) as e:
            fn(*a, **kw)
        assert "cuda device" not in str(e.value)           # refused for its own reason

    no(i4.write, k[:, :1], k[:, :1], slots, pools)
    no(i4.write, k, k[:, :, :2], slots, pools)
    no(i4.write, k, k, slots[:-1], pools)
    no(i4.write, k, k, slots.int(), pools)
    no(i4.write, k, k, slots, pools[:3])
    no(i4.write, k, k, slots, pools._replace(v_affine=pools.v_affine.float()))
    no(i4.write, k, k, slots, pools._replace(k_codes=pools.k_codes[:5]))
    no(i4.write, k, k, slots, pools._replace(k_codes=pools.k_codes[:1].expand(9, -1, -1, -1)))
    wide = torch.zeros(9, 16, 2, 64, dtype=torch.uint8).transpose(1, 2)
    no(i4.write, k, k, slots, pools._replace(k_codes=wide))
    no(i4.read, pools, t.long(), l)
    no(i4.read, pools, t, l[:1])
    no(i4.read, pools, t, l, -1)
    no(i4.paged_decode_int4, q[..., :64], pools, t, l)
    no(i4.paged_decode_int4, torch.zeros(2, 2, 17, 128, dtype=half), pools, t, l)
    no(i4.paged_decode_int4, q, pools, t[:1], l)
    x = torch.zeros(2, 50)
    tok = torch.zeros(2, dtype=torch.int64)
    no(lp.token_logprobs, x.double(), tok)
    no(lp.token_logprobs, x, tok.int())
    no(lp.token_logprobs, x, tok[:1])
    no(lp.token_logprobs, x, tok, 33)
    no(lp.token_logprobs, x[:, :4], tok, 5)
    no(lp.token_logprobs, x.requires_grad_(), tok)
    a = torch.zeros(5, 4, 3)
    no(pc.copy_pages, [a, a[:4]], [0], [1])
    no(pc.copy_pages, [a], [0, 1], [2])
    no(pc.copy_pages, [a.transpose(1, 2)], [0], [1])
    assert recorder.launched == []


def test_reference_layout_is_a_bijection():
    from tests import int4_ref as ref
    for value in (False, True):
        codes = {ref.code_at(c, value, t) for c in range(128) for t in range(16)}
        assert len(codes) == 2048 and max(b for b, _ in codes) == 1023
        aff = {i for g in range(4) for t in range(16) for i in ref.affine_at(32 * g, value, t)}
        assert aff == set(range(128))


def test_reference_pool_values_are_the_entries():
    from tests import int4_ref as ref
    kc, ka, vc, va = ref.random_pools(2, 2, 1)
    for codes, aff, value in ((kc, ka, False), (vc, va, True)):
        all_ = ref.pool_values(codes, aff, value)
        for blk, h, t in ((0, 0, 0), (1, 1, 15), (1, 0, 6)):
            np.testing.assert_array_equal(all_[blk, h, t], ref.entry(codes, aff, value, blk, h, t))
