"""The 4-bit cache's kernels against numpy in 64 bits (tests/int4_ref.py), on an
MI355X: writes and reads bit for bit, attention within its derived bound."""

from __future__ import annotations

import numpy as np
import pytest

from tests import int4_ref as ref

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def i4():
    from latentserve_amd.kernels.hip import int4_cache
    return int4_cache


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def pools_of(arrays):
    return i4().Int4Pools(*(dev(a) for a in arrays))


def host(pools):
    return [p.cpu().numpy() for p in pools]


def rows(shape, seed):
    """fp16 values with outliers, constant groups, zeros, huge and tiny ranges."""
    r = np.random.default_rng(seed)
    x = r.standard_normal(shape).astype(np.float16)
    flat = x.reshape(-1, 4, 32)
    kinds = r.integers(0, 10, flat.shape[:2])
    flat[kinds == 1] *= np.float16(100)
    flat[kinds == 2] = np.float16(0)
    flat[kinds == 3] = np.float16(-3.5)
    flat[kinds == 4] *= np.float16(1e-4)
    flat[kinds == 5] *= np.float16(2.0 ** -18)               # subnormal
    big = np.where(r.random(flat.shape) < 0.5, np.float16(65504), np.float16(-65504))
    flat[kinds == 6] = big[kinds == 6]
    ties = r.integers(0, 31, flat.shape).astype(np.float16) / np.float16(2)    # halves: ties
    ties[..., 0], ties[..., 1] = 0, 15
    flat[kinds == 7] = ties[kinds == 7]
    mixed = flat * np.float16(1e-5)                          # one far entry among tiny ones
    mixed[..., 5] = 1000
    flat[kinds == 8] = mixed[kinds == 8]
    return x


@pytest.mark.parametrize("b,h,n", [(1, 1, 1), (3, 2, 1), (16, 2, 1), (2, 3, 5), (1, 8, 37), (2, 2, 130)])
def test_write_is_bit_exact_and_leaves_the_rest(b, h, n):
    nb = b * (n // 16 + 2) + 3
    before = ref.random_pools(nb, h, 1)
    pools = pools_of(before)
    k, v = rows((b, h, n, 128), 2), rows((b, h, n, 128), 3)
    slots = np.random.default_rng(4).permutation(nb * 16)[:b * n]
    print(f"write b={b} h={h} n={n}", flush=True)
    i4().write(dev(k), dev(v), dev(slots), pools)
    after = host(pools)
    want = [a.copy() for a in before]
    for z, x in ((0, k), (1, v)):
        codes, s, m = ref.quantize(x)
        raw, aff = want[2 * z].reshape(nb, h, -1), want[2 * z + 1].reshape(nb, h, -1)
        c = np.arange(128)
        for i, slot in enumerate(slots):
            blk, t = divmod(int(slot), 16)
            for hh in range(h):
                code = codes[i // n, hh, i % n]
                for cc in c:
                    byte, shift = ref.code_at(cc, z == 1, t)
                    raw[blk, hh, byte] = (raw[blk, hh, byte] & ~(15 << shift) & 255) | (code[cc] << shift)
                for g in range(4):
                    si, mi = ref.affine_at(32 * g, z == 1, t)
                    aff[blk, hh, si], aff[blk, hh, mi] = s[i // n, hh, i % n, g], m[i // n, hh, i % n, g]
    for got, exp, name in zip(after, want, i4().Int4Pools._fields):
        np.testing.assert_array_equal(got, exp, err_msg=name)


def test_a_group_with_a_nan_or_an_infinity_reads_back_as_nan():
    x = rows((1, 2, 6, 128), 9)
    bad = np.zeros((6, 4), bool)
    for t, (c, value) in enumerate([(0, np.nan), (63, np.inf), (100, -np.inf), (37, np.nan)]):
        x[0, 1, t, c] = value
        bad[t, c // 32] = True
    x[0, 1, 4, 64:96], x[0, 1, 5, 2:4] = np.nan, (np.inf, -np.inf)
    bad[4, 2] = bad[5, 0] = True
    pools = i4().empty_pools(1, 2, "cuda")
    i4().write(dev(x), dev(x), torch.arange(6, device="cuda"), pools)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([6], device="cuda").int()
    for got in i4().read(pools, table, lens, 6):
        nan = torch.isnan(got).cpu().numpy().reshape(2, 6, 4, 32)
        assert not nan[0].any()
        np.testing.assert_array_equal(nan[1].all(-1), bad)
        np.testing.assert_array_equal(nan[1].any(-1), bad)


def test_write_takes_strided_rows_and_skips_slots_outside():
    b, h, n, nb = 2, 2, 3, 4
    x = dev(rows((b, n, 2 * h, 128), 5))
    k, v = x[:, :, :h].transpose(1, 2), x[:, :, h:].transpose(1, 2)
    slots = torch.tensor([5, -1, 17, nb * 16, 40, -(1 << 40)], device="cuda")
    one, two = i4().empty_pools(nb, h, "cuda"), i4().empty_pools(nb, h, "cuda")
    i4().write(k, v, slots, one)
    keep = torch.tensor([0, 2, 4], device="cuda")
    flat = lambda t: t.transpose(1, 2).reshape(b * n, h, 1, 128)[keep].contiguous()  # noqa: E731
    i4().write(flat(k), flat(v), slots[keep].contiguous(), two)
    for p, q in zip(one, two):
        assert torch.equal(p, q)
    assert any(p.any() for p in one)


@pytest.mark.parametrize("h,lens,length", [(1, [1], 1), (2, [0, 15, 16, 17], 20), (3, [40, 3], 48),
                                           (8, [33], 100), (2, [130, 7, 64], None)])
def test_read_is_bit_exact(h, lens, length):
    width = max(1, -(-max(lens) // 16))
    b, nb = len(lens), len(lens) * width + 3
    arrays = ref.random_pools(nb, h, 7)
    arrays[1][0, 0, 0] = np.float16(65504)               # an entry past fp16's range: inf
    tables = np.random.default_rng(8).permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    k, v = i4().read(pools_of(arrays), dev(tables), dev(np.array(lens, np.int32)), length)
    length = width * 16 if length is None else length
    assert k.shape == v.shape == (b, h, length, 128)
    for got, z in ((k, 0), (v, 1)):
        all_ = ref.pool_values(arrays[2 * z], arrays[2 * z + 1], z == 1)
        want = np.zeros((b, h, length, 128), np.float16)
        for i, n in enumerate(lens):
            pos = np.arange(min(n, length))
            want[i, :, pos] = all_[tables[i, pos // 16], :, pos % 16]
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_read_of_blocks_outside_the_pool_and_past_the_table_is_zero():
    arrays = ref.random_pools(3, 2, 9)
    tables = np.array([[1, -1, 3], [2, 1 << 30, 0]], np.int32)
    k, v = i4().read(pools_of(arrays), dev(tables), dev(np.array([60, 48], np.int32)), 64)
    kv = ref.pool_values(arrays[0], arrays[1], False)
    got = k.cpu().numpy()
    np.testing.assert_array_equal(got[0, :, :16], kv[1])
    np.testing.assert_array_equal(got[1, :, 32:48], kv[0])
    assert (got[:, :, 16:32] == 0).all() and (got[0, :, 32:] == 0).all() and (got[1, :, 48:] == 0).all()


def attend_case(lens, h=2, r=6, seed=0, width=None, scale=1.0):
    g = np.random.default_rng(seed)
    width = width or max(1, -(-max(lens) // 16))
    b, nb = len(lens), len(lens) * width + 5
    arrays = ref.random_pools(nb, h, seed + 1)
    tables = g.permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    q = (g.standard_normal((b, h, r, 128)) * scale).astype(np.float16)
    return q, arrays, tables, np.array(lens, np.int32)


def check(out, q, arrays, tables, lens, what, scale=None):
    kv, vv = (ref.pool_values(arrays[2 * z], arrays[2 * z + 1], z == 1) for z in (0, 1))
    want, tol = ref.attend(q, kv, vv, tables, lens, scale)
    got = out.float().cpu().numpy().astype(np.float64)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.abs(got - want)[bad].max(), tol[bad].min(), np.argwhere(bad)[:3])


LENS = [[1], [16], [17], [2048], [0], [0, 1, 0, 15, 16, 17, 0], [5000, 3, 700, 64],
        [31, 32, 33] * 30, [9000, 100]]


@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("h,r", [(2, 6), (1, 1), (3, 16), (8, 4)])
def test_decode_matches_64_bits(lens, h, r):
    print(f"decode lens={lens[:7]} h={h} r={r}", flush=True)
    q, arrays, tables, ln = attend_case(lens, h, r, seed=len(lens) + h)
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    check(out, q, arrays, tables, ln, (lens, h, r))


@pytest.mark.parametrize("h,r,lens", [(256, 1, [900]), (256, 1, [767]), (128, 2, [1537, 31]),
                                      (32, 2, [12000]), (32, 6, [7001, 1, 0, 5000, 300, 17]),
                                      (16, 16, [16000, 9, 8000]), (8, 4, [2000] * 13)])
def test_decode_of_runs_that_differ(h, r, lens):
    """A full launch with long runs: they take more and fewer pages in turn."""
    print(f"decode lens={lens[:7]} h={h} r={r}", flush=True)
    q, arrays, tables, ln = attend_case(lens, h, r, seed=len(lens) + h)
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    check(out, q, arrays, tables, ln, (lens, h, r))


@pytest.mark.parametrize("h", [1, 2, 3, 8, 32])
def test_decode_far_below_the_bound(h):
    """A launch sized for long sequences serves short ones, by some of its groups."""
    for lens in ([1], [128], [129, 0], [500, 2000, 7], [3, 1500]):
        q, arrays, tables, ln = attend_case(lens, h, 4, seed=h, width=400 if h < 8 else 140)
        out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
        check(out, q, arrays, tables, ln, (lens, h))


@pytest.mark.parametrize("bound", [1, 100, 4096, 100000])
def test_decode_takes_any_expected_length(bound):
    q, arrays, tables, ln = attend_case([3000, 40], seed=11)
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln), bound)
    check(out, q, arrays, tables, ln, bound)


def test_decode_of_many_sequences():
    """More sequences than a wave has lanes, and than there are groups."""
    lens = [(37 * i) % 61 for i in range(1100)]
    q, arrays, tables, ln = attend_case(lens, 1, 2, seed=12)
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    check(out, q, arrays, tables, ln, "1100")


def test_decode_of_more_heads_than_groups():
    q, arrays, tables, ln = attend_case([70, 5, 33], 700, 1, seed=13)
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    check(out, q, arrays, tables, ln, "700 heads")


def test_decode_ignores_what_lies_behind_a_sequence():
    """NaN and infinite steps in the tokens past the end, in tables past it, in blocks
    nobody holds; blocks outside the pool are skipped."""
    lens = [21, 1, 40, 64]
    q, arrays, tables, ln = attend_case(lens, seed=14, width=6)
    clean = [a.copy() for a in arrays]
    live = np.zeros((arrays[0].shape[0], 16), bool)
    for i, n in enumerate(lens):
        for p in range(n):
            live[tables[i, p // 16], p % 16] = True
    for z in (0, 1):
        aff = arrays[2 * z + 1].reshape(live.shape[0], 2, 128)
        for t in range(16):
            for g in range(4):
                si, mi = ref.affine_at(32 * g, z == 1, t)
                aff[~live[:, t], :, si] = np.nan
                aff[~live[:, t], :, mi] = np.inf
    tables[0, 1] = -1
    tables[2, 0] = arrays[0].shape[0]
    tables[1, 3:] = 1 << 30
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    assert torch.isfinite(out).all()
    check(out, q, clean, tables, ln, "behind")


def test_decode_of_no_valid_block_is_zero():
    q, arrays, tables, ln = attend_case([40, 20], seed=15)
    tables[0] = -5
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    assert (out[0] == 0).all()
    check(out, q, arrays, tables, ln, "none")


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0, 3.0])
def test_decode_scales(scale):
    q, arrays, tables, ln = attend_case([500, 77], seed=16)
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln), softmax_scale=scale)
    check(out, q, arrays, tables, ln, scale, scale)


def test_decode_takes_strided_operands():
    """q inside a fused projection's rows, out inside a wider buffer, the layers' pools in
    one allocation, a table and lengths cut from larger ones."""
    h, r = 2, 6
    q, arrays, tables, ln = attend_case([300, 45, 16], h, r, seed=17)
    b, nb = len(ln), arrays[0].shape[0]
    big_q = torch.randn(b, (h * r + 4) * 128, device="cuda").half()
    qv = big_q[:, 128:(h * r + 1) * 128].view(b, h, r, 128)
    qv.copy_(dev(q))
    pools = []
    for a in pools_of(arrays):
        wide = torch.empty((nb, 3) + a.shape[1:], dtype=a.dtype, device="cuda")
        wide[:, 1] = a
        pools.append(wide[:, 1])
    big_t = torch.full((b + 1, tables.shape[1] + 3), -7, dtype=torch.int32, device="cuda")
    big_t[1:, 2:-1] = dev(tables)
    big_o = torch.zeros(b, h, r, 256, device="cuda").half()
    big_o[..., 128:] = 7
    out = big_o[..., :128]
    got = i4().paged_decode_int4(qv, i4().Int4Pools(*pools), big_t[1:, 2:-1],
                                 torch.cat((dev(ln), dev(ln)))[b:], out=out)
    assert got is out
    check(out, q, arrays, tables, ln, "strided")
    assert (big_o[..., 128:] == 7).all()


def test_decode_past_32_bit_offsets():
    """Pages beyond 2 GiB into a pool: a page stride far larger than a page."""
    h, nb = 1, 70
    small = ref.random_pools(nb, h, 18)
    step = 1 << 26                                        # 64 MiB from page to page, 4.4 GiB
    k_codes = torch.empty(nb * step, dtype=torch.uint8, device="cuda").view(nb, step)
    k_codes = k_codes[:, :1024].view(nb, 1, 16, 64)
    k_codes.copy_(dev(small[0]))
    pools = pools_of(small)._replace(k_codes=k_codes)
    q = np.random.default_rng(19).standard_normal((1, h, 4, 128)).astype(np.float16)
    tables = np.arange(nb, dtype=np.int32)[::-1][None].copy()
    ln = np.array([nb * 16 - 3], np.int32)
    out = i4().paged_decode_int4(dev(q), pools, dev(tables), dev(ln))
    check(out, q, small, tables, ln, "far pages")
    k, _ = i4().read(pools, dev(tables), dev(ln), 16)
    np.testing.assert_array_equal(k[0].cpu().numpy(), ref.pool_values(small[0], small[1], False)[nb - 1])
    new = rows((1, h, 1, 128), 20)
    i4().write(dev(new), dev(new), torch.tensor([(nb - 1) * 16 + 2], device="cuda"), pools)
    codes, s, m = ref.quantize(new)
    k, _ = i4().read(pools, dev(tables), dev(ln), 16)
    np.testing.assert_array_equal(k[0, 0, 2].cpu().numpy(), ref.values(codes, s, m)[0, 0, 0])


def test_decode_on_two_streams_at_once():
    cases = [attend_case([4000, 900, 33], seed=30 + i) for i in range(2)]
    args = [(dev(q), pools_of(a), dev(t), dev(l)) for q, a, t, l in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(i4().paged_decode_int4(*args[i]))
    torch.cuda.synchronize()
    for i, (q, a, t, l) in enumerate(cases):
        for o in outs[i]:
            check(o, q, a, t, l, i)


def test_captured_steps_replay_beside_each_other_and_eager_calls():
    """Two graphs of a write and a decode each, replayed on two streams at once with eager
    calls between; lengths grow between replays."""
    graphs, state = [], []
    for i in range(2):
        q, a, t, l = attend_case([3000, 500, 7], seed=40 + i, width=200)
        new = rows((3, 2, 1, 128), 50 + i)
        st = dict(q=dev(q), pools=pools_of(a), t=dev(t), l=dev(l), k=dev(new),
                  slots=torch.zeros(3, dtype=torch.int64, device="cuda"), host=(q, a, t, l, new))
        i4().paged_decode_int4(st["q"], st["pools"], st["t"], st["l"])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            i4().write(st["k"], st["k"], st["slots"], st["pools"])
            st["out"] = i4().paged_decode_int4(st["q"], st["pools"], st["t"], st["l"])
        graphs.append(g)
        state.append(st)
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(4):
        for st in state:
            q, a, t, l, new = st["host"]
            l += 1
            p = l - 1
            flat = t[np.arange(3), p // 16].astype(np.int64) * 16 + p % 16
            st["l"].copy_(dev(l))
            st["slots"].copy_(dev(flat))
            for z in (0, 1):
                codes, s, m = ref.quantize(new)
                raw, aff = a[2 * z].reshape(a[0].shape[0], 2, -1), a[2 * z + 1].reshape(a[0].shape[0], 2, -1)
                for i, slot in enumerate(flat):
                    blk, tt = divmod(int(slot), 16)
                    for hh in range(2):
                        for cc in range(128):
                            byte, shift = ref.code_at(cc, z == 1, tt)
                            raw[blk, hh, byte] = (int(raw[blk, hh, byte]) & ~(15 << shift)) \
                                | (int(codes[i, hh, 0, cc]) << shift)
                        for g4 in range(4):
                            si, mi = ref.affine_at(32 * g4, z == 1, tt)
                            aff[blk, hh, si], aff[blk, hh, mi] = s[i, hh, 0, g4], m[i, hh, 0, g4]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = i4().paged_decode_int4(state[0]["q"], state[0]["pools"], state[0]["t"],
                                       state[0]["l"] - 1)
        torch.cuda.synchronize()
        for st in state:
            q, a, t, l, _ = st["host"]
            check(st["out"], q, a, t, l, rep)
        q, a, t, l, _ = state[0]["host"]
        check(eager, q, a, t, l - 1, "eager")


def test_decode_of_runs_longer_than_the_table_in_lds():
    """More heads than workgroups, so that one takes a whole sequence: runs of thousands of
    pages, in pieces.  The tables name a few blocks over and over."""
    h, pages = 520, [2100, 4097, 1, 2048]
    arrays = ref.random_pools(5, h, 60)
    g = np.random.default_rng(61)
    tables = g.integers(0, 5, (4, 4097)).astype(np.int32)
    ln = np.array([16 * n - 5 for n in pages], np.int32)
    q = g.standard_normal((4, h, 1, 128)).astype(np.float16)
    out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    for hh in (0, 257, 519):
        part = [np.ascontiguousarray(a[:, hh:hh + 1]) for a in arrays]
        check(out[:, hh:hh + 1], q[:, hh:hh + 1], part, tables, ln, hh)


def test_decode_of_lengths_past_the_table_and_below_zero():
    q, arrays, tables, ln = attend_case([64, 64, 64], seed=62)
    for lens in ([1000, 64, 65], [-3, 5, -(1 << 31)]):
        ln = np.array(lens, np.int32)
        out = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
        check(out, q, arrays, tables, ln, lens)


def test_decode_refuses_an_out_that_overlaps_q():
    q, arrays, tables, ln = attend_case([20, 3], seed=63)
    x = dev(q)
    args = (pools_of(arrays), dev(tables), dev(ln))
    with pytest.raises(ValueError):
        i4().paged_decode_int4(x, *args, out=x)
    both = torch.cat((x, x, x))
    with pytest.raises(ValueError):
        i4().paged_decode_int4(both[0:2], *args, out=both[1:3])


def test_a_row_with_a_nan_query_leaves_the_others():
    q, arrays, tables, ln = attend_case([700, 40], seed=64)
    bad = q.copy()
    bad[0, 1, 2, 5] = np.nan
    out = i4().paged_decode_int4(dev(bad), pools_of(arrays), dev(tables), dev(ln))
    assert torch.isnan(out[0, 1, 2]).all()
    clean = i4().paged_decode_int4(dev(q), pools_of(arrays), dev(tables), dev(ln))
    out[0, 1, 2] = clean[0, 1, 2]
    check(out, q, arrays, tables, ln, "nan")


def test_many_captures_have_their_own_counters():
    """More captured calls than one slab of counters holds; all replay rightly."""
    q, arrays, tables, ln = attend_case([2000, 300], seed=65)
    args = (dev(q), pools_of(arrays), dev(tables), dev(ln))
    i4().paged_decode_int4(*args)
    graphs = []
    for _ in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = [i4().paged_decode_int4(*args) for _ in range(150)]
        graphs.append((g, outs))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
        i4().paged_decode_int4(*args)
    torch.cuda.synchronize()
    for _, outs in graphs:
        for o in (outs[0], outs[77], outs[-1]):
            check(o, q, arrays, tables, ln, "captures")


def test_a_capture_without_counters_left_zeroes_its_own(monkeypatch):
    """Every slice of the slab taken: the graph clears its counters itself, each replay."""
    from latentserve_amd import _serving

    q, arrays, tables, ln = attend_case([3000, 300, 40], seed=66)
    args = (dev(q), pools_of(arrays), dev(tables), dev(ln))
    eager = i4().paged_decode_int4(*args)
    slab = _serving._slabs[0][0]
    monkeypatch.setitem(_serving._slabs, 0, [slab, _serving._SLAB_INTS])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [i4().paged_decode_int4(*args) for _ in range(3)]
    monkeypatch.undo()
    for _ in range(4):
        for o in outs:
            o.zero_()
        g.replay()
        i4().paged_decode_int4(*args)
        torch.cuda.synchronize()
        for o in outs:
            check(o, q, arrays, tables, ln, "replay")
    check(eager, q, arrays, tables, ln, "eager")
