"""What requests share, found in their tables, and attention that reads it once, against float64
(paged_model.py: every request over all of its own tokens) on caches of every type."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_model as M
import paged_q8_model as Q
from abi_ops import down, stream, up
from cdml import native as N
from test_gpu_paged import rng
from test_gpu_paged_attn_q8 import compare, normal_rows, underflow

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16", "i8", "f8"]


def tables(r, groups, prefix, lens, P, blocks, batch=None):
    """Tables in which the members of a group share their first prefix[g] pages: (table, pages)."""
    batch = batch or groups[-1]
    used = -(-np.asarray(lens) // P)
    order, at = r.permutation(int(used.sum()) + 3), 0
    table = np.full((batch, blocks), -1, np.int32)
    lead = {b: g for g in range(len(groups) - 1) for b in range(groups[g], groups[g + 1])}
    for b in range(batch):
        n = 0
        g = lead.get(b)
        if g is not None and b > groups[g]:
            n = min(prefix[g], used[b], used[groups[g]])
            table[b, :n] = table[groups[g], :n]
        table[b, n:used[b]] = order[at:at + used[b] - n]
        at += used[b] - n
    return table, len(order)


def case_of(r, kind, groups, prefix, tails, news, P, H, HK, hd, pad=2, batch=None, outside=()):
    """(q, cache, table, kv, cu, groups, o): request b has tails[b] tokens behind its group's prefix[g] pages
    (`outside`: tokens of the requests of no group, behind the groups)."""
    lens = []
    for g in range(len(groups) - 1):
        lens += [prefix[g] * P + tails[b] for b in range(groups[g], groups[g + 1])]
    lens = list(outside[:groups[0]]) + lens + list(outside[groups[0]:])
    blocks = max(1, -(-max(lens) // P)) + 1
    table, pages = tables(r, groups, prefix, lens, P, blocks, len(lens))
    c = {"kind": kind, "P": P, "heads": HK, "hd": hd}
    for side in "kv":
        Q.put(c, side, normal_rows(r, pages, P, HK, hd))
    n = sum(news) + pad
    q, o = (r.standard_normal((n, H * hd)).astype(np.float32) for _ in range(2))
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return q, c, table, np.array(lens, np.int32), cu, np.array(groups, np.int32), o


def check(q, c, table, kv, cu, groups, o, H, scale=None, force=True, **more):
    if scale is None:
        scale = float(np.float32(1) / np.sqrt(np.float32(c["hd"])))
    want, tol = M.attention(q, c["kx"], c["vx"], table, kv, cu, c["P"], H, c["heads"], scale, o)
    got, found, bad = Q.call_attention_shared(q, c, table, kv, cu, groups, H, scale, o, force=force, **more)
    np.testing.assert_array_equal(found, Q.shared(table, kv, cu, groups, c["P"], len(c["k"])))
    assert bad == 0
    compare(got, want, tol + underflow(c, kv))
    return got, found


# ---- what is shared -----------------------------------------------------------------

@pytest.mark.parametrize("P", [1, 8, 64])
def test_shared_pages_are_found(P):
    r = rng(70, P)
    groups = np.array([2, 2, 7, 8, 30, 95], np.int32)  # none, five, one, 22, 65 members; 2 and 5 requests of no group
    B, blocks = 100, 37
    table = r.integers(0, 500, (B, blocks)).astype(np.int32)
    for first, behind in zip(groups[:-1], groups[1:]):
        table[first:behind] = table[first:first + 1]
    kv = np.full(B, blocks * P, np.int32)
    new = r.integers(0, 3, B).astype(np.int32)
    for turn in range(7):
        if turn == 1:
            table[5, 20], table[29, 36], table[60, 0] = 501, 502, 503
        elif turn == 2:
            kv[3], kv[12], kv[60] = 3 * P + 1, 0, -5
        elif turn == 3:
            table[:, 9] = r.choice([-1, 500, 2 ** 31 - 1], B)
        elif turn == 4:
            table[2:7, 1] = 500
        elif turn == 5:
            new[:] = 3 * P
        elif turn == 6:
            kv[:] = 2 ** 31 - 1
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        got = Q.call_shared(table, kv, cu, groups, P, 500)
        np.testing.assert_array_equal(got, Q.shared(table, kv, cu, groups, P, 500))


def test_shared_pages_of_long_and_wide_tables():
    r = rng(71)
    for B, blocks, groups, at in ((2, 9001, [0, 2], 8990), (4096, 50, [0, 4096], 41), (600, 300, [0, 599, 600], 299)):
        table = np.repeat(r.integers(0, 10 ** 6, (1, blocks)), B, 0).astype(np.int32)
        table[B // 2, at] ^= 1
        kv, cu = np.full(B, blocks * 4, np.int32), np.arange(B + 1, dtype=np.int32)
        groups = np.array(groups, np.int32)
        got = Q.call_shared(table, kv, cu, groups, 4, 10 ** 6)
        np.testing.assert_array_equal(got, Q.shared(table, kv, cu, groups, 4, 10 ** 6))
        assert got[0] == 4 * min(at, blocks - 1)


def test_no_groups_at_all():
    table, kv, cu = np.zeros((3, 2), np.int32), np.full(3, 8, np.int32), np.arange(4, dtype=np.int32)
    assert not Q.call_shared(table, kv, cu, np.array([1], np.int32), 4, 9).any()


# ---- attention ----------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HK,hd,P", [(4, 4, 16, 16), (8, 2, 64, 16), (5, 5, 40, 8), (7, 1, 128, 32), (2, 2, 96, 2),
                                       (3, 1, 7, 4), (2, 1, 200, 16), (34, 2, 24, 16)])
def test_single_tokens_behind_a_prefix(kind, H, HK, hd, P):
    # groups of four, one, none, six and twenty members; tails of one token and more, some requests idle
    r = rng(72, hd)
    groups = [0, 4, 5, 5, 11, 31]
    prefix = [max(1, n // P) for n in (40, 17, 9, 300, 130)]
    tails = r.integers(1, 60, 31)
    tails[[0, 6, 20]] = 1
    news = [1] * 31
    news[2] = news[12] = 0
    case = case_of(r, kind, groups, prefix, tails, news, P, H, HK, hd)
    check(*case, H)
    check(*case, H, force=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HK,hd,P", [(2, 2, 32, 16), (4, 1, 64, 8), (3, 1, 128, 64), (2, 1, 136, 16), (2, 2, 50, 1)])
def test_chunks_behind_a_prefix(kind, H, HK, hd, P):
    r = rng(73, hd)
    groups = [0, 3, 8, 10]
    prefix = [max(1, n // P) for n in (70, 200, 33)]
    tails = [40, 1, 130, 9, 60, 33, 2, 300, 64, 65]
    for most in (290, 70, 20, 5):
        news = [min(n, most) for n in (40, 1, 100, 9, 0, 2, 1, 290, 64, 1)]
        case = case_of(r, kind, groups, prefix, tails, news, P, H, HK, hd)
        check(*case, H)
        check(*case, H, force=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("members", [3, 20])
def test_long_prefixes_split_over_workgroups(kind, members):
    r = rng(74, members)
    groups = [0, members, 2 * members]
    tails = list(r.integers(1, 30, 2 * members))
    tails[1] = 700
    check(*case_of(r, kind, groups, [290, 150], tails, [1] * 2 * members, 16, 4, 2, 64), 4)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 192])
def test_requests_of_no_group_and_groups_that_part_early(kind, hd):
    r = rng(75)
    groups = [2, 6, 9]
    q, c, table, kv, cu, g, o = case_of(r, kind, groups, [6, 9], [0, 0] + [20, 7, 1, 33, 9, 9, 40], [1, 2, 1, 1, 1, 2, 1, 1, 1,
                                        1, 5], 16, 2, 1, hd, outside=[50, 3, 120, 64])
    table[4, 3] = table[10, 1]  # a member whose fourth page is another request's
    table[8, 0] = table[10, 2]  # one that shares nothing
    _, found = check(q, c, table, kv, cu, g, o, 2)
    assert list(found) == [0, 0] + [48] * 4 + [0] * 5


@pytest.mark.parametrize("kind", ["bf16", "f32", "i8"])
@pytest.mark.parametrize("bounds", [(6, 4, 300, 300), (2, 4, 112, 60), (6, 4, 16, 156), (6, 4, 160, 12), (1, 4, 112, 60),
                                    (6, 4, 0, 172), (6, 4, 172, 0), (4096, 4, 112, 60), (2, 1, 70000, 60),
                                    (2, 4, 70000, 0), (6, 4, 70000, 12), (3, 1, 70000, 600), (6, 2, 70000, 70000)])
def test_bounds_only_cost_time(kind, bounds):
    # of members, prefixes and tails, larger and smaller ones than there are (their sum holds every length)
    r = rng(76)
    groups = [0, 6, 12]
    most = bounds[1]
    news = [min(n, most) for n in [1, 1, 4, 4, 1, 2] * 2]
    case = case_of(r, kind, groups, [7, 5], [60, 1, 40, 4, 9, 20] * 2, news, 16, 4, 2, 64)
    blocks = max(case[2].shape[1], -(-max(bounds[2:]) // 16), 38)
    case = list(case)
    case[2] = np.concatenate([case[2], np.full((12, blocks - case[2].shape[1]), -1, np.int32)], 1)
    check(*case, 4, bounds=bounds, force=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("news", [1, 20])
def test_what_is_not_seen_does_not_matter(kind, news):
    r = rng(77)
    groups = [0, 5, 7]
    q, c, table, kv, cu, g, o = case_of(r, kind, groups, [3, 8], [30, 21, 22, 23, 90, 33, 20], [news] * 7, 16, 4, 2, 64)
    Q.unseen_filth(c, table, kv)
    check(q, c, table, kv, cu, g, o, 4)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("members", [2, 30])
def test_a_nan_reaches_the_rows_that_see_it(kind, where, members):
    r = rng(78)
    groups = [0, members, members + 2]
    q, c, table, kv, cu, g, o = case_of(r, kind, groups, [4, 4], [20] * (members + 2), [1] * (members + 2), 16, 2, 2, 64)
    x = normal_rows(r, len(c["k"]), 16, 2, 64)
    x[table[0, 2 if where == "shared" else 4], 5, 1, 9] = np.nan
    Q.put(c, "v", x)
    got, _ = check(q, c, table, kv, cu, g, o, 2)
    broken = np.isnan(got).any(1)
    assert broken.sum() == (members if where == "shared" else 1) and broken[0]


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("members", [3, 25])
def test_pages_that_are_none(kind, members):
    # a page of a tail counts as zeros; one of a prefix ends what is shared
    r = rng(79)
    groups = [0, members]
    q, c, table, kv, cu, g, o = case_of(r, kind, groups, [6], [40] * members, [1] * members, 16, 2, 1, 64)
    n = len(c["k"])
    table[1, 7], table[:, 4] = -3, n
    zeros = np.where((table >= 0) & (table < n), table, n)
    k, v = (np.concatenate([c[s], np.zeros((1, 16, 64))]) for s in ("kx", "vx"))
    want, tol = M.attention(q, k, v, zeros, kv, cu, 16, 2, 1, 0.125, o)
    got, found, bad = Q.call_attention_shared(q, c, table, kv, cu, g, 2, 0.125, o, force=True)
    assert bad == 1 and (found == 64).all()
    compare(got, want, tol + underflow(c, kv))


@pytest.mark.parametrize("kind", ["bf16", "f8"])
def test_strided_rows_and_scales(kind):
    r = rng(80)
    for ldq, ldo, scale in ((130, 128, 0.0), (132, 140, -0.3), (128, 129, 20.0)):
        check(*case_of(r, kind, [0, 4, 8], [3, 5], [20] * 8, [1, 3, 1, 1] * 2, 16, 2, 1, 64), 2, ldq=ldq, ldo=ldo,
              scale=scale)


@pytest.mark.parametrize("kind", KINDS)
def test_scores_and_values_far_apart(kind):
    # the maximum in the prefix, then in the tails; values of the one 2^20 times the other's
    r = rng(81)
    for turn in range(4):
        q, c, table, kv, cu, g, o = case_of(r, kind, [0, 4, 24], [4, 6], [30] * 24, [1] * 24, 16, 2, 2, 64)
        x = {s: normal_rows(r, len(c["k"]), 16, 2, 64) for s in "kv"}
        pages = table[[0, 4], :4] if turn % 2 else np.unique(table[:, 6:8][table[:, 6:8] >= 0])
        x["kv"[turn // 2]][pages] *= np.float32(30 if turn < 2 else 1000)
        for s in "kv":
            Q.put(c, s, x[s])
        check(q, c, table, kv, cu, g, o, 2)


@pytest.mark.parametrize("kind", ["f32", "i8"])
def test_a_step_in_a_graph(kind):
    """Both calls recorded once, replayed over lengths and tables that change: requests part from their group."""
    r = rng(82)
    groups, P, H, HK, hd, B = [0, 4, 7], 16, 4, 2, 64, 7
    q, c, table, kv, cu, g, o = case_of(r, kind, groups, [9, 5], [70, 60, 50, 40, 30, 20, 70], [1] * B, P, H, HK, hd, pad=0)
    table, (members, new, prefix, _) = Q.forced(c, table, kv, cu, g, H)
    L, st, n_pages = N.lib(), stream(), len(c["k"])
    size = (B, B, 2, members, new, prefix, 80, H, HK, hd)
    d = Q.upload(c)
    dt, dl, dc, dg, ds = M.ints(table), M.ints(kv), M.ints(cu), M.ints(g), M.ints(np.zeros(B))
    dq, do = up(q), up(o)
    w, n = M.ws("cdml_paged_attn_shared_workspace_size", *size)

    def call():
        N.check(L.cdml_paged_shared(dt.ptr, table.shape[1], dl.ptr, dc.ptr, dg.ptr, 2, B, n_pages, P, ds.ptr, st.handle))
        N.check(L.cdml_paged_attn_shared(dq.ptr, H * hd, *(Q.ptr(b) for b in d), N.CACHE[kind], n_pages, P, dt.ptr,
                                         table.shape[1], dl.ptr, dc.ptr, dg.ptr, ds.ptr, do.ptr, H * hd, *size, 0.125,
                                         None, w.ptr, n, st.handle))
    call()
    st.synchronize()
    graph = C.c_void_p()
    N.check(L.cdml_graph_capture_begin(st.handle))
    call()
    N.check(L.cdml_graph_capture_end(st.handle, C.byref(graph)))
    for turn in range(5):
        x = r.standard_normal(q.shape).astype(np.float32)
        m = kv - turn * 4
        if turn == 2:
            table[1, 4] = table[6, 7]
        elif turn == 4:
            table[5, 0] = table[6, 8]
        for buf, a in ((dq, x), (dl, m.astype(np.int32)), (dt, table), (do, o)):
            buf.upload(a, st)
        N.check(L.cdml_graph_launch(graph, st.handle))
        got = down(do, o.shape)
        np.testing.assert_array_equal(down(ds, (B,), np.int32), Q.shared(table, m, cu, g, P, n_pages))
        want, tol = M.attention(x, c["kx"], c["vx"], table, m, cu, P, H, HK, 0.125, o)
        compare(got, want, tol + underflow(c, m))
        do.upload(o, st)
        call()
        np.testing.assert_array_equal(down(do, o.shape), got)
    N.check(L.cdml_graph_destroy(graph))


@pytest.mark.parametrize("kind", ["bf16", "i8"])
def test_two_streams_at_once(kind):
    """Calls over one cache that overlap, each with its own workspace: the bits of calls alone."""
    r = rng(83)
    P, H, HK, hd, B = 16, 8, 4, 64, 12
    q, c, table, kv, cu, g, o = case_of(r, kind, [0, 7, 12], [40, 21], [70] * B, [1] * B, P, H, HK, hd, pad=3)
    table, (members, new, prefix, _) = Q.forced(c, table, kv, cu, g, H)
    L, n_pages, rows = N.lib(), len(c["k"]), len(q)
    size = (rows, B, 2, members, new, prefix, 80, H, HK, hd)
    d = Q.upload(c)
    dt, dl, dc, dg = M.ints(table), M.ints(kv), M.ints(cu), M.ints(g)
    streams = [stream(), N.Stream()]
    queries = [q, r.standard_normal(q.shape).astype(np.float32)]
    dq, do, ds = [up(x) for x in queries], [up(o), up(o)], [M.ints(np.zeros(B)), M.ints(np.zeros(B))]
    w = [M.ws("cdml_paged_attn_shared_workspace_size", *size) for _ in streams]

    def call(i):
        st = streams[i].handle
        N.check(L.cdml_paged_shared(dt.ptr, table.shape[1], dl.ptr, dc.ptr, dg.ptr, 2, B, n_pages, P, ds[i].ptr, st))
        N.check(L.cdml_paged_attn_shared(dq[i].ptr, H * hd, *(Q.ptr(b) for b in d), N.CACHE[kind], n_pages, P, dt.ptr,
                                         table.shape[1], dl.ptr, dc.ptr, dg.ptr, ds[i].ptr, do[i].ptr, H * hd, *size,
                                         0.125, None, w[i][0].ptr, w[i][1], st))

    def results():
        for s in streams:
            s.synchronize()
        return [down(x, o.shape) for x in do]

    for i in range(2):
        call(i)
        streams[i].synchronize()
    alone = results()
    for i in range(2):
        want, tol = M.attention(queries[i], c["kx"], c["vx"], table, kv, cu, P, H, HK, 0.125, o)
        compare(alone[i], want, tol + underflow(c, kv))
    for x in do:
        x.upload(o, streams[0])
    streams[0].synchronize()
    for _ in range(8):
        call(0)
        call(1)
    for got, want in zip(results(), alone):
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("kind", ["f32", "i8", "f8"])
def test_prompts_beams_and_reordering_together(kind):
    """A run as a server makes it: ragged prompts planned and appended for the first beam of each, the tables
    copied to the others by a reordering, then steps of one token that share the prompts, with reorderings between."""
    r = rng(83)
    prompts, beams, P, H, HK, hd, steps = [37, 20, 64], 4, 16, 4, 2, 32, 12
    R, blocks = len(prompts) * beams, 8
    q8 = kind in ("i8", "f8")
    pages = R * blocks
    c = {"kind": kind, "P": P, "heads": HK, "hd": hd}
    for side in "kv":
        Q.put(c, side, np.zeros((pages, P, HK, hd), np.float32))
    refs, table, kv = np.zeros(pages, np.int32), np.full((R, blocks), -1, np.int32), np.zeros(R, np.int32)
    groups = np.arange(0, R + 1, beams, dtype=np.int32)

    def append(x, slots):
        if q8:
            codes, scales = Q.call_append(x[0], HK * hd, x[1], HK * hd, (c["k"], c["v"]), (c["ks"], c["vs"]), kind, slots, P,
                                          HK, hd)
            (c["k"], c["v"]), (c["ks"], c["vs"]) = codes, scales
            for s in "kv":
                c[s + "x"] = np.moveaxis(Q.values(c[s], c[s + "s"], kind, hd), 1, 2).reshape(pages, P, HK * hd)
        else:
            d = [up(a, a.dtype) for a in (x[0], x[1], c["k"], c["v"], slots)]
            N.check(N.lib().cdml_paged_append(d[0].ptr, HK * hd, d[1].ptr, HK * hd, d[2].ptr, d[3].ptr, 0, d[4].ptr,
                                              len(slots), pages, P, HK * hd, stream().handle))
            for i, s in enumerate("kv"):
                c[s] = down(d[2 + i], c[s].shape)
                c[s + "x"] = c[s].astype(np.float64)

    def copy(src, dst, kv):
        if q8:
            d = [up(c[s], c[s].dtype) for s in ("k", "v", "ks", "vs")] + [M.ints(a) for a in (src, dst, kv)]
            N.check(N.lib().cdml_paged_copy_q8(*(b.ptr for b in d[:4]), 1, 0, pages, P, HK, hd, *(b.ptr for b in d[4:]), R,
                                               stream().handle))
            for b, s in zip(d, ("k", "v", "ks", "vs")):
                c[s] = down(b, c[s].shape, c[s].dtype)
            for s in "kv":
                c[s + "x"] = np.moveaxis(Q.values(c[s], c[s + "s"], kind, hd), 1, 2).reshape(pages, P, HK * hd)
        else:
            d = [up(c[s]) for s in "kv"] + [M.ints(a) for a in (src, dst, kv)]
            N.check(N.lib().cdml_paged_copy(d[0].ptr, d[1].ptr, 0, 1, 0, pages, P, HK * hd, *(b.ptr for b in d[2:]), R,
                                            stream().handle))
            for i, s in enumerate("kv"):
                c[s] = down(d[i], c[s].shape)
                c[s + "x"] = c[s].astype(np.float64)

    tokens = [[] for _ in range(R)]  # every request's K rows, as they were given
    for step in range(steps):
        new = np.ones(R, np.int32)
        if step == 0:
            new[:] = 0
            new[::beams] = prompts
        rows = int(new.sum())
        refs, table, kv, cu, slots, _, status = M.call_plan(refs, table, kv, new, P, rows)
        assert status[0] == 0
        x = normal_rows(r, 2, rows, HK, hd).reshape(2, rows, HK * hd)
        append(x, slots)
        for b in range(R):
            tokens[b] += list(x[0, cu[b]:cu[b + 1]])
        q, o = (r.standard_normal((rows, H * hd)).astype(np.float32) for _ in range(2))
        check(q, c, table, kv, cu, groups, o, H)
        parents = np.repeat(groups[:-1], beams) + (0 if step == 0 else r.integers(0, beams, R))
        refs, table, kv, src, dst, status = M.call_reorder(refs, table, kv, parents.astype(np.int32), P)
        assert status[0] == 0
        copy(src, dst, kv)
        tokens = [list(tokens[p]) for p in parents]
    found = Q.shared(table, kv, np.zeros(R + 1, np.int32), groups, P, pages)
    assert [found[i] for i in range(0, R, beams)] >= [32, 16, 64]
    # what is in the cache, read back
    last = np.concatenate([[0], np.cumsum(kv)]).astype(np.int32)
    k, _, bad = Q.call_read(c, table, kv, last, int(last[-1]), HK * hd, HK * hd)
    want = np.concatenate([np.array(t) for t in tokens]).reshape(-1, HK, hd)
    if q8:
        want = Q.values(*Q.quantise(want, kind), kind, hd).astype(np.float32)
    np.testing.assert_array_equal(k.reshape(want.shape), want)
    assert bad == 0
