"""Pages whose codes lie past 2^32 bytes of an 8-bit cache, and past 2^32 values of a bf16 one: appending, reading, copying
and attention give the bits that they give over the same pages at the beginning of a small pool (which the other tests
compare with float64)."""
from __future__ import annotations

import numpy as np
import pytest

import paged_model as M
import paged_q8_model as Q
from abi_ops import down, stream, up
from cdml import native as N
from test_gpu_paged import rng
from test_gpu_paged_attn_q8 import normal_rows
from test_gpu_paged_shared import tables

pytestmark = pytest.mark.gpu

P, HK, H, HD = 16, 8, 16, 128
GROUPS, PREFIX = [0, 4, 7], [10, 7]
TAILS = [20, 1, 33, 50, 16, 40, 17]
FAR = 600_000  # pages of 16 KiB of codes a side, 32 of bf16


def cache_of(kind, n_pages, layers):
    """Zeroed (k, v, kscale, vscale) of `layers` layers."""
    rows, q8 = layers * n_pages * HK * P, kind in ("i8", "f8")
    sizes = [rows * HD * (1 if q8 else 2)] * 2 + ([4 * rows] * 2 if q8 else [])
    c = [N.DeviceBuffer(n) for n in sizes]
    for b in c:
        N.check(N.lib().cdml_zero_f32_async(b.ptr, b.nbytes // 4, stream().handle))
    return c + [None] * (4 - len(c))


def results(kind, n_pages, new):
    """Every entry's outputs over the pool's last pages."""
    L, st, r, B = N.lib(), stream().handle, rng(110), len(TAILS)
    lens = np.array([PREFIX[g] * P + TAILS[b] for g in range(2) for b in range(GROUPS[g], GROUPS[g + 1])], np.int32)
    blocks = int(-(-lens.max() // P)) + 1
    table, used = tables(r, GROUPS, PREFIX, lens, P, blocks)
    used += 2  # two more for the copies
    off = n_pages - used
    table = np.where(table >= 0, table + off, -1).astype(np.int32)
    q8 = kind in ("i8", "f8")
    c = cache_of(kind, n_pages, 2 if q8 else 1)
    p = [Q.ptr(b) for b in c]
    x = [up(normal_rows(r, used, P, HK, HD).reshape(used * P, HK * HD)) for _ in range(2)]
    slots = M.ints((r.permutation(used * P) + off * P).astype(np.int32))
    if q8:
        N.check(L.cdml_paged_append_q8(x[0].ptr, HK * HD, x[1].ptr, HK * HD, *p, N.CACHE[kind], slots.ptr, used * P, n_pages,
                                       P, HK, HD, st))
    else:
        N.check(L.cdml_paged_append(x[0].ptr, HK * HD, x[1].ptr, HK * HD, p[0], p[1], N.CACHE[kind], slots.ptr, used * P,
                                    n_pages, P, HK * HD, st))
    out = {}
    dl, bad = M.ints(lens), M.ints(np.zeros(1))

    def read(name, table, lens):
        cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        y = [N.DeviceBuffer(4 * int(cu[-1]) * HK * HD) for _ in range(2)]
        d = [M.ints(a) for a in (table, lens, cu)]
        N.check(L.cdml_paged_read(*p, N.CACHE[kind], n_pages, P, d[0].ptr, table.shape[1], d[1].ptr, d[2].ptr, y[0].ptr,
                                  HK * HD, y[1].ptr, HK * HD, int(cu[-1]), len(lens), HK, HD, bad.ptr, st))
        out[name] = [down(b, (int(cu[-1]), HK * HD)) for b in y]
    read("read", table, lens)

    news = np.minimum(new, TAILS).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    rows = int(cu[-1])
    q, o = up(r.standard_normal((rows, H * HD))), N.DeviceBuffer(4 * rows * H * HD)
    dc = M.ints(cu)
    if q8:
        t, size = M.ints(table), (rows, B, new, int(lens.max()), H, HK, HD)
        w, n = M.ws("cdml_paged_attn_q8_workspace_size", *size)
        N.check(L.cdml_paged_attn_q8(q.ptr, H * HD, *p, N.CACHE[kind], n_pages, P, t.ptr, blocks, dl.ptr, dc.ptr, o.ptr,
                                     H * HD, *size, 0.09, bad.ptr, w.ptr, n, st))
        out["attn"] = down(o, (rows, H * HD))

    # shared: only the first member's table has what the group shares
    wide, bounds = Q.forced({"kind": kind, "P": P, "heads": HK, "hd": HD}, table, lens, cu, GROUPS, H)
    t, dg, ds = M.ints(wide), M.ints(np.array(GROUPS)), M.ints(np.zeros(B))
    N.check(L.cdml_paged_shared(t.ptr, wide.shape[1], dl.ptr, dc.ptr, dg.ptr, 2, B, n_pages, P, ds.ptr, st))
    s = down(ds, (B,), np.int32)
    assert [s[0], s[4]] == [PREFIX[0] * P, PREFIX[1] * P]
    for g in range(2):
        for b in range(GROUPS[g] + 1, GROUPS[g + 1]):
            wide[b, :PREFIX[g]] = -1
    t, size = M.ints(wide), (rows, B, 2, *bounds, H, HK, HD)
    w, n = M.ws("cdml_paged_attn_shared_workspace_size", *size)
    N.check(L.cdml_paged_attn_shared(q.ptr, H * HD, *p, N.CACHE[kind], n_pages, P, t.ptr, wide.shape[1], dl.ptr, dc.ptr,
                                     dg.ptr, ds.ptr, o.ptr, H * HD, *size, 0.09, bad.ptr, w.ptr, n, st))
    out["shared"] = down(o, (rows, H * HD))
    if q8:  # an open page of both layers, the second of which is read
        src, dst = np.array([table[0, 3], -1], np.int32), np.array([n_pages - 1, -1], np.int32)
        N.check(L.cdml_memcpy_d2d_async(p[0] + c[0].nbytes // 2, p[0], c[0].nbytes // 2, st))
        N.check(L.cdml_memcpy_d2d_async(p[2] + c[2].nbytes // 2, p[2], c[2].nbytes // 2, st))
        d = [M.ints(a) for a in (src, dst, np.array([11, 0], np.int32))]
        N.check(L.cdml_paged_copy_q8(*p, 2, n_pages * P, n_pages, P, HK, HD, *(b.ptr for b in d), 2, st))
        half = [p[0] + c[0].nbytes // 2, p[1], p[2] + c[2].nbytes // 2, p[3]]
        p[:] = half
        read("copied", np.array([[n_pages - 1]], np.int32), np.array([11], np.int32))
        read("original", np.array([[table[0, 3]]], np.int32), np.array([11], np.int32))
        np.testing.assert_array_equal(out["copied"][0], out["original"][0])
    assert down(bad, (1,), np.int32)[0] == 0
    stream().synchronize()
    for b in c:
        if b:
            b.free()
    return out


@pytest.mark.parametrize("kind", ["i8", "f8", "bf16"])
@pytest.mark.parametrize("new", [1, 20])
def test_far_pages(kind, new):
    near, far = results(kind, 300, new), results(kind, FAR, new)
    for name, want in near.items():
        for a, b in zip(want, far[name]) if isinstance(want, list) else [(want, far[name])]:
            assert np.isfinite(a).all() and np.abs(a).max() > 0.1
            np.testing.assert_array_equal(a, b)
