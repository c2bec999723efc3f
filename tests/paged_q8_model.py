"""Plain restatements of the 8-bit paged cache in numpy and float64 (test helper), and
numpy-in, numpy-out calls of its C-ABI entries."""
from __future__ import annotations

import numpy as np
import torch

from abi_ops import down, stream, up
from cdml import native as N
from paged_model import from_bits, ints, raw_dtype, to_bits, ws


def width(hd):
    return -(-hd // 16) * 16


def quantise(x, kind):
    """fp32 [..., hd] -> (codes uint8 [..., width], scales fp32 [...])."""
    x = np.asarray(x, np.float32)
    codes = np.zeros(x.shape[:-1] + (width(x.shape[-1]),), np.uint8)
    finite = np.isfinite(x).all(-1)
    x = np.where(finite[..., None], x, 0).astype(np.float64)
    most = np.abs(x).max(-1)
    if kind == "i8":
        s = np.maximum((most / 127).astype(np.float32), np.float32(2.0 ** -126)).astype(np.float64)
        c = np.rint(x / s[..., None]).astype(np.int8).view(np.uint8)  # (a quotient that is no tie is 2^-33 from one)
    else:
        s = np.full(most.shape, 2.0 ** -126)
        while (448 * s < most).any():
            s = np.where(448 * s < most, 2 * s, s)
        q = torch.from_numpy((x / s[..., None]).astype(np.float32))  # exact, or below 2^-10 and rounded to 0
        c = q.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    codes[..., :x.shape[-1]] = c
    codes[most == 0] = 0
    return codes, np.where(finite, np.where(most > 0, s, 0), np.nan).astype(np.float32)


def values(codes, scales, kind, hd):
    """float64 values [..., hd]."""
    c = np.ascontiguousarray(codes[..., :hd])
    c = c.view(np.int8).astype(np.float64) if kind == "i8" else (
        torch.from_numpy(c).view(torch.float8_e4m3fn).to(torch.float64).numpy())
    with np.errstate(invalid="ignore"):
        return c * np.asarray(scales, np.float64)[..., None]


def in_place(cache, slots, P):
    """Rows [len(slots), heads, ...] of a cache [pages, heads, P, ...]."""
    return cache[slots // P, :, slots % P]


def random_rows(r, n, heads, hd):
    """Rows of very different sizes, a few channels larger than the others."""
    x = r.standard_normal((n, heads, hd)) * 10.0 ** r.integers(-3, 3, (n, heads, 1))
    x[..., 3::16] *= 8
    return x.astype(np.float32)


def random_cache(r, kind, pages, P, heads, hd):
    """{"kind", "k", "v": raw arrays, "ks", "vs": scales or None, "kx", "vx": float64 [pages, P, heads * hd]}."""
    c = {"kind": kind, "P": P, "heads": heads, "hd": hd}
    for side in "kv":
        x = random_rows(r, pages * P, heads, hd) if kind in ("i8", "f8") else r.standard_normal(
            (pages * P, heads, hd)).astype(np.float32)
        put(c, side, x.reshape(pages, P, heads, hd))
    return c


def put(c, side, x):
    """Fills a side of a cache from fp32 [pages, P, heads, hd]."""
    pages, P, heads, hd = x.shape
    if c["kind"] in ("i8", "f8"):
        codes, scales = quantise(np.moveaxis(x, 2, 1), c["kind"])
        c[side], c[side + "s"] = np.ascontiguousarray(codes), np.ascontiguousarray(scales)
        val = np.moveaxis(values(codes, scales, c["kind"], hd), 1, 2)
    else:
        c[side], c[side + "s"] = to_bits(x.reshape(pages, P, heads * hd), c["kind"]), None
        val = from_bits(c[side], c["kind"]).astype(np.float64)
    c[side + "x"] = np.ascontiguousarray(val).reshape(pages, P, heads * hd)


def upload(c):
    """(k, v, kscale, vscale) as device buffers, None for the scales that a type has not."""
    raw = np.uint8 if c["kind"] in ("i8", "f8") else raw_dtype(c["kind"])
    return [up(c["k"], raw), up(c["v"], raw)] + [None if c[s] is None else up(c[s]) for s in ("ks", "vs")]


def ptr(b):
    return None if b is None else b.ptr


# ---- calls -------------------------------------------------------------------------

def call_append(k, ldk, v, ldv, codes, scales, kind, slots, P, heads, hd):
    """codes, scales: pairs of the caches' arrays before; returns them after."""
    d = [up(a, a.dtype) for a in (k, v, *codes, *scales, slots)]
    N.check(N.lib().cdml_paged_append_q8(d[0].ptr, ldk, d[1].ptr, ldv, *(b.ptr for b in d[2:6]), N.CACHE[kind],
                                         d[6].ptr, len(slots), len(codes[0]), P, heads, hd, stream().handle))
    return ([down(b, a.shape, np.uint8) for b, a in zip(d[2:4], codes)],
            [down(b, a.shape) for b, a in zip(d[4:6], scales)])


def call_read(c, table, kv, cu, rows, ldk, ldv, fill=7.0, n_pages=None):
    """([rows, ldk], [rows, ldv], bad)."""
    d = upload(c)
    out = [up(np.full((rows, ld), fill, np.float32)) for ld in (ldk, ldv)]
    t, l, u, bad = ints(table), ints(kv), ints(cu), ints(np.zeros(1))
    N.check(N.lib().cdml_paged_read(*(ptr(b) for b in d), N.CACHE[c["kind"]], n_pages or len(c["k"]), c["P"], t.ptr,
                                    table.shape[1], l.ptr, u.ptr, out[0].ptr, ldk, out[1].ptr, ldv, rows, len(kv),
                                    c["heads"], c["hd"], bad.ptr, stream().handle))
    return down(out[0], (rows, ldk)), down(out[1], (rows, ldv)), int(down(bad, (1,), np.int32)[0])


def call_attention(q, c, table, kv, cu, H, scale, o, max_new=None, max_len=None, ldq=None, ldo=None, n_pages=None,
                   filth=True):
    """cdml_paged_attn_q8; q, o [rows, H * hd]; returns (o, bad)."""
    rows, B, hd = len(q), len(kv), c["hd"]
    ldq, ldo = ldq or q.shape[1], ldo or o.shape[1]
    wide = np.full((rows, ldq), np.nan, np.float32)
    wide[:, :q.shape[1]] = q
    out = np.full((rows, ldo), 7.0, np.float32)
    out[:, :o.shape[1]] = o
    max_new = int(np.max(np.diff(cu), initial=0)) if max_new is None else max_new
    max_len = int(np.max(kv, initial=0)) if max_len is None else max_len
    dq, do, d = up(wide), up(out), upload(c)
    dt, dl, dc, bad = ints(table), ints(kv), ints(cu), ints(np.zeros(1))
    size = (rows, B, max_new, max_len, H, c["heads"], hd)
    w, n = ws("cdml_paged_attn_q8_workspace_size", *size)
    if filth:
        w.upload(np.full(max(n // 4, 1), np.nan, np.float32), stream())
    N.check(N.lib().cdml_paged_attn_q8(dq.ptr, ldq, *(b.ptr for b in d), N.CACHE[c["kind"]], n_pages or len(c["k"]),
                                       c["P"], dt.ptr, table.shape[1], dl.ptr, dc.ptr, do.ptr, ldo, *size, scale, bad.ptr,
                                       w.ptr, n, stream().handle))
    out = down(do, out.shape)
    assert (out[:, o.shape[1]:] == 7.0).all()
    return out[:, :o.shape[1]], int(down(bad, (1,), np.int32)[0])


def unseen_filth(c, table, lens):
    """NaN scales, and codes that are NaN as e4m3, in every slot that no request has."""
    if c["kind"] not in ("i8", "f8"):
        for s in "kv":
            used = np.zeros((len(c["k"]), c["P"]), bool)
            mark(used, table, lens, c["P"])
            c[s][~used] = to_bits(np.full(1, np.nan), c["kind"])[0]
        return
    used = np.zeros((len(c["k"]), c["P"]), bool)
    mark(used, table, lens, c["P"])
    for s in "kv":
        c[s] = np.where(used[:, None, :, None], c[s], np.uint8(0x7f if c["kind"] == "f8" else 0x80))
        c[s + "s"] = np.where(used[:, None], c[s + "s"], np.float32(np.nan))


def mark(used, table, lens, P):
    for b, m in enumerate(lens):
        at = np.arange(m)
        used[table[b, at // P], at % P] = True


# ---- shared prefixes ---------------------------------------------------------------

def shared(table, kv, cu, groups, P, n_pages):
    """Tokens that every request shares with its group (groups: group_start)."""
    B, blocks = table.shape
    out = np.zeros(B, np.int32)
    for first, behind in zip(groups[:-1], groups[1:]):
        if behind - first < 2:
            continue
        pages = min([blocks] + [max(0, int(kv[b]) - int(cu[b + 1] - cu[b])) // P for b in range(first, behind)])
        n = 0
        while n < pages and 0 <= table[first, n] < n_pages and (table[first:behind, n] == table[first, n]).all():
            n += 1
        out[first:behind] = n * P
    return out


def call_shared(table, kv, cu, groups, P, n_pages, fill=-9):
    d = [ints(a) for a in (table, kv, cu, groups, np.full(max(len(kv), 1), fill))]
    N.check(N.lib().cdml_paged_shared(d[0].ptr, table.shape[1], d[1].ptr, d[2].ptr, d[3].ptr, len(groups) - 1, len(kv),
                                      n_pages, P, d[4].ptr, stream().handle))
    return down(d[4], (len(kv),), np.int32)


def forced(c, table, kv, cu, groups, H):
    """Bounds (max_members, max_new, max_prefix, max_tail) for which the entry shares, whatever there is to be shared,
    and a table of as many columns; None where no length of a prefix is worth it.  (The entry's own estimate: requests
    of few rows read at 6 TB/s, tiles of 128 rows and 32 keys take a time of their own, a launch and a join 12 us.)"""
    (B, blocks), P, hd, kv_heads = table.shape, c["P"], c["hd"], c["heads"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "f8": 1}[c["kind"]]
    members, new = int(np.max(np.diff(groups), initial=0)), int(np.max(np.diff(cu), initial=0))
    tile = (0.5 if hd <= 32 else 0.85 if hd <= 64 else 1.5) * (1.8 if size == 4 else 1)

    def us(readers, rows):  # a key
        if rows <= 16:
            return readers * kv_heads * 2 * hd * size / 6e6
        return readers * kv_heads / 32 * -(-rows // 128) * tile * (0.6 if rows <= 64 else 1) / 256
    rows = new * (H // kv_heads)
    gain = us(B, rows) - us(len(groups) - 1, rows * members)
    if hd > 128 or members < 2 or gain <= 0 or 13 / gain > 2 ** 22:
        return None
    most = max(int(13 / gain) + 1, blocks * P)
    more = -(-most // P) - blocks
    return np.concatenate([table, np.full((B, more), -1, np.int32)], 1), (members, new, most, blocks * P)


def call_attention_shared(q, c, table, kv, cu, groups, H, scale, o, bounds=None, ldq=None, ldo=None, n_pages=None,
                          force=False):
    """cdml_paged_shared and cdml_paged_attn_shared; bounds: max_members, max_new, max_prefix, max_tail.  force:
    bounds for which it shares, shown by tables in which only the first member of a group holds what is shared.
    Returns (o, shared, bad)."""
    lead = forced(c, table, kv, cu, groups, H) if force else None
    if lead:
        table, bounds = lead
    rows, B, hd, P = len(q), len(kv), c["hd"], c["P"]
    n_pages = n_pages or len(c["k"])
    ldq, ldo = ldq or q.shape[1], ldo or o.shape[1]
    wide = np.full((rows, ldq), np.nan, np.float32)
    wide[:, :q.shape[1]] = q
    out = np.full((rows, ldo), 7.0, np.float32)
    out[:, :o.shape[1]] = o
    if bounds is None:
        s = shared(table, kv, cu, groups, P, n_pages)
        bounds = (int(np.max(np.diff(groups), initial=0)), int(np.max(np.diff(cu), initial=0)), int(np.max(s, initial=0)),
                  int(np.max(kv - s, initial=0)))
    dq, do, d = up(wide), up(out), upload(c)
    dt, dl, dc, dg, ds, bad = (ints(a) for a in (table, kv, cu, groups, np.full(max(B, 1), -9), np.zeros(1)))
    size = (rows, B, len(groups) - 1, *bounds, H, c["heads"], hd)
    w, n = ws("cdml_paged_attn_shared_workspace_size", *size)
    w.upload(np.full(max(n // 4, 1), np.nan, np.float32), stream())
    N.check(N.lib().cdml_paged_shared(dt.ptr, table.shape[1], dl.ptr, dc.ptr, dg.ptr, len(groups) - 1, B, n_pages, P,
                                      ds.ptr, stream().handle))
    if lead:
        alone, s = table.copy(), down(ds, (B,), np.int32)
        for first, behind in zip(groups[:-1], groups[1:]):
            for b in range(first + 1, behind):
                alone[b, :s[b] // P] = -1
        dt = ints(alone)
    N.check(N.lib().cdml_paged_attn_shared(dq.ptr, ldq, *(ptr(b) for b in d), N.CACHE[c["kind"]], n_pages, P, dt.ptr,
                                           table.shape[1], dl.ptr, dc.ptr, dg.ptr, ds.ptr, do.ptr, ldo, *size, scale,
                                           bad.ptr, w.ptr, n, stream().handle))
    out = down(do, out.shape)
    assert (out[:, o.shape[1]:] == 7.0).all()
    return out[:, :o.shape[1]], down(ds, (B,), np.int32), int(down(bad, (1,), np.int32)[0])
