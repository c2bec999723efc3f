"""Plain restatements of the paged-cache and beam-search operators in numpy and float64
(test helper), and numpy-in, numpy-out calls of their C-ABI entries."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from abi_ops import down, stream, up
from cdml import native as N

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cached values as bits ---------------------------------------------------

def to_bits(x, kind):
    """float values rounded to a cache type, as its raw array."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[kind])
    return t.numpy() if kind == "f32" else t.view(torch.int16).numpy()


def from_bits(b, kind):
    t = torch.from_numpy(np.ascontiguousarray(b))
    return t.numpy() if kind == "f32" else t.view(TORCH[kind]).float().numpy()


def raw_dtype(kind):
    return np.float32 if kind == "f32" else np.int16


# ---- plain forms ---------------------------------------------------------------

def plan(refs, table, kv, new, P, rows):
    refs, table, kv = refs.copy(), table.copy(), kv.copy()
    B, blocks = table.shape
    code = need = 0
    toks = 0
    for b in range(B):
        if kv[b] < 0 or new[b] < 0 or kv[b] + new[b] > blocks * P:
            code |= 2
            continue
        need += -(-(int(kv[b]) + int(new[b])) // P) - -(-int(kv[b]) // P)
        toks += int(new[b])
    free = list(np.flatnonzero(refs == 0))
    code |= (1 if need > len(free) else 0) | (4 if toks > rows else 0)
    cu, slots, pos = np.zeros(B + 1, np.int32), np.full(rows, -1, np.int32), np.zeros(rows, np.int32)
    status = np.array([code, need, toks], np.int64)
    if code == 0:
        r = 0
        for b in range(B):
            for t in range(int(kv[b]), int(kv[b] + new[b])):
                if t % P == 0:
                    table[b, t // P] = free.pop(0)
                    refs[table[b, t // P]] = 1
                slots[r], pos[r] = table[b, t // P] * P + t % P, t
                r += 1
            kv[b] += new[b]
            cu[b + 1] = r
    return refs, table, kv, cu, slots, pos, status


def reorder(refs, table, kv, parents, P):
    refs, old, old_kv = refs.copy(), table.copy(), kv.copy()
    table, kv = table.copy(), kv.copy()
    R = len(kv)
    src, dst = np.full(R, -1, np.int32), np.full(R, -1, np.int32)
    for r in range(R):
        for j in range(-(-int(old_kv[r]) // P)):
            refs[old[r, j]] -= 1
    waits, seen, wrong = [], set(), 0
    for r, p in enumerate(parents):
        if not 0 <= p < R:
            wrong += p != -1
            kv[r] = 0
            continue
        n = int(old_kv[p])
        table[r, :n // P] = old[p, :n // P]
        for j in range(n // P):
            refs[old[p, j]] += 1
        kv[r] = n
        if n % P:
            if p in seen:
                waits.append(r)
            else:
                table[r, n // P] = old[p, n // P]
                refs[old[p, n // P]] += 1
        seen.add(p)
    free = list(np.flatnonzero(refs == 0))
    missing = 0
    for r in waits:
        n = int(kv[r])
        if free:
            dst[r] = free.pop(0)
            src[r] = old[parents[r], n // P]
            table[r, n // P] = dst[r]
            refs[dst[r]] = 1
        else:
            kv[r] = n // P * P
            missing += 1
    return refs, table, kv, src, dst, np.array([missing, len(waits) - missing, wrong])


def attention(q, k, v, table, kv, cu, P, H, HK, scale, o):
    """k, v: float64 [pages, P, HK * hd].  (output, the error bound of each of its values).

    Bound: a score is a sum of hd rounded products (hd + 8 steps of 2^-24 of the products'
    absolute sum, pieces and the scaled Q among them), which moves a probability and the
    softmax's sum by as much each; sums over T keys are T steps, the exponential and the
    divisions a few.  (2 (hd + 8) a + 2 T + 32) 2^-24 sum p |v|, a the largest such sum."""
    out, tol = o.astype(np.float64), np.zeros(o.shape)
    hd = q.shape[1] // H
    with np.errstate(all="ignore"):
        for b in range(len(kv)):
            n, T = int(cu[b + 1] - cu[b]), int(kv[b])
            at = np.arange(T)
            rows = slice(int(cu[b]), int(cu[b + 1]))
            kb, vb = k[table[b, at // P], at % P], v[table[b, at // P], at % P]
            for h in range(H):
                g = h // (H // HK)
                kh, vh = kb[:, g * hd:(g + 1) * hd], vb[:, g * hd:(g + 1) * hd]
                for i in range(n):
                    x = q[rows][i, h * hd:(h + 1) * hd].astype(np.float64)
                    seen = max(0, T - n + i + 1)
                    at_out = (int(cu[b]) + i, slice(h * hd, (h + 1) * hd))
                    if not seen:
                        out[at_out] = 0
                        continue
                    s = kh[:seen] @ x * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[at_out] = p @ vh[:seen]
                    a = (np.abs(kh[:seen]) @ np.abs(x)).max() * abs(scale)
                    tol[at_out] = (2 * (hd + 8) * a + 2 * seen + 32) * 2.0 ** -24 * (p @ np.abs(vh[:seen]))
    return out, tol


def beam(x, scores, lengths, done, K, eos, alpha):
    R, V = x.shape
    out = [np.zeros(R, t) for t in (np.float64, np.int32, np.uint8, np.int32, np.int32)]
    for b in range(R // K):
        found = []
        for r in range(b * K, (b + 1) * K):
            s = float(scores[r])
            if not np.isfinite(s):
                continue
            if done[r]:
                found.append((s / max(int(lengths[r]), 1) ** float(np.float32(alpha)), -r, 0, max(eos, 0), s, lengths[r], 1))
                continue
            w = np.where(np.isnan(x[r]), -np.inf, x[r]).astype(np.float64)
            m = w.max()
            if not np.isfinite(m):
                continue
            log_sum = np.log(np.exp(w - m).sum())
            for rank, t in enumerate(np.argsort(-w, kind="stable")[:K]):
                if w[t] > -np.inf:
                    total = s + ((w[t] - m) - log_sum)
                    found.append((total / (int(lengths[r]) + 1) ** float(np.float32(alpha)), -r, -rank, int(t), total,
                                  lengths[r] + 1, int(t == eos)))
        found.sort(key=lambda f: f[:3], reverse=True)
        for k in range(K):
            r = b * K + k
            if k < len(found):
                _, parent, _, t, total, n, d = found[k]
                vals = (total, n, d, -parent, t)
            else:
                vals = (-np.inf, lengths[r], 1, r, max(eos, 0))
            for o, val in zip(out, vals):
                o[r] = val
    return out


# ---- calls -------------------------------------------------------------------------

def ws(name, *args):
    size = C.c_size_t(0)
    N.check(getattr(N.lib(), name)(*args, C.byref(size)))
    return N.DeviceBuffer(max(256, size.value)), size.value


def ints(a):
    return up(a, np.int32)


def call_plan(refs, table, kv, new, P, rows):
    B, blocks = table.shape
    d = [ints(a) for a in (refs, table, kv, new)]
    cu, slots, pos, status = (N.DeviceBuffer(4 * max(n, 1)) for n in (B + 1, rows, rows, 3))
    N.check(N.lib().cdml_paged_plan(d[0].ptr, len(refs), P, d[1].ptr, blocks, d[2].ptr, d[3].ptr, B, rows, cu.ptr,
                                    slots.ptr, pos.ptr, status.ptr, stream().handle))
    return (down(d[0], refs.shape, np.int32), down(d[1], table.shape, np.int32), down(d[2], kv.shape, np.int32),
            down(cu, (B + 1,), np.int32), down(slots, (rows,), np.int32), down(pos, (rows,), np.int32),
            down(status, (3,), np.int32))


def call_reorder(refs, table, kv, parents, P):
    R, blocks = table.shape
    d = [ints(a) for a in (refs, table, kv, parents)]
    src, dst, status = (N.DeviceBuffer(4 * max(n, 1)) for n in (R, R, 3))
    w, n = ws("cdml_paged_reorder_workspace_size", R, blocks)
    N.check(N.lib().cdml_paged_reorder(d[0].ptr, len(refs), P, d[1].ptr, blocks, d[2].ptr, d[3].ptr, R, src.ptr,
                                       dst.ptr, status.ptr, w.ptr, n, stream().handle))
    return (down(d[0], refs.shape, np.int32), down(d[1], table.shape, np.int32), down(d[2], kv.shape, np.int32),
            down(src, (R,), np.int32), down(dst, (R,), np.int32), down(status, (3,), np.int32))


def call_attention(q, kbits, vbits, kind, table, kv, cu, P, H, HK, scale, o, max_new=None, max_len=None, ldq=None,
                   n_pages=None, ldo=None):
    """q, o [rows, H * hd]; returns (o, bad)."""
    rows, B, hd = len(q), len(kv), q.shape[1] // H
    ldq = ldq or q.shape[1]
    wide = np.full((rows, ldq), np.nan, np.float32)
    wide[:, :q.shape[1]] = q
    max_new = int(np.max(np.diff(cu), initial=0)) if max_new is None else max_new
    max_len = int(np.max(kv, initial=0)) if max_len is None else max_len
    ldo = ldo or o.shape[1]
    out = np.full((rows, ldo), 7.0, np.float32)
    out[:, :o.shape[1]] = o
    dq, dk, dv, do = up(wide), up(kbits, raw_dtype(kind)), up(vbits, raw_dtype(kind)), up(out)
    dt, dl, dc, bad = ints(table), ints(kv), ints(cu), ints(np.zeros(1))
    w, n = ws("cdml_paged_attn_workspace_size", rows, B, max_new, max_len, H, HK, hd)
    N.check(N.lib().cdml_paged_attn(dq.ptr, ldq, dk.ptr, dv.ptr, N.CACHE[kind], n_pages or len(kbits), P, dt.ptr,
                                    table.shape[1], dl.ptr, dc.ptr, do.ptr, ldo, rows, B, max_new, max_len, H, HK,
                                    hd, scale, bad.ptr, w.ptr, n, stream().handle))
    out = down(do, out.shape)
    assert (out[:, o.shape[1]:] == 7.0).all()
    return out[:, :o.shape[1]], int(down(bad, (1,), np.int32)[0])


def call_beam(x, scores, lengths, done, K, eos, alpha, in_place=False, ldl=None):
    R, V = x.shape
    ldl = ldl or V
    wide = np.full((R, ldl), np.nan, np.float32)
    wide[:, :V] = x
    dx, ds, dl, dd = up(wide), up(scores), ints(lengths), up(done, np.uint8)
    out = [ds, dl, dd] if in_place else [N.DeviceBuffer(4 * R), N.DeviceBuffer(4 * R), N.DeviceBuffer(R)]
    par, tok = N.DeviceBuffer(4 * R), N.DeviceBuffer(4 * R)
    w, n = ws("cdml_beam_select_workspace_size", R // K, K, V)
    N.check(N.lib().cdml_beam_select(dx.ptr, ldl, ds.ptr, dl.ptr, dd.ptr, R // K, K, V, eos, alpha, out[0].ptr,
                                     out[1].ptr, out[2].ptr, par.ptr, tok.ptr, w.ptr, n, stream().handle))
    return (down(out[0], (R,)), down(out[1], (R,), np.int32), down(out[2], (R,), np.uint8), down(par, (R,), np.int32),
            down(tok, (R,), np.int32))
