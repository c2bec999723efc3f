"""What the entries of 8-bit caches refuse, before they touch a device."""
from __future__ import annotations

import ctypes as C

from cdml import native as N
from test_paged_refusals import BIG, ODD, P, POOL, refused


def test_append_refusals():
    good = dict(k=P, ldk=128, v=P, ldv=128, kc=P, vc=P, ks=P, vs=P, type=3, slots=P, rows=3, n_pages=8, page_size=16,
                heads=2, hd=64, stream=None)
    refused("cdml_paged_append_q8", good, POOL + [
        {"type": 0}, {"type": 2}, {"type": 5}, {"type": -1}, {"rows": -1}, {"heads": 0}, {"heads": -2}, {"hd": 0},
        {"hd": 257}, {"ldk": 127}, {"ldv": 127}, {"rows": BIG}, {"heads": BIG}, {"kc": ODD}, {"vc": ODD}] + [
        {k: None} for k in ("k", "v", "kc", "vc", "ks", "vs", "slots")])
    assert N.lib().cdml_paged_append_q8(*{**good, "rows": 0, "k": None}.values()) == N.OK


def test_read_refusals():
    good = dict(kc=P, vc=P, ks=P, vs=P, type=4, n_pages=8, page_size=16, table=P, max_blocks=4, kv_len=P, cu=P, k=P,
                ldk=128, v=P, ldv=128, rows=6, batch=2, heads=2, hd=64, bad=None, stream=None)
    refused("cdml_paged_read", good, POOL + [
        {"type": 5}, {"type": -1}, {"max_blocks": 0}, {"max_blocks": BIG}, {"batch": -1}, {"batch": 4097}, {"rows": -1},
        {"heads": 0}, {"hd": 0}, {"hd": 257}, {"ldk": 127}, {"ldv": 127}, {"kc": ODD}] + [
        {k: None} for k in ("kc", "vc", "ks", "vs", "table", "kv_len", "cu", "k", "v")])
    for empty in ({"rows": 0}, {"batch": 0}):
        assert N.lib().cdml_paged_read(*{**good, **empty, "k": None}.values()) == N.OK


def test_copy_refusals():
    good = dict(kc=P, vc=P, ks=P, vs=P, layers=2, stride=8 * 16, n_pages=8, page_size=16, heads=2, hd=64, src=P, dst=P,
                kv_len=P, batch=5, stream=None)
    refused("cdml_paged_copy_q8", good, POOL + [
        {"layers": -1}, {"layers": 40000}, {"stride": 8 * 16 - 1}, {"heads": 0}, {"hd": 0}, {"hd": 257}, {"batch": -1},
        {"heads": 2 ** 22, "hd": 64, "page_size": 4096}, {"kc": ODD}, {"vc": ODD}] + [
        {k: None} for k in ("kc", "vc", "ks", "vs", "src", "dst", "kv_len")])
    for empty in ({"batch": 0}, {"layers": 0}):
        assert N.lib().cdml_paged_copy_q8(*{**good, **empty, "kc": None}.values()) == N.OK


ATTN = dict(q=P, ldq=256, kc=P, vc=P, ks=P, vs=P, type=3, n_pages=8, page_size=16, table=P, max_blocks=4, kv_len=P, cu=P,
            o=P, ldo=256, rows=6, batch=2, max_new=5, max_len=64, heads=4, kv_heads=2, hd=64, scale=0.125, bad=None,
            ws=P, bytes=1 << 30, stream=None)


def test_attention_refusals():
    refused("cdml_paged_attn_q8", ATTN, POOL + [
        {"type": 0}, {"type": 2}, {"type": 5}, {"max_blocks": 0}, {"batch": -1}, {"batch": 4097}, {"rows": -1},
        {"max_new": -1}, {"max_len": -1}, {"max_len": 65}, {"heads": 0}, {"kv_heads": 0}, {"kv_heads": 3}, {"hd": 0},
        {"hd": 257}, {"ldq": 255}, {"ldo": 255}, {"max_new": BIG}, {"kc": ODD}, {"vc": ODD},
        {"hd": 200, "ldq": 800, "ldo": 800, "max_new": 100_000}] + [
        {k: None} for k in ("q", "kc", "vc", "ks", "vs", "table", "kv_len", "cu", "o")])
    for empty in ({"rows": 0}, {"batch": 0}, {"max_new": 0}):
        assert N.lib().cdml_paged_attn_q8(*{**ATTN, **empty, "q": None}.values()) == N.OK


def test_attention_workspace():
    size = C.c_size_t(0)
    n = N.lib().cdml_paged_attn_q8_workspace_size
    assert n(6, 2, 5, 64, 4, 2, 64, None) == N.E_INVALID
    assert n(6, 2, 5, 64, 4, 3, 64, C.byref(size)) == N.E_INVALID
    long = {**ATTN, "max_blocks": 1024, "max_len": 16384, "n_pages": 4096}
    assert n(6, 2, 5, 16384, 4, 2, 64, C.byref(size)) == N.OK and size.value > 0
    refused("cdml_paged_attn_q8", {**long, "bytes": size.value}, [{"bytes": size.value - 1}, {"ws": None}, {"ws": ODD}])
