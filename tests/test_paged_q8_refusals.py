"""What the entries of 8-bit caches refuse, before they touch a device."""
from __future__ import annotations

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
