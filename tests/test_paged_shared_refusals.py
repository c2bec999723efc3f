"""What the entries of shared prefixes refuse, before they touch a device."""
from __future__ import annotations

import ctypes as C

from cdml import native as N
from test_paged_refusals import BIG, ODD, P, POOL, refused


def test_find_refusals():
    good = dict(table=P, max_blocks=4, kv_len=P, cu=P, group_start=P, groups=2, batch=5, n_pages=8, page_size=16, shared=P,
                stream=None)
    refused("cdml_paged_shared", good, POOL + [
        {"max_blocks": 0}, {"max_blocks": BIG}, {"batch": -1}, {"batch": 4097}, {"groups": -1}, {"groups": 6}] + [
        {k: None} for k in ("table", "kv_len", "cu", "group_start", "shared")])
    assert N.lib().cdml_paged_shared(*{**good, "batch": 0, "groups": 0, "table": None}.values()) == N.OK


ATTN = dict(q=P, ldq=256, kc=P, vc=P, ks=P, vs=P, type=3, n_pages=8, page_size=16, table=P, max_blocks=4, kv_len=P, cu=P,
            group_start=P, shared=P, o=P, ldo=256, rows=6, batch=6, groups=2, max_members=3, max_new=1, max_prefix=32,
            max_tail=32, heads=4, kv_heads=2, hd=64, scale=0.125, bad=None, ws=P, bytes=1 << 30, stream=None)


def test_attention_refusals():
    refused("cdml_paged_attn_shared", ATTN, POOL + [
        {"type": 5}, {"type": -1}, {"max_blocks": 0}, {"batch": -1}, {"batch": 4097}, {"rows": -1}, {"max_new": -1},
        {"groups": -1}, {"groups": 7}, {"max_members": -1}, {"max_prefix": -1}, {"max_tail": -1}, {"max_tail": 65},
        {"max_prefix": 65},
        {"max_prefix": BIG, "max_tail": BIG}, {"heads": 0}, {"kv_heads": 0}, {"kv_heads": 3}, {"hd": 0}, {"hd": 257},
        {"ldq": 255}, {"ldo": 255}, {"max_new": BIG}, {"kc": ODD}, {"vc": ODD}, {"rows": 2 ** 30}, {"rows": 2 ** 24}] + [
        {k: None} for k in ("q", "kc", "vc", "ks", "vs", "table", "kv_len", "cu", "group_start", "shared", "o")])
    for empty in ({"rows": 0}, {"batch": 0, "groups": 0}, {"max_new": 0}):
        assert N.lib().cdml_paged_attn_shared(*{**ATTN, **empty, "q": None}.values()) == N.OK


# Sizes that are worth sharing; those above run as every request's own, which needs no workspace.
SHARING = {**ATTN, "max_blocks": 1024, "ldq": 4096, "ldo": 4096, "rows": 64, "batch": 64, "groups": 1, "max_members": 64,
           "max_prefix": 8192, "max_tail": 512, "heads": 32, "kv_heads": 8, "hd": 128}


def test_attention_workspace():
    size = C.c_size_t(0)
    n = N.lib().cdml_paged_attn_shared_workspace_size
    assert n(6, 6, 2, 3, 1, 32, 32, 4, 2, 64, None) == N.E_INVALID
    assert n(6, 6, 7, 3, 1, 32, 32, 4, 2, 64, C.byref(size)) == N.E_INVALID
    assert n(6, 6, 2, 3, 1, 32, 32, 4, 3, 64, C.byref(size)) == N.E_INVALID
    assert n(6, 6, 2, 3, 1, 32, 32, 4, 2, 64, C.byref(size)) == N.OK and size.value == 0
    assert n(64, 64, 1, 64, 1, 8192, 512, 32, 8, 128, C.byref(size)) == N.OK and size.value > 0
    refused("cdml_paged_attn_shared", {**SHARING, "bytes": size.value}, [
        {"ws": None}, {"ws": ODD}, {"bytes": 4}, {"bytes": size.value - 1}])
