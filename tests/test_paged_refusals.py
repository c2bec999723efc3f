"""What the paged-cache and beam-search entries refuse, before they touch a device."""
from __future__ import annotations

import ctypes as C

import pytest

from cdml import native as N

P = C.c_void_p(4096)  # never dereferenced: every case fails a host check
ODD = C.c_void_p(4100)
BIG = 2 ** 31 - 1


def refused(name, good, changes):
    """`good` as {argument: value}; each change of it has to be refused with a message that names the entry."""
    for change in changes:
        rc = getattr(N.lib(), name)(*{**good, **change}.values())
        assert rc == N.E_INVALID, (change, rc)
        assert name.encode() in N.lib().cdml_last_error(), change


POOL = [{"page_size": n} for n in (0, -1, 3, 24, 8192)] + [
    {"n_pages": 0}, {"n_pages": -4}, {"n_pages": BIG}, {"n_pages": 2 ** 30 + 1, "page_size": 1}]


def test_plan_refusals():
    good = dict(refs=P, n_pages=8, page_size=16, table=P, max_blocks=4, kv_len=P, new_len=P, batch=2, rows=3, cu=P,
                slots=P, positions=P, status=P, stream=None)
    refused("cdml_paged_plan", good, POOL + [
        {"max_blocks": 0}, {"max_blocks": BIG}, {"batch": -1}, {"batch": 4097}, {"rows": -1}, {"rows": BIG},
        {"refs": ODD}] + [
        {k: None} for k in ("refs", "table", "kv_len", "new_len", "cu", "slots", "positions", "status")])


def test_append_refusals():
    good = dict(k=P, ldk=64, v=P, ldv=64, kc=P, vc=P, type=0, slots=P, rows=3, n_pages=8, page_size=16, kv_dim=64,
                stream=None)
    refused("cdml_paged_append", good, POOL + [
        {"type": 3}, {"type": -1}, {"rows": -1}, {"kv_dim": 0}, {"ldk": 63}, {"ldv": 63}] + [
        {k: None} for k in ("k", "v", "kc", "vc", "slots")])
    assert N.lib().cdml_paged_append(*{**good, "rows": 0, "k": None}.values()) == N.OK


ATTN = dict(q=P, ldq=256, kc=P, vc=P, type=2, n_pages=8, page_size=16, table=P, max_blocks=4, kv_len=P, cu=P, o=P,
            ldo=256, rows=6, batch=2, max_new=5, max_len=64, heads=4, kv_heads=2, hd=64, scale=0.125, bad=None, ws=P,
            bytes=1 << 30, stream=None)


def test_attention_refusals():
    refused("cdml_paged_attn", ATTN, POOL + [
        {"type": 7}, {"max_blocks": 0}, {"batch": -1}, {"batch": 4097}, {"rows": -1}, {"max_new": -1}, {"max_len": -1},
        {"max_len": 65}, {"heads": 0}, {"kv_heads": 0}, {"kv_heads": 3}, {"hd": 0}, {"hd": 257}, {"ldq": 255},
        {"ldo": 255}, {"heads": 65536, "kv_heads": 65536, "hd": 1, "ldq": 65536, "ldo": 65536},
        {"max_new": BIG}, {"hd": 200, "ldq": 800, "ldo": 800, "max_new": 100_000}] + [
        {k: None} for k in ("q", "kc", "vc", "table", "kv_len", "cu", "o")])
    for empty in ({"rows": 0}, {"batch": 0}, {"max_new": 0}):
        assert N.lib().cdml_paged_attn(*{**ATTN, **empty, "q": None}.values()) == N.OK


def test_attention_workspace():
    size = C.c_size_t(0)
    n = N.lib().cdml_paged_attn_workspace_size
    assert n(6, 2, 5, 64, 4, 2, 64, None) == N.E_INVALID
    assert n(6, 2, 5, 64, 4, 3, 64, C.byref(size)) == N.E_INVALID
    long = {**ATTN, "max_blocks": 1024, "max_len": 16384, "n_pages": 4096}
    assert n(6, 2, 5, 16384, 4, 2, 64, C.byref(size)) == N.OK and size.value > 0
    refused("cdml_paged_attn", {**long, "bytes": size.value}, [{"bytes": size.value - 1}, {"ws": None}, {"ws": ODD}])


def test_reorder_refusals():
    size = C.c_size_t(0)
    assert N.lib().cdml_paged_reorder_workspace_size(5, 7, C.byref(size)) == N.OK and size.value == 4 * 5 * 8
    assert N.lib().cdml_paged_reorder_workspace_size(5, 0, C.byref(size)) == N.E_INVALID
    assert N.lib().cdml_paged_reorder_workspace_size(4097, 7, C.byref(size)) == N.E_INVALID
    assert N.lib().cdml_paged_reorder_workspace_size(5, 7, None) == N.E_INVALID
    good = dict(refs=P, n_pages=8, page_size=16, table=P, max_blocks=7, kv_len=P, parents=P, batch=5, src=P, dst=P,
                status=P, ws=P, bytes=160, stream=None)
    refused("cdml_paged_reorder", good, POOL + [
        {"max_blocks": 0}, {"batch": -1}, {"batch": 4097}, {"bytes": 159}, {"ws": C.c_void_p(4097)},
        {"refs": ODD}] + [
        {k: None} for k in ("refs", "table", "kv_len", "parents", "src", "dst", "status", "ws")])


def test_copy_refusals():
    good = dict(kc=P, vc=P, type=1, layers=2, stride=8 * 16 * 64, n_pages=8, page_size=16, kv_dim=64, src=P, dst=P,
                kv_len=P, batch=5, stream=None)
    refused("cdml_paged_copy", good, POOL + [
        {"type": 3}, {"layers": -1}, {"layers": 40000}, {"stride": 8 * 16 * 64 - 1}, {"kv_dim": 0}, {"kv_dim": BIG},
        {"batch": -1}] + [{k: None} for k in ("kc", "vc", "src", "dst", "kv_len")])
    for empty in ({"batch": 0}, {"layers": 0}):
        assert N.lib().cdml_paged_copy(*{**good, **empty, "kc": None}.values()) == N.OK


def test_beam_refusals():
    size = C.c_size_t(0)
    n = N.lib().cdml_beam_select_workspace_size
    assert n(2, 4, 50, C.byref(size)) == N.OK and size.value % 16 == 0
    for bad in ((-1, 4, 50), (2, 0, 50), (2, 65, 50), (2, 4, 0), (1100, 60, 50)):
        assert n(*bad, C.byref(size)) == N.E_INVALID, bad
    assert n(2, 4, 50, None) == N.E_INVALID
    assert n(2, 4, 50, C.byref(size)) == N.OK
    good = dict(x=P, ldl=50, scores=P, lengths=P, finished=P, batch=2, beams=4, vocab=50, eos=2, penalty=0.0, ns=P, nl=P,
                nf=P, parents=P, tokens=P, ws=P, bytes=size.value, stream=None)
    refused("cdml_beam_select", good, [
        {"ldl": 49}, {"eos": 50}, {"beams": 0}, {"beams": 65}, {"vocab": 0}, {"batch": -1}, {"bytes": size.value - 1},
        {"ws": ODD}, {"penalty": float("nan")}, {"penalty": 17.0}, {"penalty": -17.0}] + [
        {k: None} for k in ("x", "scores", "lengths", "finished", "ns", "nl", "nf", "parents", "tokens", "ws")])
    assert N.lib().cdml_beam_select(*{**good, "batch": 0, "x": None}.values()) == N.OK


@pytest.mark.parametrize("name", ["cdml_paged_plan", "cdml_paged_attn", "cdml_beam_select"])
def test_entries_are_bound(name):
    assert name in N.SIGNATURES and name in N.header_functions()
