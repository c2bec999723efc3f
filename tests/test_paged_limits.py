"""Sizes at the limits of the paged attention's launches, refused or accepted before a device is touched."""
from __future__ import annotations

import ctypes as C

import pytest

from cdml import native as N

ROWS = 128 * (2 ** 24 // 64 - 1)  # tiles of 64 K/V heads: one request below 2^24 workgroups


def size(rows, batch, max_new, heads, kv_heads, hd):
    n = C.c_size_t(0)
    return N.lib().cdml_paged_attn_workspace_size(rows, batch, max_new, 64, heads, kv_heads, hd, C.byref(n))


@pytest.mark.parametrize("rows,batch,heads,kv_heads", [(ROWS, 1, 64, 64), (2 ** 26, 1, 64, 64), (ROWS // 4, 1, 256, 64),
                                                       (2 ** 30, 1, 8, 2)])
def test_more_tiles_than_a_launch_holds_are_refused(rows, batch, heads, kv_heads):
    assert size(rows, batch, 1000, heads, kv_heads, 8) == N.E_INVALID
    assert b"too large" in N.lib().cdml_last_error()
    p = C.c_void_p(4096)  # never dereferenced
    assert N.lib().cdml_paged_attn(p, 8 * heads, p, p, 0, 8, 16, p, 4, p, p, p, 8 * heads, rows, batch, 1000, 64, heads,
                                   kv_heads, 8, 0.1, None, p, 1 << 60, None) == N.E_INVALID


def test_the_largest_launches_are_accepted():
    assert size(ROWS - 128, 1, 1000, 64, 64, 8) == N.OK
    assert size(2 ** 26, 4096, 1, 64, 64, 8) == N.OK      # single tokens: no tiles
    assert size(2 ** 20, 4096, 1000, 16, 16, 256) == N.OK  # nor above head dim 128
