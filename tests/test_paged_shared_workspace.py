"""cdml_paged_attn_shared takes exactly the workspace that its size entry names, for every cache type:
where it shares, and where it runs each request over its own table."""
from __future__ import annotations

import ctypes as C
import itertools

import pytest

from cdml import native as N
from test_paged_refusals import P

TYPES = sorted(N.CACHE.values())


def accepted(batch, groups, members, new, prefix, tail, heads, kv_heads, hd, page=16):
    """Calls of every cache type with what the size entry says get as far as the device that is not there."""
    size, rows = C.c_size_t(0), batch * new
    N.check(N.lib().cdml_paged_attn_shared_workspace_size(rows, batch, groups, members, new, prefix, tail, heads, kv_heads,
                                                          hd, C.byref(size)))
    blocks = max(1, -(-(prefix + tail) // page))
    for kind in TYPES:
        rc = N.lib().cdml_paged_attn_shared(
            P, heads * hd, P, P, P, P, kind, batch * blocks, page, P, blocks, P, P, P, P, P, heads * hd, rows, batch, groups,
            members, new, prefix, tail, heads, kv_heads, hd, 0.125, None, P if size.value else None, size.value, None)
        assert rc == N.E_NODEVICE, (kind, batch, groups, members, new, prefix, tail, heads, kv_heads, hd,
                                    N.lib().cdml_last_error())


@pytest.fixture(autouse=True)
def no_device():
    if N.device_count() > 0:
        pytest.skip("a device is visible: the calls would run")


# (4-byte values of these sizes are worth sharing, 2-byte ones are not)
@pytest.mark.parametrize("case", [(4, 2, 2, 1, 8000, 1000, 32, 8, 128), (8, 1, 8, 1, 1749, 348, 32, 8, 128),
                                  (42, 1, 42, 1, 819, 525, 32, 8, 64)])
def test_sizes_that_only_wide_values_share(case):
    accepted(*case)


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (32, 8), (12, 4), (16, 8), (7, 1), (34, 2)])
def test_what_the_size_entry_says_is_taken(heads, kv_heads):
    for (batch, groups), new, prefix, tail, hd in itertools.product(
            [(1, 0), (2, 1), (4, 2), (7, 3), (16, 1), (64, 8), (300, 2)], [1, 2, 30], [0, 100, 819, 1749, 8000],
            [0, 1, 348, 1000, 5000], [7, 64, 128, 200]):
        accepted(batch, groups, -(-batch // max(groups, 1)), new, prefix, tail, heads, kv_heads, hd)
