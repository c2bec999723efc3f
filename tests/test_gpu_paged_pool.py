"""The paged cache's tables where their arrays share one buffer, and where an entry is no page."""
from __future__ import annotations

import numpy as np
import pytest

import paged_model as M
from abi_ops import down, stream
from cdml import native as N
from test_gpu_paged import rng, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [2, 8, 16, 40])
@pytest.mark.parametrize("odd", [4, 20, 28])
def test_references_beside_tables_in_one_buffer(R, odd):
    """refs | table | kv_len | parents without a gap, refs ending inside a cache line; the pages that the copies
    take are among the last, some of them freed by the call itself.  Repeated on the same buffer."""
    r = rng(60, R, odd)
    P, blocks = 4, 3
    n_pages = 32 * 6 + odd
    for turn in range(6):
        refs, table = np.ones(n_pages, np.int32), np.full((R, blocks), -1, np.int32)
        kv = np.full(R, P + 2, np.int32)
        pages = n_pages - 1 - r.permutation(min(2 * R, n_pages))  # the last ones
        table[:, :2] = pages.reshape(R, 2)
        refs[table[:, :2]] = 1
        parents = np.zeros(R, np.int32)
        parents[R // 2:] = r.integers(0, R, R - R // 2)  # the others' pages become free
        want = M.reorder(refs, table, kv, parents, P)
        d = M.ints(np.concatenate([refs, table.ravel(), kv, parents]))
        at = [4 * n for n in np.cumsum([0, n_pages, R * blocks, R])]
        src, dst, status = (N.DeviceBuffer(4 * max(n, 1)) for n in (R, R, 3))
        w, n = M.ws("cdml_paged_reorder_workspace_size", R, blocks)
        ptr = [d.ptr + int(a) for a in at]
        N.check(N.lib().cdml_paged_reorder(ptr[0], n_pages, P, ptr[1], blocks, ptr[2], ptr[3], R, src.ptr, dst.ptr,
                                           status.ptr, w.ptr, n, stream().handle))
        got = down(d, (n_pages + R * (blocks + 2),), np.int32)
        same([got[:n_pages], got[n_pages:n_pages + R * blocks].reshape(R, blocks), got[-2 * R:-R], got[-R:]],
             [*want[:3], parents])
        same([down(x, (m,), np.int32) for x, m in ((src, R), (dst, R), (status, 3))], want[3:])


@pytest.mark.parametrize("rows", [40, 9000])
def test_an_open_page_that_is_none_has_no_slots(rows):
    # entries that pass 32 bits once shifted would else name slots of other requests
    P, n_pages = 16, 40
    refs, kv = np.zeros(n_pages, np.int32), np.array([5, 20, 3, 7], np.int32)
    table = np.full((4, 3), -1, np.int32)
    table[0, 0], table[1, :2], table[2, 0], table[3, 0] = 2 ** 28, [0, n_pages], 2 ** 28 + 7, -2 ** 28
    refs[0] = 1
    new = np.array([13, 2, 1, 1], np.int32)
    got = M.call_plan(refs, table, kv, new, P, rows)
    assert list(got[6]) == [0, 1, 17]
    slots = got[4]
    assert (slots[:11] == -1).all() and list(slots[11:13]) == [16, 17] and (slots[13:] == -1).all()
    assert list(got[5][:17]) == [*range(5, 18), 20, 21, 3, 7]
