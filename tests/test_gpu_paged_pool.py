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
