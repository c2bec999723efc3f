"""cdml_paged_read of as many rows as one axis of a launch has no room for: a workgroup a row from 2^24 rows on."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_model as M
import paged_q8_model as Q
from abi_ops import down, stream
from cdml import native as N
from test_gpu_paged import rng

pytestmark = pytest.mark.gpu

SEVEN = int(np.float32(7).view(np.int32))


def test_read_of_more_rows_than_a_launch_axis_holds():
    heads, hd, P = 5, 205, 64
    dim, rows = heads * hd, 2 ** 24 + 5
    st, L = stream(), N.lib()
    if N.device_info()["total_memory"] < 160 << 30:
        pytest.skip("137 GB of outputs do not fit")
    r = rng(37)
    c = Q.random_cache(r, "f32", 4, P, heads, hd)
    table, kv = np.array([[2, 0], [1, 1], [3, 2]], np.int32), np.array([100, 0, 70], np.int32)
    # five rows and two of no request; a request's last tokens (100, none and the last 12 of 70), zeros before them
    cu = np.array([5, 2 ** 23 + 7, 2 ** 24 - 9, rows - 2], np.int32)
    out = [N.DeviceBuffer(4 * rows * dim) for _ in range(2)]
    for x in out:
        N.check(L.cdml_fill_i32_async(x.ptr, rows * dim, SEVEN, st.handle))
    d, t, l, u, bad = Q.upload(c), M.ints(table), M.ints(kv), M.ints(cu), M.ints(np.zeros(1))
    N.check(L.cdml_paged_read(*(Q.ptr(b) for b in d), N.CACHE["f32"], 4, P, t.ptr, 2, l.ptr, u.ptr, out[0].ptr, dim,
                              out[1].ptr, dim, rows, 3, heads, hd, bad.ptr, st.handle))
    size = C.c_size_t(0)
    N.check(L.cdml_sum_squares_workspace_size(C.byref(size)))
    work, total = N.DeviceBuffer(size.value), N.DeviceBuffer(4)
    for x, side in zip(out, "kv"):

        def rows_of(first, end):
            y = np.empty((end - first, dim), np.float32)
            N.check(L.cdml_memcpy_d2h_async(y.ctypes.data, x.ptr + 4 * dim * first, y.nbytes, st.handle))
            st.synchronize()
            return y
        assert (rows_of(0, 5) == 7).all() and (rows_of(rows - 2, rows) == 7).all()
        for b in range(3):
            first, end = int(cu[b]), int(cu[b + 1])
            n = min(int(kv[b]), end - first)
            at = np.arange(kv[b] - n, kv[b])
            if n:
                want = c[side + "x"][table[b, at // P], at % P].astype(np.float32)
                np.testing.assert_array_equal(rows_of(end - n, end), want)
            N.check(L.cdml_sum_squares(x.ptr + 4 * dim * first, (end - n - first) * dim, total.ptr, work.ptr, size.value,
                                       st.handle))
            assert down(total, (1,))[0] == 0
    assert down(bad, (1,), np.int32)[0] == 0
    for x in out:
        x.free()
