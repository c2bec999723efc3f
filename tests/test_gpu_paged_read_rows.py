"""cdml_paged_read of as many rows as one axis of a launch has no room for: a workgroup a row from 2^24 rows on."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_model as M
import paged_q8_model as Q
from abi_ops import stream
from cdml import native as N
from test_gpu_paged import rng

pytestmark = pytest.mark.gpu


def test_read_of_more_rows_than_a_launch_axis_holds():
    heads, hd, P = 5, 205, 64
    dim, rows = heads * hd, 2 ** 24 + 5
    stream()
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("137 GB of outputs do not fit")
    r = rng(37)
    c = Q.random_cache(r, "f32", 4, P, heads, hd)
    table, kv = np.array([[2, 0], [1, 1], [3, 2]], np.int32), np.array([100, 0, 70], np.int32)
    # five rows and two of no request; a request's last tokens (100, none and the last 12 of 70), zeros before them
    cu = np.array([5, 2 ** 23 + 7, 2 ** 24 - 9, rows - 2], np.int32)
    out = [torch.empty((rows, dim), device="cuda") for _ in range(2)]
    for x in out:
        x[:5], x[-2:] = 7.0, 7.0
    torch.cuda.synchronize()
    d, t, l, u, bad = Q.upload(c), M.ints(table), M.ints(kv), M.ints(cu), M.ints(np.zeros(1))
    N.check(N.lib().cdml_paged_read(*(Q.ptr(b) for b in d), N.CACHE["f32"], 4, P, t.ptr, 2, l.ptr, u.ptr,
                                    out[0].data_ptr(), dim, out[1].data_ptr(), dim, rows, 3, heads, hd, bad.ptr,
                                    stream().handle))
    stream().synchronize()
    for x, side in zip(out, "kv"):
        assert (x[:5] == 7).all() and (x[-2:] == 7).all()
        for b in range(3):
            first, end = int(cu[b]), int(cu[b + 1])
            n = min(int(kv[b]), end - first)
            at = np.arange(kv[b] - n, kv[b])
            want = torch.from_numpy(c[side + "x"][table[b, at // P], at % P].astype(np.float32)).cuda()
            assert torch.equal(x[end - n:end], want)
            for i in range(first, end - n, 2 ** 20):
                assert not x[i:min(i + 2 ** 20, end - n)].any()
    del out, x
    torch.cuda.empty_cache()
