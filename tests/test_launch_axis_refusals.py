"""Sizes that take more workgroups than an axis of a launch holds (2^32 threads) are refused, before a device is touched:
such a launch runs short without an error (cdml_cross_entropy of 2^24 + 3 rows left its gradients unwritten)."""
from __future__ import annotations

import pytest

from cdml import native as N
from test_paged_refusals import P, refused

WS = 1 << 60  # bytes of workspace, never touched


def bwd(batch, lq, dim, heads):
    return dict(q=P, ldq=dim, k=P, ldk=dim, v=P, ldv=dim, do=P, lddo=dim, dq=P, lddq=dim, dk=P, lddk=dim, dv=P, lddv=dim,
                batch=batch, lq=lq, lk=lq, dim=dim, heads=heads, scale=1.0, causal=0, mask=None, ws=P, bytes=WS, stream=None)


def fwd(batch, lq, dim, heads):
    return dict(q=P, ldq=dim, k=P, ldk=dim, v=P, ldv=dim, o=P, ldo=dim, batch=batch, lq=lq, lk=lq, dim=dim, heads=heads,
                scale=1.0, causal=0, mask=None, stream=None)


def ln_bwd(rows, features):
    return dict(dout=P, dout2=None, norm=P, gamma=P, x=P, mean=P, var=P, dx=P, dgamma=P, dbeta=P, rows=rows,
                features=features, eps=1e-5, accumulate=0, ws=P, bytes=WS, stream=None)


# entry, arguments of the largest launch, the changes that are one workgroup more
CASES = [
    ("cdml_argmax_rows", dict(x=P, rows=2 ** 26 - 4, cols=2, ld=2, out=P, stride=1, stream=None),
     [{"rows": 2 ** 26 - 3}, {"rows": 2 ** 31 - 1}]),
    ("cdml_embed_tokens", dict(ids=P, count=2 ** 26 - 1, table=P, vocab=9, dim=4, out=P, bad=None, stream=None),
     [{"count": 2 ** 26}, {"count": 2 ** 31 - 1}]),
    ("cdml_kv_cache_append", dict(k=P, v=P, kc=P, vc=P, pos=P, batch=2 ** 24 - 1, t_max=3, dim=4, stream=None),
     [{"batch": 2 ** 24}]),
    ("cdml_residual_layernorm", dict(a=P, b=P, gamma=P, beta=P, y=P, rows=2 ** 26 - 4, features=8, eps=1e-5, stream=None),
     [{"rows": 2 ** 26 - 3}, {"rows": 2 ** 31 - 1}]),
    ("cdml_residual_layernorm_fwd", dict(a=P, b=P, gamma=P, beta=P, out=P, mean=None, var=None, res=None, norm=None,
                                         rows=2 ** 26 - 4, features=8, eps=1e-5, stream=None),
     [{"rows": 2 ** 26 - 3}, {"rows": 2 ** 31 - 1}]),
    ("cdml_layernorm_backward", ln_bwd(2 ** 28 - 64, 8), [{"rows": 2 ** 28 - 63}, {"rows": 2 ** 31 - 1}]),
    ("cdml_cross_entropy", dict(x=P, ldl=2, targets=P, rows=2 ** 24 - 1, dim=2, eff=5, gs=1.0, ls=1.0, loss=P, dx=P, lddl=2,
                                ws=P, bytes=WS, stream=None), [{"rows": 2 ** 24}]),
    ("cdml_sdpa_fwd", fwd(2 ** 22 - 1, 5, 32, 4), [{"batch": 2 ** 22}, {"batch": 2 ** 21, "lq": 129, "lk": 129},
                                                 {"batch": 2 ** 31 - 1, "lq": 2 ** 31 - 1, "heads": 32}]),
    ("cdml_sdpa_fwd", fwd(2 ** 23 - 1, 2, 200, 1), [{"batch": 2 ** 23}, {"batch": 2 ** 20, "lq": 16}]),
    ("cdml_sdpa_bwd", bwd(2 ** 22 - 1, 5, 32, 4), [{"batch": 2 ** 22}, {"batch": 2 ** 21, "lq": 129},
                                                 {"batch": 2 ** 31 - 1, "lq": 2 ** 31 - 1, "heads": 32}]),
    ("cdml_sdpa_bwd", bwd(2 ** 21 - 1, 5, 160, 4), [{"batch": 2 ** 21}]),
]


@pytest.mark.parametrize("name,good,changes", CASES)
def test_more_workgroups_than_a_launch_holds(name, good, changes):
    refused(name, good, changes)


@pytest.mark.parametrize("name,good,changes", CASES)
def test_the_largest_launch_is_allowed(name, good, changes):
    if N.device_count() > 0:
        pytest.skip("a device is visible: the call would run")
    assert getattr(N.lib(), name)(*good.values()) == N.E_NODEVICE, N.lib().cdml_last_error()
