"""Window attention where one wrong key shows: NaN and infinities in keys that
are seen.

Tolerance: that of test_layer_ops_gpu.py, (2 u + 2e-4) max|v| with u the unit
roundoff of the operand type.
"""

import pytest
import torch

import fastdialoguesidon_b200 as F
from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])


def _qkv(B, Lq, Lk, H, Hk, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(B, n, h, 64, generator=g).to(dtype).cuda() for n, h in ((Lq, H), (Lk, Hk), (Lk, Hk)))


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _check(q, k, v, left, right, sinks, q_start=None, kv_len=None, **kw):
    ref = O.window_attention_by_head(q, k, v, left, right, sinks, q_start, kv_len, **kw)
    got = F.window_attention(q, k, v, left, right, sinks, q_start=q_start, kv_len=kv_len, **kw)
    F.check_status()
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), bad), (int(torch.isnan(got).sum()), int(bad.sum()))
    err = float((got.double() - ref).masked_fill(bad, 0).abs().max())
    assert err <= (2 * U[q.dtype] + 2e-4) * float(v.float().abs().max()), err
    return got


# one query, several queries of a step, whole units, a unit split over a cluster
FORMS = [(1, 400, 60), (5, 400, 60), (150, 400, 60), (40, 2500, 2000)]


@BOTH
@pytest.mark.parametrize("Lq,Lk,left", FORMS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_window_keys_that_are_not_finite(cuda_device, dtype, Lq, Lk, left, value):
    """A key that a query sees counts as it stands: a NaN score, or one of plus
    infinity, makes the query's output NaN, minus infinity weighs nothing. Over 24
    places of the key, so that it meets every way the exponentials are computed."""
    q, k, v = _qkv(1, Lq, Lk, 2, 2, dtype, seed=Lq)
    q = q.abs()  # the score of an infinite key is infinite
    for at in range(24):
        kb = k.clone()
        kb[0, Lk - 40 + at - (Lq > 40) * 60, 0] = value
        _check(q, kb, v, left, 0, 4, _i32([Lk - Lq]))


@BOTH
@pytest.mark.parametrize("Lq,Lk,left", FORMS)
def test_window_queries_that_are_nan(cuda_device, dtype, Lq, Lk, left):
    """All scores of the query are NaN: its output is, and no other one."""
    q, k, v = _qkv(1, Lq, Lk, 4, 2, dtype, seed=Lq)
    q[0, Lq // 2, 1, 7] = float("nan")
    got = _check(q, k, v, left, 0, 4, _i32([Lk - Lq]))
    assert int(torch.isnan(got).sum()) == 64
    q[0, Lq // 2, 1, 7] = 0.0
    _check(q, k, v, left, 0, 4, _i32([Lk - Lq]))
