"""Window attention where one wrong key shows: NaN and infinities in keys that
are seen, keys that outweigh all others at every edge and seam, and launches of
more units than run at once.

Tolerance: that of test_layer_ops_gpu.py, (2 u + 2e-4) max|v| with u the unit
roundoff of the operand type. A planted key scores 16 above the others' mean
(they deviate by 1), so it weighs 0.99 of 5000 keys, and to see it wrongly, or not
to see it, is an error of the size of a value. (Without one, a key of 3000 that is
left out changes bf16 outputs by 0.002 to 0.015, where the tolerance is 0.036.)
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


# ---------------------------------------------------------------- one key that outweighs all others


def _planted(B, Lq, Lk, H, Hk, dtype, seed, places):
    """Random q, k, v; in every window and key head one key of `places` (taken in
    turn) scores 16 against every query, the others by their random parts."""
    q, k, v = _qkv(B, Lq, Lk, H, Hk, dtype, seed)
    q[..., 0], k[..., 0] = 8.0, 0.0
    for i in range(B * Hk):
        k[i // Hk, places[i % len(places)], i % Hk, 0] = 16.0
    return q, k, v


@BOTH
@pytest.mark.parametrize("Lq,H,Hk,left,sinks", [(9, 32, 32, 3000, 4), (40, 32, 32, 2000, 0), (128, 16, 16, 3700, 16),
                                                (130, 16, 16, 1500, 200), (42, 24, 8, 2500, 7)])
def test_window_planted_keys_in_a_split_unit(cuda_device, dtype, Lq, H, Hk, left, sinks):
    """A unit's tiles dealt to a cluster: a planted key on either side of every
    multiple of 128 columns, at the window's first and last keys and at the ends of
    the sinks. The rows before and after the place see it at an edge of their own."""
    Lk = 4133
    start = Lk - Lq
    begin = max(0, start - left)
    tiles = range(begin, Lk, 128)
    places = [j for t in tiles for j in (t - 1, t, t + 1)] + [Lk - 1, Lk - 2, start, start + 1]
    places += [0, max(0, sinks - 1), sinks, sinks + 1]
    places = sorted({min(max(j, 0), Lk - 1) for j in places})
    for i in range(0, len(places), Hk):
        _check(*_planted(1, Lq, Lk, H, Hk, dtype, i, places[i:i + Hk]), left, 0, sinks, _i32([start]))


@BOTH
@pytest.mark.parametrize("Lq,H,Hk", [(1, 32, 32), (1, 32, 8), (3, 32, 8), (16, 8, 8)])
@pytest.mark.parametrize("left,sinks", [(4099, 0), (1000, 5), (2047, 37)])
def test_window_planted_keys_in_a_step(cuda_device, dtype, Lq, H, Hk, left, sinks):
    """Steps read blocks of 32 keys, the sinks first: a planted key on either side
    of every block's end, at the window's edges and the ends of the sinks."""
    Lk = 4100
    start = Lk - Lq
    begin = max(0, start - left)
    places = [begin, begin + 1, Lk - 1, Lk - 2, 0, max(0, sinks - 1), sinks]
    places += [begin - min(sinks, begin) + t + d for t in range(32, Lk - begin, 32) for d in (-1, 0)]
    places = sorted({min(max(j, 0), Lk - 1) for j in places})
    B = -(-len(places) // (4 * Hk))  # (a launch takes a quarter of the places)
    for i in range(0, len(places), B * Hk):
        q, k, v = _planted(B, Lq, Lk, H, Hk, dtype, i, places[i:i + B * Hk])
        _check(q, k, v, left, 0, sinks, _i32([start] * B))


@BOTH
@pytest.mark.parametrize("left,right,sinks", [(130, 0, 0), (200, 77, 5), (64, 300, 129)])
def test_window_planted_keys_in_whole_units(cuda_device, dtype, left, right, sinks):
    """A planted key at every 13th place of a self-attention: for each, the rows that see it at either edge."""
    L, H = 600, 12
    places = list(range(0, L, 13)) + [sinks, max(0, sinks - 1), L - 1]
    _check(*_planted(4, L, L, H, H, dtype, 1, places), left, right, sinks)


# ---------------------------------------------------------------- more units than run at once


@BOTH
@pytest.mark.parametrize("H,Hk,left,right,sinks", [(12, 12, 150, 40, 6), (12, 4, 150, 40, 6), (12, 4, 700, 0, 130), (16, 4, 300, 0, 0),
                                                   (10, 2, 20, 20, 9)])
def test_window_units_handed_on(cuda_device, dtype, H, Hk, left, right, sinks):
    """At least 1.3 times the units that two CTAs per SM hold, so CTAs take over the
    units of others: some see nothing, some one tile, some several, in turn. Groups
    of 1, 3, 4 and 5 heads (units of 126 and 125 rows too). The second of two
    calls has the same bits."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    Lq, Lk = 700, 1400
    units = Hk * -(-Lq // (128 // (H // Hk)))
    B = -(-26 * sms // (10 * units)) + 1
    assert B * units >= 2.6 * sms
    # positions and lengths: ahead of all keys, past kv_len, an empty window, a few keys, all of them
    start = [(0, -2000, 350, 1300, 700, 20, 1390)[b % 7] for b in range(B)]
    kv = [(1400, 1400, 0, 600, 900, 33, 1400, 1, 710)[b % 9] for b in range(B)]
    q, k, v = _planted(B, Lq, Lk, H, Hk, dtype, H + left, [0, 5, 127, 349, 500, 699, 700, 899, 1000, 1399])
    got = _check(q, k, v, left, right, sinks, _i32(start), _i32(kv))
    for _ in range(3):
        assert torch.equal(got, F.window_attention(q, k, v, left, right, sinks, q_start=_i32(start), kv_len=_i32(kv)))


# ---------------------------------------------------------------- forms of a step


@BOTH
@pytest.mark.parametrize("Lq,H,Hk", [(3, 8, 2), (7, 4, 2), (16, 2, 2), (9, 3, 3), (4, 16, 4), (2, 5, 1), (1, 32, 2)])
@pytest.mark.parametrize("left,right,sinks", [(2000, 0, 4), (700, 5, 33)])
def test_window_steps_over_a_cluster(cuda_device, dtype, Lq, H, Hk, left, right, sinks):
    """Several queries and 2 to 16 rows a key head over keys dealt to up to 8 CTAs; kv_len within the last query's window."""
    Lk = 2600
    q, k, v = _qkv(2, Lq, Lk, H, Hk, dtype, seed=Lq + H)
    _check(q, k, v, left, right, sinks, _i32([Lk - Lq, 2100]), _i32([Lk - 1, 2100 + Lq]))


@BOTH
@pytest.mark.parametrize("Lq,Lk,left", FORMS)
@pytest.mark.parametrize("scale", [0.02, 0.125, 0.5])
def test_window_scale(cuda_device, dtype, Lq, Lk, left, scale):
    q, k, v = _qkv(1, Lq, Lk, 2, 2, dtype, seed=3)
    _check(q, k, v, left, 0, 4, _i32([Lk - Lq]), scale=scale)
