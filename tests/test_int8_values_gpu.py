"""The 8-bit projections' results do not depend on which kernel or tiling computes them."""

import pytest
import torch

import fastdialoguesidon_b200 as F
from test_layer_ops_gpu import _cuda, _int8_operands

pytestmark = pytest.mark.gpu

TILINGS = [(False, 64), (False, 128), (False, 256), (True, 128), (True, 256)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,heads,length", [(1, 768, 12, 6000), (3, 144, 2, 2), (8, 1040, 3, 5), (300, 256, 4, 117)])
def test_int8_rope_tilings_agree_bit_for_bit(cuda_device, m, k, heads, length, dtype):
    """The kernel for up to eight rows and the tensor-core tilings round a rotation alike."""
    n = 192 * heads
    x, xs, w, ws, b = _cuda(*_int8_operands(m, k, n, dtype, bias=True, seed=m + k))
    cos, sin = F.rope_tables(length, "cuda")
    for bias in (b, None):
        args = (x, xs, w, ws, bias, cos, sin, length, heads)
        want = F.linear_int8_rope(*args, dtype=dtype)
        for pair, tile_n in TILINGS:
            assert torch.equal(F.linear_int8_rope(*args, dtype=dtype, pair=pair, tile_n=tile_n), want), (pair, tile_n)
    F.check_status()


@pytest.mark.parametrize("m,k,n", [(1, 768, 264), (5, 2064, 520), (8, 144, 1032), (300, 400, 776)])
def test_int8_accumulate_tilings_agree_bit_for_bit(cuda_device, m, k, n):
    x, xs, w, ws, b = _cuda(*_int8_operands(m, k, n, torch.float16, bias=True, seed=m + k))
    r = torch.randn(m, n, generator=torch.Generator().manual_seed(m)).cuda()
    for bias in (b, None):
        want = r.clone()
        F.accumulate_int8(want, x, xs, w, ws, bias)
        for pair, tile_n in TILINGS:
            got = r.clone()
            F.accumulate_int8(got, x, xs, w, ws, bias, pair=pair, tile_n=tile_n)
            assert torch.equal(got, want), (pair, tile_n)
    F.check_status()
