"""The residual norm and the row quantiser over rows enough that every launch
shape runs its groups of rows, its ring and its reductions several times over.

Tolerances as in test_layer_ops_gpu.py: 2^-17 of a row's largest term for the
sums of a norm, u |h| and u |x'| for values stored in 16 bits.
"""

import pytest
import torch

import fastdialoguesidon_b200 as F
from oracle import layer_oracle as O
from test_layer_ops_gpu import U, V, _norm_case, _terms, _to

pytestmark = pytest.mark.gpu

# columns; the warps of a CTA follow from them: 1, 1, 2, 3, 5, 8, 16, and 10 and 9 of wider chunks
SHAPES = [(8, "none", "layer", "window", True), (256, "rms", "rms", "layer", False), (256, "layer", "layer", "none", True),
          (264, "layer", "layer", "window", True), (768, "none", "layer", "window", True), (1160, "rms", "rms", "layer", False),
          (2048, "layer", "rms", "window", True), (4096, "rms", "layer", "layer", False), (5000, "layer", "layer", "window", True),
          (9000, "rms", "rms", "window", False)]


def _rows(c):
    """Twenty rows a CTA and some (six where a CTA's ring holds two or four)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    chunks = 1 if c <= 4096 else (2 if c <= 8192 else 4)
    warps = -(-c // (256 * chunks))
    return (20 if chunks == 1 else 6) * sms * max(1, 16 // warps) + 13


@pytest.mark.parametrize("c,post,norm,gate,mod", SHAPES)
@pytest.mark.parametrize("dtype,stream,pdtype", [(torch.float16, torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16, torch.bfloat16),
                                                 (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float16, torch.float32)])
def test_residual_norm_many_groups_of_rows(cuda_device, c, post, norm, gate, mod, dtype, stream, pdtype):
    rows = _rows(c)
    windows = -(-rows // 37)  # windows of 37 rows: no multiple of a group
    case = _to(_norm_case(rows, c, dtype, stream, post, norm, gate, mod, windows, pdtype, seed=c))
    case["length"] = 37
    rx, rh = O.residual_norm(residual_scale=0.5, **case)
    big_x, big_h = _terms(case, rx, rh)
    x0, keep = case["x"].clone(), torch.empty_like(case["x"])
    x1, h = F.residual_norm(residual_scale=0.5, residual_out=keep, **case)
    assert torch.equal(case["x"], x0)
    ux = 0.0 if stream == torch.float32 else U[stream]
    assert bool(((x1.double() - rx).abs() <= ux * rx.abs() + 2.0 ** -17 * big_x).all())
    assert bool(((h.double() - rh).abs() <= U[dtype] * rh.abs() + 2.0 ** -17 * big_h + 2.0 ** -25).all())
    _, (q, s) = F.residual_norm(residual_scale=0.5, residual_out=keep, quantize=True, **case)
    s = s.double()[:, None]
    assert bool(((s - rh.abs().amax(1, keepdim=True) / 127).abs() <= 2.0 ** -17 * big_h / 127 + 4 * V * s).all())
    assert bool(((q.double() * s - rh).abs() <= s / 2 + 2.0 ** -17 * big_h * 2 + 4 * V * 127 * s).all())
    x2, h2 = F.residual_norm(residual_scale=0.5, **case)  # in place
    assert x2.data_ptr() == case["x"].data_ptr() and torch.equal(x2, x1) and torch.equal(h2, h)


@pytest.mark.parametrize("c", [8, 256, 768, 1160, 4096, 5000, 9000])
@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
def test_norm_without_a_block_many_groups_of_rows(cuda_device, c, stream):
    rows = _rows(c)
    case = _norm_case(rows, c, torch.bfloat16, stream, "none", "layer", "none", True, -(-rows // 37), torch.bfloat16, seed=c)
    case["length"], case["y"] = 37, None
    case = _to(case)
    _, rh = O.residual_norm(**case)
    _, big = _terms(case, case["x"].double(), rh)
    _, h = F.residual_norm(dtype=torch.bfloat16, **case)
    assert bool(((h.double() - rh).abs() <= U[torch.bfloat16] * rh.abs() + 2.0 ** -17 * big).all())
    _, (q, s) = F.residual_norm(dtype=torch.bfloat16, quantize=True, **case)
    s = s.double()[:, None]
    assert bool(((q.double() * s - rh).abs() <= s / 2 + 2.0 ** -17 * big * 2 + 4 * V * 127 * s).all())


@pytest.mark.parametrize("off_x,off_out", [(0, 0), (4, 0), (0, 4), (4, 4)])
@pytest.mark.parametrize("rows", [1, 50, 4000])
def test_residual_norm_stream_alignments(cuda_device, off_x, off_out, rows):
    """fp32 rows on 16- or 32-byte boundaries, on either side: the same bits, and what lies beside them stays."""
    g = torch.Generator().manual_seed(rows)
    x, y = torch.randn(rows, 512, generator=g).cuda(), torch.randn(rows, 512, generator=g).half().cuda()
    want, h = F.residual_norm(x, y, residual_out=torch.empty_like(x))
    wide, keep = torch.randn(rows, 520, device="cuda"), torch.zeros(rows, 520, device="cuda")
    wide[:, off_x:off_x + 512] = x
    x1, h1 = F.residual_norm(wide[:, off_x:off_x + 512], y, residual_out=keep[:, off_out:off_out + 512])
    assert torch.equal(x1, want) and torch.equal(h1, h)
    keep[:, off_out:off_out + 512] = 0
    assert float(keep.abs().max()) == 0.0


@pytest.mark.parametrize("c", [248, 264, 512, 520, 776, 1032, 1544, 2056, 3000, 4088, 8192, 8200])
@pytest.mark.parametrize("rows", [1, 7, 1001])
def test_quantize_rows_widths(cuda_device, c, rows):
    """Every number of chunks a lane holds, whole and ragged; odd rows, strided ones; values as defined."""
    g = torch.Generator().manual_seed(c + rows)
    x = (torch.randn(rows, c + 8, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).half().cuda()[:, 8:]
    out = torch.full((rows, c + 16), 99, dtype=torch.int8, device="cuda")
    q, s = F.quantize_rows(x, out=out[:, 8:c + 8])
    qr, sr = O.quantize_rows(x.cpu())  # (on a GPU torch divides by a number as a product with its reciprocal: not one rounding)
    assert torch.equal(q.cpu(), qr) and torch.equal(s.cpu(), sr)
    assert bool((out[:, :8] == 99).all()) and bool((out[:, c + 8:] == 99).all())
