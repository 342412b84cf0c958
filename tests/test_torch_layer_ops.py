"""The layer ops as torch operators: every argument of the functions, shapes and
types without a GPU, and a layer traced whole."""

import pytest
import torch

import fastdialoguesidon_b200 as F

ops = torch.ops.fds
H, HIDDEN = 2, 128


def _empty(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_shapes_and_types_without_a_gpu():
    q, cache = _empty(2, 5, 4, 64), _empty(2, 90, 2, 64)
    assert ops.window_attention(q, cache, cache, 30, scale=0.1).shape == q.shape
    assert ops.window_attention(q, cache, cache, 30, 0, 2, scale=0.1, out=q) is q
    x, xs = ops.quantize_rows(_empty(7, HIDDEN))
    assert (x.dtype, x.shape, xs.dtype, xs.shape) == (torch.int8, (7, HIDDEN), torch.float32, (7,))
    w, ws, b = _empty(192 * H, HIDDEN, dtype=torch.int8), _empty(192 * H, dtype=torch.float32), _empty(192 * H, dtype=torch.bfloat16)
    table = _empty(7, 64, dtype=torch.float32)
    for bias, dtype, want in ((None, None, torch.float16), (b, None, torch.bfloat16), (None, torch.bfloat16, torch.bfloat16)):
        for y in (ops.linear_int8(x, xs, w, ws, bias, dtype=dtype), ops.linear_int8_rope(x, xs, w, ws, bias, table, table, 7, H, dtype=dtype)):
            assert (y.dtype, y.shape) == (want, (7, 192 * H))
    assert ops.accumulate_int8(_empty(7, 192 * H, dtype=torch.float32), x, xs, w, ws, b) is None
    r = _empty(7, HIDDEN, dtype=torch.float32)
    assert ops.residual_norm_(r, _empty(7, HIDDEN, dtype=torch.bfloat16), gate=b).dtype == torch.bfloat16
    assert ops.residual_norm_(r).dtype == torch.float16 and ops.residual_norm_(r, dtype=torch.bfloat16).dtype == torch.bfloat16
    assert ops.residual_norm_int8_(r, norm="rms")[0].dtype == torch.int8


def _operands(device, rows=130):
    g = torch.Generator().manual_seed(0)

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).half().to(device)

    def weight(n, k):
        return torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).to(device), (torch.rand(n, generator=g) * 1e-3).to(device)

    return dict(x=rnd(rows, HIDDEN).float(), qkv=weight(192 * H, HIDDEN), out=weight(HIDDEN, HIDDEN), b=rnd(192 * H), gate=rnd(HIDDEN),
                scale=rnd(HIDDEN, scale=0.1), shift=rnd(HIDDEN), tables=F.rope_tables(rows, device))


def _layer(x, o):
    n = x.shape[0]
    h, hs = ops.residual_norm_int8_(x, scale=o["scale"], shift=o["shift"], dtype=torch.float16)
    q, k, v = ops.linear_int8_rope(h, hs, *o["qkv"], o["b"], *o["tables"], n, H).view(1, n, 3, H, 64).unbind(2)
    c, cs = ops.quantize_rows(ops.window_attention(q, k, v, 40, 9, 3, scale=0.1).view(n, HIDDEN))
    ops.accumulate_int8(x, c, cs, *o["out"])
    return ops.residual_norm_(x, ops.linear_int8(c, cs, *o["out"]), gate=o["gate"], norm="rms")


def _layer_functions(x, o):
    n = x.shape[0]
    _, (h, hs) = F.residual_norm(x, scale=o["scale"], shift=o["shift"], quantize=True, dtype=torch.float16)
    q, k, v = F.linear_int8_rope(h, hs, *o["qkv"], o["b"], *o["tables"], n, H).view(1, n, 3, H, 64).unbind(2)
    c, cs = F.quantize_rows(F.window_attention(q, k, v, 40, 9, 3, scale=0.1).view(n, HIDDEN))
    F.accumulate_int8(x, c, cs, *o["out"])
    return F.residual_norm(x, F.linear_int8(c, cs, *o["out"]), gate=o["gate"], norm="rms")[1]


@pytest.mark.gpu
def test_a_layer_of_operators_is_the_functions_and_can_be_traced(cuda_device):
    o = _operands("cuda")
    want_x, got_x, traced_x = (o["x"].clone() for _ in range(3))
    want, got = _layer_functions(want_x, o), _layer(got_x, o)
    traced = torch.compile(_layer, backend="aot_eager", fullgraph=True)(traced_x, o)
    F.check_status()
    assert torch.equal(got, want) and torch.equal(got_x, want_x)
    assert torch.equal(traced, want) and torch.equal(traced_x, want_x)


@pytest.mark.gpu
def test_operators_declare_what_they_do(cuda_device):
    """Aliasing, mutation, and the shapes and types of the traced form, against a call."""
    o = _operands("cuda", rows=20)
    x16 = o["x"].half()
    x8, xs = F.quantize_rows(x16)
    q = torch.randn(1, 20, H, 64, device="cuda").half()
    f16 = torch.empty(20, 192 * H, dtype=torch.float16, device="cuda")
    calls = [
        (ops.window_attention.default, (q, q, q, 5, 1, 2), dict(scale=0.1)), (ops.window_attention.out, (q, q, q, 5), dict(out=q.clone())),
        (ops.quantize_rows.default, (x16,), {}), (ops.quantize_rows.out, (x16,), dict(out=x8.clone(), scale=xs.clone())),
        (ops.linear_int8.default, (x8, xs, *o["qkv"]), dict(dtype=torch.bfloat16)), (ops.linear_int8.out, (x8, xs, *o["qkv"], o["b"]), dict(out=f16)),
        (ops.linear_int8_rope.default, (x8, xs, *o["qkv"], o["b"], *o["tables"], 20, H), {}),
        (ops.linear_int8_rope.out, (x8, xs, *o["qkv"], None, *o["tables"], 20, H), dict(out=f16)),
        (ops.accumulate_int8.default, (o["x"].clone(), x8, xs, *o["out"]), {}),
        (ops.residual_norm_.default, (o["x"].clone(), x16), dict(gate=o["gate"], residual_scale=0.5, post="rms")),
        (ops.residual_norm_int8_.default, (x16.clone(),), dict(norm="rms"))]
    for op, args, kw in calls:
        torch.library.opcheck(op, args, kw, test_utils=("test_schema", "test_faketensor"))
    F.check_status()
