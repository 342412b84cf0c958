"""Refusals of the layer ops without a GPU (the C ABI's checks before any
launch, the Python layer's checks before any pointer is used), the struct
mirrors, and the oracle's own identities."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

import fastdialoguesidon_b200 as F
from fastdialoguesidon_b200 import _native as N
from oracle import flexrel_oracle
from oracle import layer_oracle as O

HEADER = Path(__file__).resolve().parents[1] / "include" / "fds_b200.h"


def test_struct_layouts_match_header():
    text = HEADER.read_text()
    for struct, cls in (("FdsLinearInt8Args", N.FdsLinearInt8Args), ("FdsResidualNormArgs", N.FdsResidualNormArgs),
                        ("FdsWindowArgs", N.FdsWindowArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
        fields = re.findall(r"^\s*[\w\s\*]+?\b(\w+)(?:\[3\])?;", body, re.M)
        assert fields == [f[0] for f in cls._fields_], (struct, fields)


def _refused(rc):
    assert rc == N.FDS_ERR_INVALID_ARGUMENT
    assert N.last_error()


def _window(**kw):
    st = (ctypes.c_int64 * 3)(64000, 128, 64)
    base = dict(q=16, k=16, v=16, out=16, q_stride=st, k_stride=st, v_stride=st, out_stride=st, batch=2, heads=2, kv_heads=2,
                q_len=100, k_len=100, head_dim=64, dtype=N.FDS_DTYPE_FP16, left=8, right=0, sinks=0, scale=0.125)
    base.update(kw)
    return N.FdsWindowArgs(**base)


def _strides(*v):
    return (ctypes.c_int64 * 3)(*v)


@pytest.mark.parametrize("bad", [
    dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(q=18), dict(v=24), dict(head_dim=128), dict(dtype=2), dict(batch=0), dict(heads=3),
    dict(kv_heads=0), dict(q_len=-1), dict(k_len=0), dict(k_len=1 << 29), dict(left=-1), dict(right=-1), dict(sinks=-1),
    dict(scale=0.0), dict(scale=float("nan")), dict(q_stride=_strides(64000, 128, 60)), dict(k_stride=_strides(64000, 0, 64)),
    dict(v_stride=_strides(64001, 128, 64)), dict(out_stride=_strides(64000, -128, 64))])
def test_window_c_abi_refuses(bad):
    _refused(N.load().fds_window_attn_fwd(ctypes.byref(_window(**bad)), None))


def _int8(**kw):
    base = dict(a=16, a_row_stride=128, a_scale=16, w=16, w_row_stride=128, w_scale=16, bias=None, out=16, out_row_stride=128,
                m=4, n=128, k=128, dtype=N.FDS_DTYPE_FP16, epilogue=N.FDS_EPILOGUE_STORE)
    base.update(kw)
    return N.FdsLinearInt8Args(**base)


@pytest.mark.parametrize("bad", [
    dict(a=0), dict(w=0), dict(out=0), dict(a_scale=0), dict(w_scale=0), dict(a=24), dict(w_scale=20), dict(a_scale=18), dict(bias=8),
    dict(dtype=3), dict(epilogue=3), dict(m=-1), dict(n=0), dict(n=12), dict(k=24), dict(k=0), dict(k=65552, a_row_stride=65552, w_row_stride=65552),
    dict(a_row_stride=120), dict(a_row_stride=136), dict(w_row_stride=64), dict(out_row_stride=64), dict(out_row_stride=132),
    dict(epilogue=N.FDS_EPILOGUE_ROPE), dict(tile_n=96), dict(cta_pair=3), dict(cta_pair=N.FDS_GEMM_PAIR, tile_n=64),
    dict(epilogue=N.FDS_EPILOGUE_ROPE, cos=16, sin=16, seq_len=0), dict(epilogue=N.FDS_EPILOGUE_ROPE, cos=16, sin=16, seq_len=4, rope_cols=96)])
def test_int8_c_abi_refuses(bad):
    _refused(N.load().fds_linear_int8_fwd(ctypes.byref(_int8(**bad)), None))


def _norm(**kw):
    base = dict(x=16, x_stride=64, y=16, y_stride=64, x_out=16, x_out_stride=64, h=16, h_stride=64, rows=4, c=64, length=4,
                dtype=N.FDS_DTYPE_FP16, x_f32=1, post=0, norm=1, alpha=1.0, eps=1e-5)
    base.update(kw)
    return N.FdsResidualNormArgs(**base)


@pytest.mark.parametrize("bad", [
    dict(x=0), dict(x_out=0), dict(x=20), dict(y=18), dict(h=4), dict(dtype=5), dict(rows=-1), dict(length=0), dict(c=0), dict(c=20),
    dict(c=16392, x_stride=16392, y_stride=16392, x_out_stride=16392, h_stride=16392), dict(post=3), dict(norm=-1), dict(eps=-1.0),
    dict(eps=float("nan")), dict(x_stride=60), dict(x_stride=66), dict(y_stride=32), dict(h_stride=68), dict(gate=4), dict(w=8),
    dict(gate_stride=-64), dict(mod_stride=12), dict(y=None, gate=16), dict(y=None, post=1), dict(h=None, h_scale=16),
    dict(y=None, x_out=None, h=None)])
def test_norm_c_abi_refuses(bad):
    _refused(N.load().fds_residual_norm_fwd(ctypes.byref(_norm(**bad)), None))


def test_empty_calls_are_no_ops():
    lib = N.load()
    assert lib.fds_window_attn_fwd(ctypes.byref(_window(q_len=0)), None) == N.FDS_OK
    assert lib.fds_linear_int8_fwd(ctypes.byref(_int8(m=0)), None) == N.FDS_OK
    assert lib.fds_residual_norm_fwd(ctypes.byref(_norm(rows=0)), None) == N.FDS_OK
    for fn in (lib.fds_window_attn_fwd, lib.fds_linear_int8_fwd, lib.fds_residual_norm_fwd):
        _refused(fn(None, None))


def test_no_cpu_fallback():
    h = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    i8, f32 = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: F.window_attention(h, h, h, 4), lambda: F.quantize_rows(h.view(-1, 64)),
                 lambda: F.linear_int8(i8, f32, torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8)),
                 lambda: F.accumulate_int8(torch.zeros(4, 8), i8, f32, torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8)),
                 lambda: F.residual_norm(torch.zeros(4, 64))):
        with pytest.raises(F.FdsError, match="CUDA"):
            call()


def test_python_refuses_types():
    with pytest.raises(F.FdsError, match="torch.Tensor"):
        F.window_attention([1], None, None, 4)
    with pytest.raises(F.FdsError, match="float16"):
        F.window_attention(torch.zeros(1, 4, 2, 64), None, None, 4)
    with pytest.raises(F.FdsError, match="int8"):
        F.linear_int8(torch.zeros(4, 64), None, None, None)


def test_oracle_window_is_full_attention_when_wide():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 40, 3, 64, generator=g) for _ in range(3))
    a = O.window_attention(q, k, v, 40, 40)
    s = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double()) / 8, -1)
    assert float((a - torch.einsum("bhqk,bkhd->bqhd", s, v.double())).abs().max()) < 1e-12


def test_oracle_rope_matches_the_models():
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(30, 3 * 2 * 64, generator=g)
    cos, sin = F.rope_tables(10)
    want = flexrel_oracle.rope_split(qkv, 10, 2, cos, sin)
    got = O.rope(qkv.double(), cos, sin, 10, 256)
    assert float((torch.cat([want[0], want[1]], -1).reshape(30, -1).double() - got[:, :256]).abs().max()) < 1e-5
