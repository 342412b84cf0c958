"""``torch.ops.fds.*`` registrations of the hot-path ops (CUDA only).

Schemas (the reference op ``flexrel_attention(qkv, batch, heads, rel,
out=None)``, triton/src/fds_triton/kernels.py:422, as an operator with an
out= overload, the way ATen registers its out variants):

    fds::flexrel_attention(Tensor qkv, int batch, int heads, Tensor rel,
                           Tensor? kv_len=None) -> Tensor
    fds::flexrel_attention.out(Tensor qkv, int batch, int heads, Tensor rel,
                               Tensor? kv_len=None, *, Tensor(a!) out) -> Tensor(a!)
    fds::rope_attention(Tensor qkv, int batch, int heads, Tensor cos,
                        Tensor sin) -> Tensor
    fds::rope_attention.out(Tensor qkv, int batch, int heads, Tensor cos,
                            Tensor sin, *, Tensor(a!) out, Tensor(b!) scratch) -> Tensor(a!)
    fds::window_attention(Tensor q, Tensor k, Tensor v, int left, int right=0, int sinks=0,
                          Tensor? q_start=None, Tensor? kv_len=None, *, float? scale=None) -> Tensor
    fds::quantize_rows(Tensor x) -> (Tensor, Tensor)
    fds::linear_int8(Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, Tensor? b=None, *,
                     ScalarType? dtype=None) -> Tensor
    fds::linear_int8_rope(Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, Tensor? b, Tensor cos,
                          Tensor sin, SymInt length, int heads, *, ScalarType? dtype=None) -> Tensor
    fds::accumulate_int8(Tensor(a!) x, Tensor a, Tensor a_scale, Tensor w, Tensor w_scale,
                         Tensor? b=None) -> ()
    fds::residual_norm_(Tensor(a!) x, Tensor? y=None, *, <the function's keywords>) -> Tensor
    fds::residual_norm_int8_(<the same>) -> (Tensor, Tensor)

``window_attention``, ``quantize_rows``, ``linear_int8`` and ``linear_int8_rope``
have ``.out`` overloads too. ``residual_norm_`` leaves x' in x and returns h,
``residual_norm_int8_`` returns h's 8-bit rows and their scales.

``torch.ops.fds.flexrel_attention(qkv, b, h, rel, out=buf)`` resolves to the
``.out`` overload, writes the context into ``buf`` and returns it: nothing is
allocated, so the call can sit inside a CUDA-graph capture with a fixed memory
plan. The functional overloads allocate their result. All of them route to the
same C-ABI calls as :mod:`.kernels`; the fake (meta) implementations let
``torch.compile`` / export trace through them.
"""

from __future__ import annotations

import torch

from . import kernels as _k
from . import layer_ops as _l

_lib = torch.library.Library("fds", "DEF")
_lib.define("flexrel_attention(Tensor qkv, int batch, int heads, Tensor rel, Tensor? kv_len=None) -> Tensor")
_lib.define("flexrel_attention.out(Tensor qkv, int batch, int heads, Tensor rel, Tensor? kv_len=None, *, "
            "Tensor(a!) out) -> Tensor(a!)")
_lib.define("rope_attention(Tensor qkv, int batch, int heads, Tensor cos, Tensor sin) -> Tensor")
_lib.define("rope_attention.out(Tensor qkv, int batch, int heads, Tensor cos, Tensor sin, *, "
            "Tensor(a!) out, Tensor(b!) scratch) -> Tensor(a!)")
_WINDOW = ("Tensor q, Tensor k, Tensor v, int left, int right=0, int sinks=0, Tensor? q_start=None, Tensor? kv_len=None, *, "
           "float? scale=None")
_lib.define(f"window_attention({_WINDOW}) -> Tensor")
_lib.define(f"window_attention.out({_WINDOW}, Tensor(a!) out) -> Tensor(a!)")
_lib.define("quantize_rows(Tensor x) -> (Tensor, Tensor)")
_lib.define("quantize_rows.out(Tensor x, *, Tensor(a!) out, Tensor(b!) scale) -> (Tensor(a!), Tensor(b!))")
_INT8 = "Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, Tensor? b=None"
_ROPE8 = "Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, Tensor? b, Tensor cos, Tensor sin, SymInt length, int heads"
for _name, _args in (("linear_int8", _INT8), ("linear_int8_rope", _ROPE8)):
    _lib.define(f"{_name}({_args}, *, ScalarType? dtype=None) -> Tensor")
    _lib.define(f"{_name}.out({_args}, *, Tensor(a!) out) -> Tensor(a!)")
_lib.define("accumulate_int8(Tensor(a!) x, Tensor a, Tensor a_scale, Tensor w, Tensor w_scale, Tensor? b=None) -> ()")
_NORM = ("Tensor(a!) x, Tensor? y=None, *, Tensor? gate=None, float residual_scale=1.0, str post='none', Tensor? post_weight=None, "
         "Tensor? post_bias=None, str norm='layer', Tensor? weight=None, Tensor? bias=None, Tensor? scale=None, "
         "Tensor? shift=None, SymInt? length=None, float eps=1e-5, ScalarType? dtype=None")
_lib.define(f"residual_norm_({_NORM}) -> Tensor")
_lib.define(f"residual_norm_int8_({_NORM}) -> (Tensor, Tensor)")


def _flexrel(qkv, batch, heads, rel, kv_len=None):
    return _k.flexrel_attention(qkv, batch, heads, rel, kv_len=kv_len)


def _flexrel_out(qkv, batch, heads, rel, kv_len=None, *, out):
    return _k.flexrel_attention(qkv, batch, heads, rel, out=out, kv_len=kv_len)


def _rope(qkv, batch, heads, cos, sin):
    return _k.rope_attention(qkv, batch, heads, cos, sin)


def _rope_out(qkv, batch, heads, cos, sin, *, out, scratch):
    return _k.rope_attention(qkv, batch, heads, cos, sin, out=out, scratch=scratch)


_lib.impl("flexrel_attention", _flexrel, "CUDA")
_lib.impl("flexrel_attention.out", _flexrel_out, "CUDA")
_lib.impl("rope_attention", _rope, "CUDA")
_lib.impl("rope_attention.out", _rope_out, "CUDA")


def _window(q, k, v, left, right=0, sinks=0, q_start=None, kv_len=None, *, scale=None, out=None):
    return _l.window_attention(q, k, v, left, right, sinks, q_start, kv_len, out, scale=scale)


def _linear8(x, x_scale, w, w_scale, b=None, *, dtype=None):
    return _l.linear_int8(x, x_scale, w, w_scale, b, dtype=dtype)


def _linear8_out(x, x_scale, w, w_scale, b=None, *, out):
    return _l.linear_int8(x, x_scale, w, w_scale, b, out, dtype=out.dtype)


def _rope8(x, x_scale, w, w_scale, b, cos, sin, length, heads, *, dtype=None):
    return _l.linear_int8_rope(x, x_scale, w, w_scale, b, cos, sin, length, heads, dtype=dtype)


def _rope8_out(x, x_scale, w, w_scale, b, cos, sin, length, heads, *, out):
    return _l.linear_int8_rope(x, x_scale, w, w_scale, b, cos, sin, length, heads, out, dtype=out.dtype)


_lib.impl("window_attention", _window, "CUDA")
_lib.impl("window_attention.out", _window, "CUDA")
_lib.impl("quantize_rows", lambda x: _l.quantize_rows(x), "CUDA")
_lib.impl("quantize_rows.out", lambda x, *, out, scale: _l.quantize_rows(x, out, scale), "CUDA")
_lib.impl("linear_int8", _linear8, "CUDA")
_lib.impl("linear_int8.out", _linear8_out, "CUDA")
_lib.impl("linear_int8_rope", _rope8, "CUDA")
_lib.impl("linear_int8_rope.out", _rope8_out, "CUDA")
_lib.impl("accumulate_int8", lambda *a: _l.accumulate_int8(*a), "CUDA")
_lib.impl("residual_norm_", lambda x, y=None, **kw: _l.residual_norm(x, y, **kw)[1], "CUDA")
_lib.impl("residual_norm_int8_", lambda x, y=None, **kw: _l.residual_norm(x, y, quantize=True, **kw)[1], "CUDA")


def _context_like(qkv):
    return qkv.new_empty(qkv.shape[0], qkv.shape[1] // 3)


@torch.library.register_fake("fds::flexrel_attention", lib=_lib)
def _(qkv, batch, heads, rel, kv_len=None):
    return _context_like(qkv)


@torch.library.register_fake("fds::rope_attention", lib=_lib)
def _(qkv, batch, heads, cos, sin):
    return _context_like(qkv)


@torch.library.register_fake("fds::window_attention", lib=_lib)
def _(q, k, v, left, right=0, sinks=0, q_start=None, kv_len=None, *, scale=None):
    return q.new_empty(q.shape)


def _int8_rows(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32)


def _projected(x, x_scale, w, w_scale, b=None, *_, dtype=None):
    return x.new_empty(x.shape[0], w.shape[0], dtype=dtype or (torch.float16 if b is None else b.dtype))


def _normed(x, y=None, *, dtype=None, **_):
    return x.new_empty(x.shape, dtype=dtype or (y.dtype if y is not None else torch.float16 if x.dtype == torch.float32 else x.dtype))


torch.library.register_fake("fds::quantize_rows", _int8_rows, lib=_lib)
torch.library.register_fake("fds::linear_int8", _projected, lib=_lib)
torch.library.register_fake("fds::linear_int8_rope", _projected, lib=_lib)
torch.library.register_fake("fds::accumulate_int8", lambda *a: None, lib=_lib)
torch.library.register_fake("fds::residual_norm_", _normed, lib=_lib)
torch.library.register_fake("fds::residual_norm_int8_", lambda x, y=None, **_: _int8_rows(x), lib=_lib)


# the out= overloads return their (caller-owned) `out` argument
_lib.impl("flexrel_attention.out", lambda qkv, batch, heads, rel, kv_len=None, *, out: out, "Meta")
_lib.impl("rope_attention.out", lambda qkv, batch, heads, cos, sin, *, out, scratch: out, "Meta")
for _name in ("window_attention", "linear_int8", "linear_int8_rope"):
    _lib.impl(f"{_name}.out", lambda *a, out, **kw: out, "Meta")
_lib.impl("quantize_rows.out", lambda x, *, out, scale: (out, scale), "Meta")

# kept as module attributes for callers of the earlier Python-level names
flexrel_attention_op = torch.ops.fds.flexrel_attention
rope_attention_op = torch.ops.fds.rope_attention
