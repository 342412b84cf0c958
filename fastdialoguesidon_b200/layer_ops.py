"""What a layer needs around the 120 s attention and the 16-bit projections:
attention over a sliding window with sinks, projections in 8-bit integers, and
the step between two blocks (norms, gate, residual scale) in one pass.

* :func:`window_attention` -- a window of keys per query and a few first keys
  that stay visible, from one query (a stream's next frame against a cache) to
  a whole recording, at a cost linear in its length.
* :func:`quantize_rows`, :func:`linear_int8`, :func:`linear_int8_rope`,
  :func:`accumulate_int8` -- ``linear``, ``linear_rope`` and ``accumulate`` of
  :mod:`.kernels` over int8 operands with one fp32 scale per token and per
  output channel.
* :func:`residual_norm` -- the norm after a block, its gate, the residual scale
  and the norm (with the adaLN modulation) before the next block; can quantise
  its rows for the 8-bit projections.

The calls keep the rules of :mod:`.kernels`: they launch on the current stream,
never synchronise, allocate nothing but the outputs that are not given, raise
:class:`FdsError` before any launch on an invalid argument, and have no CPU
fallback. They compute forward only.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .kernels import (
    _DTYPES,
    HEAD_DIM,
    FdsError,
    _check,
    _on_device,
    _raise_if_timed_out,
    _raise_rc,
    _rope_tables,
    _status,
    _status_mirror,
    _stream_ptr,
)

_NORMS = {"none": N.FDS_NORM_NONE, "layer": N.FDS_NORM_LAYER, "rms": N.FDS_NORM_RMS}
_Strides = ctypes.c_int64 * 3


def _call(fn_name: str, args, dev: torch.device) -> None:
    fn = getattr(N.load(), fn_name)
    with _on_device(dev):
        rc = fn(args, _stream_ptr(dev))
    if rc != N.FDS_OK:
        _raise_rc(rc, fn_name)


def _tensor(t, name: str, dtypes, dev: torch.device | None = None) -> None:
    _check(isinstance(t, torch.Tensor), lambda: f"{name} must be a torch.Tensor")
    _check(t.dtype in dtypes, lambda: f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if dev is None:
        _check(t.is_cuda, lambda: f"{name} must be on a CUDA device (there is no CPU fallback)")
    else:
        _check(t.device == dev, lambda: f"{name} must be on {dev}, got {t.device}")


def _rows(t, name: str, dtypes, dev: torch.device | None = None, align: int = 16) -> None:
    """2-D, contiguous columns, rows on ``align``-byte boundaries."""
    _tensor(t, name, dtypes, dev)
    _check(t.dim() == 2, lambda: f"{name} must be 2-D [rows, columns], got {tuple(t.shape)}")
    rows, cols = t.shape
    _check(cols <= 1 or t.stride(1) == 1, lambda: f"{name} columns must be contiguous (stride(1) == 1)")
    _check(t.data_ptr() % align == 0 and (rows <= 1 or (t.stride(0) >= cols and t.stride(0) * t.element_size() % align == 0)),
           lambda: f"{name} rows must be {align}-byte aligned and not overlap")


def _stride(t: torch.Tensor) -> int:
    """Row stride in elements; the width of a single row is never stepped over."""
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 16) * 16


# ---------------------------------------------------------------- window attention


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: int, right: int = 0, sinks: int = 0,
                     q_start: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, *, scale: float | None = None, timeout_ns: int = 0) -> torch.Tensor:
    """Softmax attention of each query over a window of keys and the first ``sinks`` keys.

    q [B, Lq, H, 64], k and v [B, Lk, Hk, 64] fp16 / bf16, H a multiple of Hk
    (query head h reads key head ``h // (H / Hk)``) -> [B, Lq, H, 64], written
    into ``out`` when given. Query i of window b sits at position
    ``p = q_start[b] + i`` (``q_start`` int32 CUDA [B], default 0) and sees key j
    iff ``j < kv_len[b]`` (int32 CUDA [B], default Lk), ``j <= p + right`` and
    (``j >= p - left`` or ``j < sinks``). A query that sees no key yields zeros.
    ``scale`` defaults to 1/sqrt(64).

    The tensors may be views: any strides that are multiples of 8 elements with
    contiguous 64-element heads, so ``qkv.view(B, L, 3, H, 64)[:, :, 0]`` of a
    projection's output and a ``[B, H, L, 64]`` cache transposed to
    ``[B, L, H, 64]`` are read in place. Rows of k and v that no query of a
    128-row block sees (a cache's unwritten tail) may hold anything.

    A stream's next frame: ``q`` with Lq = 1, its cache as k and v with the
    frame's own key and value written at ``q_start``, ``right=0``.
    """
    _tensor(q, "q", _DTYPES)
    dev, dt = q.device, q.dtype
    _tensor(k, "k", (dt,), dev)
    _tensor(v, "v", (dt,), dev)
    _check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k and v must be 4-D [batch, length, heads, 64]")
    batch, q_len, heads, dim = q.shape
    _check(dim == HEAD_DIM, lambda: f"head_dim must be 64, got {dim}")
    _check(k.shape == v.shape and k.shape[0] == batch and k.shape[3] == dim,
           lambda: f"k and v must be [{batch}, length, heads, {dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
    k_len, kv_heads = k.shape[1], k.shape[2]
    _check(batch >= 1 and kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0,
           lambda: f"heads ({heads}) must be a positive multiple of the key heads ({kv_heads})")
    _check(left >= 0 and right >= 0 and sinks >= 0, "left, right and sinks must be >= 0")
    if out is None:
        out = torch.empty((batch, q_len, heads, dim), dtype=dt, device=dev)
    else:
        _tensor(out, "out", (dt,), dev)
        _check(out.shape == q.shape, lambda: f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        _check(t.stride(3) == 1, lambda: f"{name} heads must be contiguous (stride(3) == 1)")
    for name, t in (("q_start", q_start), ("kv_len", kv_len)):
        if t is not None:
            _tensor(t, name, (torch.int32,), dev)
            _check(t.shape == (batch,) and t.is_contiguous(), lambda: f"{name} must be a contiguous [{batch}] tensor")
    if q_len == 0:
        return out
    if k_len == 0:
        return out.zero_()
    _raise_if_timed_out(dev)
    top = 1 << 28
    args = N.FdsWindowArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _Strides(*q.stride()[:3]), _Strides(*k.stride()[:3]),
        _Strides(*v.stride()[:3]), _Strides(*out.stride()[:3]), None if q_start is None else q_start.data_ptr(),
        None if kv_len is None else kv_len.data_ptr(), _status(dev).data_ptr(), _status_mirror(dev).data_ptr(),
        batch, heads, kv_heads, q_len, k_len, dim, _DTYPES[dt], min(left, top), min(right, top), min(sinks, top),
        0.125 if scale is None else scale, timeout_ns)
    _call("fds_window_attn_fwd", args, dev)
    return out


# ---------------------------------------------------------------- 8-bit projections


def quantize_rows(x: torch.Tensor, out: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] fp16 / bf16 -> (int8 [M, K], fp32 [M]) with
    ``scale = max|x| / 127`` per row and ``q = rint(x * (127 / max|x|))`` (ties to
    even): the tokens of the 8-bit projections. K a multiple of 8, at most
    16384. A row whose maximum is below 2^-100 is zero with scale 0; one with an
    infinity or a NaN gets the scale NaN."""
    _rows(x, "x", _DTYPES)
    rows, c = x.shape
    dev = x.device
    out, scale = _int8_rows(out, scale, rows, c, dev, "out")
    if rows == 0:
        return out, scale
    args = N.FdsResidualNormArgs(
        x.data_ptr(), _stride(x), None, 0, None, 0, out.data_ptr(), _stride(out), scale.data_ptr(),
        None, 0, None, None, None, None, None, None, 0, rows, c, rows, _DTYPES[x.dtype], 0, 0,
        N.FDS_NORM_NONE, N.FDS_NORM_NONE, 1.0, 0.0)
    _call("fds_residual_norm_fwd", args, dev)
    return out, scale


def _int8_rows(out, scale, rows: int, c: int, dev: torch.device, name: str):
    if out is None:
        out = torch.empty((rows, c), dtype=torch.int8, device=dev)
    else:
        _rows(out, name, (torch.int8,), dev, align=8)
        _check(out.shape == (rows, c), lambda: f"{name} must be [{rows}, {c}], got {tuple(out.shape)}")
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=dev)
    else:
        _vector(scale, "scale", rows, (torch.float32,), dev, align=4)
    return out, scale


def _vector(t, name: str, n: int, dtypes, dev: torch.device, align: int = 16) -> None:
    _tensor(t, name, dtypes, dev)
    _check(t.shape == (n,) and (n <= 1 or t.stride(0) == 1) and t.data_ptr() % align == 0,
           lambda: f"{name} must be a contiguous, {align}-byte aligned [{n}] tensor, got {tuple(t.shape)}")


def _linear_int8(x, x_scale, w, w_scale, b, out, dtype, epilogue, cos=None, sin=None, seq_len: int = 0, rope_cols: int = 0,
                 pair: bool | None = None, tile_n: int = 0):
    _rows(x, "x", (torch.int8,))
    dev = x.device
    _rows(w, "w", (torch.int8,), dev)
    m, k = x.shape
    n, kw = w.shape
    _check(kw == k, lambda: f"w is [{n}, {kw}] but x has {k} columns")
    _check(k % 16 == 0 and 0 < k <= 65536, lambda: f"in_features must be a multiple of 16, at most 65536 (got {k})")
    _check(n % 8 == 0 and n > 0, lambda: f"out_features must be a multiple of 8 (got {n})")
    _vector(x_scale, "x_scale", m, (torch.float32,), dev, align=4)
    _vector(w_scale, "w_scale", n, (torch.float32,), dev)
    accum = epilogue == N.FDS_EPILOGUE_ACCUMULATE_F32
    if dtype is None:
        dtype = b.dtype if isinstance(b, torch.Tensor) else torch.float16
    _check(dtype in _DTYPES, lambda: f"dtype must be float16 or bfloat16, got {dtype}")
    if b is not None:
        _vector(b, "b", n, (dtype,), dev)
    out_dtype = torch.float32 if accum else dtype
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=dev)
    else:
        _rows(out, "x" if accum else "out", (out_dtype,), dev)
        _check(out.shape == (m, n), lambda: f"the output must be [{m}, {n}], got {tuple(out.shape)}")
    if m == 0:
        return out
    _raise_if_timed_out(dev)
    args = N.FdsLinearInt8Args(
        x.data_ptr(), _stride(x), x_scale.data_ptr(), w.data_ptr(), _stride(w), w_scale.data_ptr(),
        None if b is None else b.data_ptr(), out.data_ptr(), out.stride(0) if m > 1 else n,
        None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(),
        _status(dev).data_ptr(), _status_mirror(dev).data_ptr(), m, n, k, _DTYPES[dtype], epilogue, seq_len, rope_cols, 0,
        tile_n, N.FDS_GEMM_AUTO if pair is None else (N.FDS_GEMM_PAIR if pair else N.FDS_GEMM_SINGLE))
    _call("fds_linear_int8_fwd", args, dev)
    return out


def linear_int8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                b: torch.Tensor | None = None, out: torch.Tensor | None = None, *, dtype: torch.dtype | None = None,
                pair: bool | None = None, tile_n: int = 0) -> torch.Tensor:
    """``(x @ w.T) * x_scale[:, None] * w_scale[None, :] + b`` with x [M, K] and
    w [N, K] (nn.Linear layout) int8, x_scale [M] and w_scale [N] fp32, rounded
    once to ``dtype`` (fp16 / bf16; b's, or fp16, when not given). The products
    are summed exactly, in 32-bit integers. K a multiple of 16 up to 65536, N a
    multiple of 8, rows 16-byte aligned. The 8-bit :func:`linear`.

    Up to 8 rows run on a kernel that reads w once over all SMs. ``pair`` and
    ``tile_n`` (64, 128, 256) force the tensor-core tiling that is chosen by
    shape otherwise; every choice gives the same result bit for bit."""
    return _linear_int8(x, x_scale, w, w_scale, b, out, dtype, N.FDS_EPILOGUE_STORE, pair=pair, tile_n=tile_n)


def linear_int8_rope(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                     b: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, length: int, heads: int,
                     out: torch.Tensor | None = None, *, dtype: torch.dtype | None = None, pair: bool | None = None,
                     tile_n: int = 0) -> torch.Tensor:
    """The DiT's QKV projection with RoPE in its epilogue (:func:`linear_rope`)
    over int8 operands: the q and k column blocks of :func:`linear_int8`'s
    result rotated in fp32 at position ``row % length``, then rounded once."""
    _check(isinstance(w, torch.Tensor) and w.dim() == 2, "w must be a 2-D tensor")
    n = w.shape[0]
    _check(heads >= 1 and n == 3 * heads * HEAD_DIM, lambda: f"w must have 3*heads*64 = {3 * heads * HEAD_DIM} rows (got {n})")
    _check(length >= 1, "length must be >= 1")
    _rows(x, "x", (torch.int8,))
    seq_len = min(length, max(1, x.shape[0]))  # rows past a table are never addressed
    _rope_tables(cos, sin, seq_len, x)
    return _linear_int8(x, x_scale, w, w_scale, b, out, dtype, N.FDS_EPILOGUE_ROPE, cos, sin, seq_len, 2 * heads * HEAD_DIM,
                        pair=pair, tile_n=tile_n)


def accumulate_int8(x: torch.Tensor, a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                    b: torch.Tensor | None = None, *, pair: bool | None = None, tile_n: int = 0) -> None:
    """``x += (a @ w.T) * a_scale[:, None] * w_scale[None, :] (+ b)`` in place, x
    [M, N] the fp32 residual: :func:`accumulate` over int8 operands."""
    _rows(x, "x", (torch.float32,))
    _linear_int8(a, a_scale, w, w_scale, b, x, None, N.FDS_EPILOGUE_ACCUMULATE_F32, pair=pair, tile_n=tile_n)


# ---------------------------------------------------------------- between two blocks


def residual_norm(x: torch.Tensor, y: torch.Tensor | None = None, *, gate: torch.Tensor | None = None,
                  residual_scale: float = 1.0, post: str = "none", post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, norm: str = "layer", weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, scale: torch.Tensor | None = None, shift: torch.Tensor | None = None,
                  length: int | None = None, eps: float = 1e-5, dtype: torch.dtype | None = None,
                  residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None, quantize: bool = False,
                  out_scale: torch.Tensor | None = None):
    """The step between two blocks, in one pass over the rows:

        z  = post(y) * post_weight + post_bias
        x' = residual_scale * x + gate * z
        h  = (norm(x') * weight + bias) * (1 + scale) + shift

    x [R, C] is the residual stream (fp32, or y's type), y [R, C] fp16 / bf16 the
    block's output; ``post`` and ``norm`` are "none", "layer" (LayerNorm) or "rms"
    (RMS norm) with ``eps`` inside the root. gate, scale and shift are [C], or
    [windows, C] read at ``row // length`` (adaLN). All vectors are optional and
    of one type, fp32 or that of y. Returns ``(x', h)``: x' written to
    ``residual_out`` (x itself when not given), h in ``dtype`` (y's type, x's
    16-bit type, or fp16) to ``out``. h is computed from the 32-bit x', not from
    its rounding to a 16-bit stream. With ``quantize`` h is
    ``(int8 [R, C], fp32 [R])`` as :func:`quantize_rows` defines it, from the
    32-bit h. Without y, x' is x, untouched. C a multiple of 8, at most 16384.

    Reference: ``res_norm`` (triton/src/fds_triton/kernels.py:61), without the
    norm after the block."""
    _rows(x, "x", (torch.float32, *_DTYPES))
    dev = x.device
    rows, c = x.shape
    t = dtype if dtype is not None else (y.dtype if isinstance(y, torch.Tensor) else
                                         (x.dtype if x.dtype in _DTYPES else torch.float16))
    _check(t in _DTYPES, lambda: f"dtype must be float16 or bfloat16, got {t}")
    _check(c % 8 == 0 and 8 <= c <= 16384, lambda: f"columns must be a multiple of 8, at most 16384 (got {c})")
    _check(x.dtype in (torch.float32, t), lambda: f"x must be float32 or {t}, got {x.dtype}")
    _check(post in _NORMS and norm in _NORMS, lambda: f"post and norm must be 'none', 'layer' or 'rms' (got {post!r}, {norm!r})")
    length = max(1, rows) if length is None else length
    _check(length >= 1, "length must be >= 1")
    if y is not None:
        _rows(y, "y", (t,), dev)
        _check(y.shape == (rows, c), lambda: f"y must be [{rows}, {c}], got {tuple(y.shape)}")
        residual_out = x if residual_out is None else residual_out
        _rows(residual_out, "residual_out", (x.dtype,), dev)
        _check(residual_out.shape == (rows, c), lambda: f"residual_out must be [{rows}, {c}], got {tuple(residual_out.shape)}")
    else:
        _check(gate is None and post == "none" and post_weight is None and post_bias is None and residual_scale == 1.0
               and residual_out is None, "gate, residual_scale, residual_out and the norm after the block need y")
    pt = next((p.dtype for p in (gate, post_weight, post_bias, weight, bias, scale, shift) if isinstance(p, torch.Tensor)), t)
    _check(pt in (torch.float32, t), lambda: f"parameter vectors must be float32 or {t}, got {pt}")
    for name, p in (("post_weight", post_weight), ("post_bias", post_bias), ("weight", weight), ("bias", bias)):
        if p is not None:
            _vector(p, name, c, (pt,), dev)
    gate_stride = _per_window(gate, "gate", rows, c, length, pt, dev)
    mod_stride = _per_window(scale, "scale", rows, c, length, pt, dev)
    shift_stride = _per_window(shift, "shift", rows, c, length, pt, dev)
    if scale is not None and shift is not None:
        _check(mod_stride == shift_stride, "scale and shift must have the same layout")
    mod_stride = max(mod_stride, shift_stride)
    if quantize:
        out, out_scale = _int8_rows(out, out_scale, rows, c, dev, "out")
    else:
        _check(out_scale is None, "out_scale is for quantize=True")
        if out is None:
            out = torch.empty((rows, c), dtype=t, device=dev)
        else:
            _rows(out, "out", (t,), dev)
            _check(out.shape == (rows, c), lambda: f"out must be [{rows}, {c}], got {tuple(out.shape)}")
    new_x = x if y is None else residual_out
    h = (out, out_scale) if quantize else out
    if rows == 0:
        return new_x, h
    ptr = (lambda p: None if p is None else p.data_ptr())
    args = N.FdsResidualNormArgs(
        x.data_ptr(), _stride(x), ptr(y), 0 if y is None else _stride(y), ptr(residual_out),
        0 if y is None else _stride(residual_out), out.data_ptr(), _stride(out), ptr(out_scale),
        ptr(gate), gate_stride, ptr(post_weight), ptr(post_bias), ptr(weight), ptr(bias), ptr(scale), ptr(shift), mod_stride,
        rows, c, length, _DTYPES[t], x.dtype == torch.float32, pt == torch.float32, _NORMS[post], _NORMS[norm],
        residual_scale, eps)
    _call("fds_residual_norm_fwd", args, dev)
    return new_x, h


def _per_window(t, name: str, rows: int, c: int, length: int, dtype, dev: torch.device) -> int:
    """Elements between the rows of a [C] (0) or [windows, C] vector; 0 when absent."""
    if t is None:
        return 0
    _tensor(t, name, (dtype,), dev)
    if t.dim() == 1:
        _vector(t, name, c, (dtype,), dev)
        return 0
    windows = -(-rows // length)
    _rows(t, name, (dtype,), dev)
    _check(t.shape[1] == c and t.shape[0] >= windows, lambda: f"{name} must be [{c}] or [{windows}, {c}], got {tuple(t.shape)}")
    return t.stride(0) if t.shape[0] > 1 else 0


__all__ = ["FdsError", "accumulate_int8", "linear_int8", "linear_int8_rope", "quantize_rows", "residual_norm",
           "window_attention"]
