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
import importlib.util
import threading

import torch

from . import _native as N
from . import build as _build
from .kernels import FdsError, _raise_if_timed_out, _status, _status_mirror

_ext = None
_lock = threading.Lock()


def _status_addresses(index: int) -> tuple[int, int]:
    dev = torch.device("cuda", index)
    return _status(dev).data_ptr(), _status_mirror(dev).data_ptr()


def _load():
    """The extension that checks the arguments and calls the C ABI
    (``csrc/torch_shim.cpp``), bound to the loaded library."""
    global _ext
    with _lock:
        if _ext is None:
            lib = N.load()
            path = _build.extension_path()
            if not path.exists():
                _build.build_extension()
            spec = importlib.util.spec_from_file_location("_fds_torch", path)
            ext = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(ext)
            ext.bind(FdsError, _status_addresses, lambda i: _raise_if_timed_out(torch.device("cuda", i)),
                     *(ctypes.cast(fn, ctypes.c_void_p).value for fn in (
                         lib.fds_last_error, lib.fds_linear_int8_fwd, lib.fds_residual_norm_fwd, lib.fds_window_attn_fwd)))
            _ext = ext
    return _ext


# ---------------------------------------------------------------- window attention


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: int, right: int = 0, sinks: int = 0,
                     q_start: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, *, scale: float | None = None, timeout_ns: int = 0,
                     debug_flags: int = 0) -> torch.Tensor:
    """Softmax attention of each query over a window of keys and the first ``sinks`` keys.

    q [B, Lq, H, 64], k and v [B, Lk, Hk, 64] fp16 / bf16, H a multiple of Hk
    (query head h reads key head ``h // (H / Hk)``) -> [B, Lq, H, 64], written
    into ``out`` when given. Query i of window b sits at position
    ``p = q_start[b] + i`` (``q_start`` int32 CUDA [B], default 0) and sees key j
    iff ``j < kv_len[b]`` (int32 CUDA [B], default Lk), ``j <= p + right`` and
    (``j >= p - left`` or ``j < sinks``). A query that sees no key, or none whose
    score is above minus infinity, yields zeros; one with a score that is NaN or
    plus infinity yields NaN. ``scale`` defaults to 1/sqrt(64).

    Scores, maxima, sums and the output before its rounding are fp32. The weights
    are rounded to the operand type before their product with v, which the tensor
    cores take in one type, and where more than 16 query rows share a key head 3 in
    10 exponentials come from a polynomial within 7.5e-5: the error against 64 bits
    is 1.2 to 1.4 times that of one rounding of the output. There is no relative-key
    bias (the encoder's is :func:`flexrel_attention`).

    The tensors may be views: any strides that are multiples of 8 elements, at least
    64 where a dimension is longer than one, with contiguous 64-element heads, so ``qkv.view(B, L, 3, H, 64)[:, :, 0]`` of a
    projection's output and a ``[B, H, L, 64]`` cache transposed to
    ``[B, L, H, 64]`` are read in place. Rows of k and v that no query of a
    128-row block sees (a cache's unwritten tail) may hold anything.

    A stream's next frame: ``q`` with Lq = 1, its cache as k and v with the
    frame's own key and value written at ``q_start``, ``right=0``.
    """
    return (_ext or _load()).window_attention(q, k, v, left, right, sinks, q_start, kv_len, out, scale, timeout_ns,
                                              debug_flags)


# ---------------------------------------------------------------- 8-bit projections

_PAIR = {None: N.FDS_GEMM_AUTO, True: N.FDS_GEMM_PAIR, False: N.FDS_GEMM_SINGLE}


def quantize_rows(x: torch.Tensor, out: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] fp16 / bf16 -> (int8 [M, K], fp32 [M]) with
    ``scale = max|x| / 127`` per row and ``q = rint(x * (127 / max|x|))`` (ties to
    even): the tokens of the 8-bit projections. K a multiple of 8, at most
    16384. A row whose maximum is below 2^-100 is zero with scale 0; one with an
    infinity or a NaN gets the scale NaN."""
    return (_ext or _load()).quantize_rows(x, out, scale)


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
    return (_ext or _load()).linear_int8(x, x_scale, w, w_scale, b, out, dtype, N.FDS_EPILOGUE_STORE, None, None, 0, 0,
                                         _PAIR[pair], tile_n)


def linear_int8_rope(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                     b: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, length: int, heads: int,
                     out: torch.Tensor | None = None, *, dtype: torch.dtype | None = None, pair: bool | None = None,
                     tile_n: int = 0) -> torch.Tensor:
    """The DiT's QKV projection with RoPE in its epilogue (:func:`linear_rope`)
    over int8 operands: the q and k column blocks of :func:`linear_int8`'s
    result rotated in fp32 at position ``row % length``, then rounded once. The two
    32-column halves of ``cos`` and ``sin`` are equal, as :func:`rope_tables` builds
    them: only the first is read."""
    return (_ext or _load()).linear_int8(x, x_scale, w, w_scale, b, out, dtype, N.FDS_EPILOGUE_ROPE, cos, sin, length, heads,
                                         _PAIR[pair], tile_n)


def accumulate_int8(x: torch.Tensor, a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                    b: torch.Tensor | None = None, *, pair: bool | None = None, tile_n: int = 0) -> None:
    """``x += (a @ w.T) * a_scale[:, None] * w_scale[None, :] (+ b)`` in place, x
    [M, N] the fp32 residual: :func:`accumulate` over int8 operands."""
    (_ext or _load()).linear_int8(a, a_scale, w, w_scale, b, x, None, N.FDS_EPILOGUE_ACCUMULATE_F32, None, None, 0, 0,
                                  _PAIR[pair], tile_n)


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
    return (_ext or _load()).residual_norm(x, y, gate, residual_scale, post, post_weight, post_bias, norm, weight, bias, scale,
                                           shift, length, eps, dtype, residual_out, out, quantize, out_scale)


__all__ = ["FdsError", "accumulate_int8", "linear_int8", "linear_int8_rope", "quantize_rows", "residual_norm",
           "window_attention"]
