"""64-bit CPU oracle for the window attention, the 8-bit projections and the
residual norm -- TEST INFRASTRUCTURE, as :mod:`oracle.flexrel_oracle`.

Each function is the operator's definition in float64, from the same (already
rounded) inputs, with no blocking and no rounding of intermediates.
"""

from __future__ import annotations

import torch


def window_attention(q, k, v, left, right=0, sinks=0, q_start=None, kv_len=None, scale=0.125):
    """q [B, Lq, H, D], k / v [B, Lk, Hk, D] -> [B, Lq, H, D] float64; a query
    that sees no key gives zeros. Excluded keys are dropped, not weighted by 0,
    so they may hold anything."""
    batch, q_len, heads, dim = q.shape
    k_len, group = k.shape[1], heads // k.shape[2]
    out = torch.zeros(batch, q_len, heads, dim, dtype=torch.float64)
    for b in range(batch):
        start = 0 if q_start is None else int(q_start[b])
        end = k_len if kv_len is None else min(max(int(kv_len[b]), 0), k_len)
        for i in range(q_len):
            p = start + i
            seen = [j for j in range(min(end, max(0, p + right + 1))) if j >= p - left or j < sinks]
            if not seen:
                continue
            for h in range(heads):
                s = (k[b, seen, h // group].double() @ q[b, i, h].double()) * scale
                w = torch.exp(s - s.max())
                out[b, i, h] = (w @ v[b, seen, h // group].double()) / w.sum()
    return out


def window_attention_by_head(q, k, v, left, right=0, sinks=0, q_start=None, kv_len=None, scale=0.125):
    """:func:`window_attention` as one product per window and head, on the tensors'
    device, for sizes the loop over queries is too slow for. Excluded keys weigh 0,
    and those that no query of a window sees are dropped."""
    batch, q_len, heads, dim = q.shape
    k_len, group, dev = k.shape[1], heads // k.shape[2], q.device
    out = torch.zeros(batch, q_len, heads, dim, dtype=torch.float64, device=dev)
    j = torch.arange(k_len, device=dev)
    for b in range(batch):
        end = k_len if kv_len is None else min(max(int(kv_len[b]), 0), k_len)
        p = (0 if q_start is None else int(q_start[b])) + torch.arange(q_len, device=dev)[:, None]
        seen = (j < end) & (j <= p + right) & ((j >= p - left) | (j < sinks))
        ids = seen.any(0).nonzero()[:, 0]
        if len(ids) == 0:
            continue
        seen, some = seen[:, ids], seen.any(1)
        for h in range(heads):
            s = (q[b, :, h].double() @ k[b, ids, h // group].double().t()) * scale
            s = torch.where(seen, s, -torch.inf)
            w = torch.exp(s - torch.where(some, s.amax(1), 0.0)[:, None])
            o = (w @ v[b, ids, h // group].double()) / w.sum(1, keepdim=True)
            out[b, :, h] = torch.where(some[:, None], o, 0.0)
    return out


def quantize_rows(x):
    """(int8, fp32 scale) by the operator's definition, in fp32 as it states it."""
    x = x.float()
    big = x.abs().amax(1, keepdim=True)
    tiny = big < 2.0 ** -100
    inv = torch.where(tiny, torch.zeros_like(big), torch.full_like(big, 127.0) / big)  # one rounding; 127.0 / big has two
    q = torch.round(x * inv).to(torch.int8)
    return q, torch.where(tiny, torch.zeros_like(big), big / 127.0)[:, 0]


def linear_int8(x, x_scale, w, w_scale, b=None):
    """(product term, result) in float64; the product term alone bounds the rounding."""
    y = (x.double() @ w.double().t()) * x_scale.double()[:, None] * w_scale.double()[None]
    return y, (y if b is None else y + b.double())


def rope(y, cos, sin, length, cols):
    """Rotate-half RoPE of the 64-column heads of y[:, :cols] at row % length."""
    y = y.clone()
    t = torch.arange(y.shape[0]) % length
    c, s = cos.double()[t], sin.double()[t]
    for at in range(0, cols, 64):
        u = y[:, at:at + 64]
        y[:, at:at + 64] = u * c + torch.cat([-u[:, 32:], u[:, :32]], 1) * s
    return y


def _norm(t, kind, weight, bias, eps):
    if kind == "layer":
        t = t - t.mean(1, keepdim=True)
    if kind != "none":
        t = t / torch.sqrt((t * t).mean(1, keepdim=True) + eps)
    if weight is not None:
        t = t * weight.double()
    return t if bias is None else t + bias.double()


def residual_norm(x, y=None, gate=None, residual_scale=1.0, post="none", post_weight=None, post_bias=None, norm="layer",
                  weight=None, bias=None, scale=None, shift=None, length=None, eps=1e-5):
    """(x', h) in float64."""
    x = x.double()
    win = torch.arange(x.shape[0]) // (length or max(1, x.shape[0]))

    def per_row(t):
        return t.double() if t.dim() == 1 else t.double()[win]

    if y is not None:
        z = _norm(y.double(), post, post_weight, post_bias, eps)
        x = residual_scale * x + (z if gate is None else z * per_row(gate))
    h = _norm(x, norm, weight, bias, eps)
    if scale is not None:
        h = h * (1 + per_row(scale))
    if shift is not None:
        h = h + per_row(shift)
    return x, h


