"""A DiT layer in 8 bits over a recording of any length, and frame by frame.

The layer's parts are the package's operators, in the order a model runs them:

    residual_norm (adaLN, 8-bit rows out) -> linear_int8_rope (QKV) ->
    window_attention (a window of frames and the first ones) -> quantize_rows ->
    linear_int8 (out-projection) -> residual_norm (gate, residual, next adaLN)

``forward`` takes a whole recording; its attention costs length x window.
``step`` takes the next frames of a stream against a cache of keys and values and
gives what ``forward`` with ``right=0`` gives for those frames. ``forward_fp32`` is
the layer in plain fp32 torch with the weights before quantisation.

    python examples/long_recording_int8.py [frames]
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

REPO = Path(__file__).resolve().parents[1]
if str(REPO) not in sys.path:
    sys.path.insert(0, str(REPO))

import fastdialoguesidon_b200 as F  # noqa: E402

HEADS, HIDDEN = 12, 768
LEFT, RIGHT, SINKS = 500, 500, 8  # 10 s either side at 50 frames a second


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[N, K] -> int8 and one scale per output channel."""
    scale = w.abs().amax(1) / 127
    return torch.round(w / scale[:, None]).to(torch.int8), scale


class DitLayer:
    """Random weights of the DiT head's architecture (12 x 64 heads)."""

    def __init__(self, max_frames: int, device="cuda", seed: int = 0):
        g = torch.Generator().manual_seed(seed)

        def rnd(*shape, scale):
            return (torch.randn(*shape, generator=g) * scale).to(device)

        self.qkv_w, self.out_w = rnd(3 * HIDDEN, HIDDEN, scale=0.04), rnd(HIDDEN, HIDDEN, scale=0.04)
        self.qkv_b, self.out_b = rnd(3 * HIDDEN, scale=0.02).half(), rnd(HIDDEN, scale=0.02).half()
        # adaLN vectors of the speaker / time condition: before the attention, its gate, before the FFN
        self.scale, self.shift, self.gate = (rnd(HIDDEN, scale=0.2).half() for _ in range(3))
        self.ffn_scale, self.ffn_shift = (rnd(HIDDEN, scale=0.2).half() for _ in range(2))
        self.qkv8, self.out8 = quantize_weight(self.qkv_w), quantize_weight(self.out_w)
        self.cos, self.sin = F.rope_tables(max_frames, device)

    def qkv(self, x: torch.Tensor, first: int) -> torch.Tensor:
        """Rotated q | k | v of frames at positions first, first + 1, ...: [frames, 3, heads, 64]."""
        n = x.shape[0]
        _, (h, hs) = F.residual_norm(x, scale=self.scale, shift=self.shift, quantize=True, dtype=torch.float16)
        y = F.linear_int8_rope(h, hs, *self.qkv8, self.qkv_b, self.cos[first:first + n], self.sin[first:first + n], n, HEADS)
        return y.view(n, 3, HEADS, 64)

    def finish(self, x: torch.Tensor, context: torch.Tensor):
        """Out-projection, gate and residual; -> (x in place, the FFN's input)."""
        y = F.linear_int8(*F.quantize_rows(context.reshape(-1, HIDDEN)), *self.out8, self.out_b)
        return F.residual_norm(x, y, gate=self.gate, scale=self.ffn_scale, shift=self.ffn_shift)

    def forward(self, x: torch.Tensor, left: int = LEFT, right: int = RIGHT, sinks: int = SINKS):
        q, k, v = self.qkv(x, 0)[None].unbind(2)
        return self.finish(x, F.window_attention(q, k, v, left, right, sinks))

    def new_cache(self, frames: int) -> torch.Tensor:
        """Keys and values of one stream, unwritten: [2, 1, frames, heads, 64]."""
        return torch.empty(2, 1, frames, HEADS, 64, dtype=torch.float16, device=self.cos.device)

    def step(self, x: torch.Tensor, cache: torch.Tensor, first: int, left: int = LEFT, sinks: int = SINKS):
        """The frames at positions first, ... (x [n, HIDDEN]) of a stream."""
        n = x.shape[0]
        qkv = self.qkv(x, first)
        cache[:, 0, first:first + n] = qkv[:, 1:].transpose(0, 1)
        start = torch.tensor([first], dtype=torch.int32, device=x.device)
        return self.finish(x, F.window_attention(qkv[None, :, 0], cache[0], cache[1], left, 0, sinks, q_start=start))

    def forward_fp32(self, x: torch.Tensor, left: int = LEFT, right: int = RIGHT, sinks: int = SINKS) -> torch.Tensor:
        def norm(t):
            t = t - t.mean(1, keepdim=True)
            return t / torch.sqrt(t.square().mean(1, keepdim=True) + 1e-5)

        n = x.shape[0]
        h = norm(x) * (1 + self.scale.float()) + self.shift.float()
        q, k, v = (h @ self.qkv_w.t() + self.qkv_b.float()).view(n, 3, HEADS, 64).permute(1, 2, 0, 3)

        def rotate(t):
            return t * self.cos[:n] + torch.cat([-t[..., 32:], t[..., :32]], -1) * self.sin[:n]

        pos = torch.arange(n, device=x.device)
        d = pos[None, :] - pos[:, None]
        seen = (d <= right) & ((d >= -left) | (pos < sinks)[None, :])
        a = (rotate(q) @ rotate(k).transpose(-1, -2) / 8).masked_fill(~seen, -torch.inf).softmax(-1)
        ctx = (a @ v).permute(1, 0, 2).reshape(n, HIDDEN)
        return x + self.gate.float() * (ctx @ self.out_w.t() + self.out_b.float())


def snr_db(ref: torch.Tensor, got: torch.Tensor) -> float:
    return float(10 * torch.log10(ref.double().square().sum() / (ref.double() - got.double()).square().sum()))


def main(frames: int = 3000) -> dict:
    layer = DitLayer(frames)
    x0 = torch.randn(frames, HIDDEN, generator=torch.Generator().manual_seed(1)).cuda()
    x, _ = layer.forward(x0.clone())
    ref = layer.forward_fp32(x0)
    # the same causally, then as a stream: a first chunk, then frame by frame
    causal, _ = layer.forward(x0.clone(), right=0)
    cache, got, first = layer.new_cache(frames), [], min(frames, 200)
    got.append(layer.step(x0[:first].clone(), cache, 0)[0])
    for t in range(first, min(frames, first + 20)):
        got.append(layer.step(x0[t:t + 1].clone(), cache, t)[0])
    F.check_status()
    stream = torch.cat(got)
    n = stream.shape[0]
    result = {"frames": frames,
              "update_snr_db": snr_db(ref - x0, x - x0),                     # the layer's contribution, 8 bits against fp32
              "stream_snr_db": snr_db(causal[:n] - x0[:n], stream - x0[:n])}  # the stream against the whole recording
    print(f"{frames} frames: update within {result['update_snr_db']:.1f} dB of fp32; "
          f"streamed frames within {result['stream_snr_db']:.1f} dB of the whole recording")
    return result


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 3000)
