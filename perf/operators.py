"""The operators of an 8-bit DiT / encoder layer over long recordings, as measurable cases.

Three operators that a layer of this package's models needs next to its
attention and its fp16 / bf16 projections:

* ``window``: attention over a sliding window of keys with a few first tokens
  that stay visible (sinks), from one query token to a whole recording;
* ``linear``: the projections in 8-bit integers with one scale per token and
  per output channel, the tokens quantised within the call where the caller
  has them in 16 bits, with the epilogues of the 16-bit projections (bias,
  rotate-half RoPE, accumulation into the fp32 residual);
* ``norm``: the step between two blocks -- the norm after a block, its gate,
  the residual scale, and the norm (with the adaLN modulation) before the next
  block -- in one pass.

``own`` selects the form of :func:`run`: False computes the definition with
elementary torch operations in 32 bits, True calls the package.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------- the cases


def listed():
    return [
        # one new frame of a streaming DiT head (12 x 64 heads) against 120 s of
        # cached keys: the last 20 s and the first frames
        dict(name="window_step_b1", op="window", batch=1, q_len=1, k_len=6000, heads=12, kv_heads=12, left=999, right=0,
             sinks=4, start=5800, kv=0, dtype="fp16"),
        # sixteen streams served together, each at its own position in a 10 min
        # cache, query heads sharing key heads
        dict(name="window_step_b16_shared", op="window", batch=16, q_len=1, k_len=30000, heads=16, kv_heads=4, left=4095,
             right=0, sinks=16, start=29990, kv=0, dtype="bf16"),
        # a chunk of 1.5 s appended to a stream (odd sizes throughout)
        dict(name="window_chunk_b3", op="window", batch=3, q_len=77, k_len=2111, heads=12, kv_heads=12, left=411, right=9,
             sinks=3, start=1900, kv=1, dtype="fp16"),
        # one DiT layer of a 120 s window, 10 s either side
        dict(name="window_layer_120s", op="window", batch=1, q_len=6000, k_len=6000, heads=12, kv_heads=12, left=500,
             right=500, sinks=8, start=0, kv=0, dtype="fp16"),
        # one layer of the encoder's heads over a whole 10 min recording
        dict(name="window_layer_600s", op="window", batch=1, q_len=30000, k_len=30000, heads=16, kv_heads=16, left=750,
             right=250, sinks=16, start=0, kv=0, dtype="bf16"),
        # the QKV projection of one frame (weights read once: latency)
        dict(name="linear_row", op="linear", rows=1, k=768, n=2304, x="int8", epi="store", bias=1, length=1, dtype="fp16"),
        # the encoder's QKV projection of a 120 s window, tokens quantised in the call
        dict(name="linear_qkv_120s", op="linear", rows=6000, k=1024, n=3072, x="16bit", epi="store", bias=1, length=6000,
             dtype="fp16"),
        # the DiT's QKV projection with RoPE of a ragged batch (3 x 1367 frames)
        dict(name="linear_rope_ragged", op="linear", rows=4101, k=768, n=2304, x="int8", epi="rope", bias=1, length=1367,
             dtype="bf16"),
        # the second FFN projection into the fp32 residual, eight 120 s windows
        dict(name="linear_ffn_accumulate", op="linear", rows=48000, k=4096, n=1024, x="16bit", epi="accumulate", bias=0,
             length=6000, dtype="fp16"),
        # one frame through a DiT block boundary (gate, adaLN)
        dict(name="norm_row", op="norm", rows=1, c=768, length=1, stream="fp32", post="none", pre="layer", gate="window",
             mod=1, alpha=1.0, dtype="fp16"),
        # DiT block boundary of a 120 s window
        dict(name="norm_dit_120s", op="norm", rows=6000, c=768, length=6000, stream="fp32", post="none", pre="layer",
             gate="window", mod=1, alpha=1.0, dtype="fp16"),
        # sandwich norms with a layer scale and a residual scale, ragged rows, 16-bit stream
        dict(name="norm_sandwich_ragged", op="norm", rows=29777, c=1160, length=29777, stream="bf16", post="rms", pre="rms",
             gate="layer", mod=0, alpha=0.5, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    op = rng.choice(["window", "linear", "norm"])
    if op == "window":
        heads = rng.choice([4, 8, 12, 16])
        kv_heads = heads // rng.choice([1, 1, 2, 4])
        step = rng.random() < 0.35
        q_len = rng.choice([1, 1, 1, 2, 3, 7]) if step else _log(rng, 8, 30000)
        batch = rng.randint(1, 16) if step else max(1, min(8, 30000 // q_len // rng.randint(1, 8)))
        right = 0 if step or rng.random() < 0.4 else _log(rng, 1, 400)
        k_len = _log(rng, max(64, q_len), 30000) if q_len < 20000 else q_len
        if batch * k_len > 400000:
            batch = max(1, 400000 // k_len)
        return dict(op="window", batch=batch, q_len=q_len, k_len=k_len, heads=heads, kv_heads=kv_heads,
                    left=_log(rng, 16, 4096 if step else 800), right=right, sinks=rng.choice([0, 1, 4, 16, rng.randint(2, 64)]),
                    start=rng.randint(0, k_len - q_len), kv=rng.choice([0, 1]), dtype=dtype)
    if op == "linear":
        epi = rng.choice(["store", "rope", "accumulate"])
        rows = _log(rng, 1, 24000)
        heads = rng.randint(2, 16)
        k = 16 * _log(rng, 8, 256)
        n = 3 * 64 * heads if epi == "rope" else 8 * _log(rng, 16, 512)
        return dict(op="linear", rows=rows, k=k, n=n, x=rng.choice(["int8", "16bit"]), epi=epi, bias=rng.choice([0, 1]),
                    length=max(1, rows // rng.randint(1, 4)), dtype=dtype)
    rows, c = _log(rng, 1, 30000), 8 * _log(rng, 8, 512)
    if rows * c > 40_000_000:
        rows = 40_000_000 // c
    return dict(op="norm", rows=rows, c=c, length=max(1, rows // rng.randint(1, 6)), stream=rng.choice(["fp32", dtype]),
                post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["layer", "rms"]),
                gate=rng.choice(["none", "layer", "window"]), mod=rng.choice([0, 1]), alpha=rng.choice([1.0, 0.5]),
                dtype=dtype)


# ---------------------------------------------------------------- inputs


def _positions(case):
    """(position of each window's first query, valid keys of each window), host lists."""
    starts, lens = [], []
    for b in range(case["batch"]):
        # streams of a batch are not at the same position; the last key a query may see exists
        s = max(0, case["start"] - 53 * b)
        starts.append(s)
        lens.append(min(case["k_len"], s + case["q_len"] + 31 * b % 17) if case["kv"] else case["k_len"])
    return starts, lens


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[case["dtype"]]

    def rnd(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    s = {"case": case, "op": case["op"]}
    if case["op"] == "window":
        B, Lq, Lk, H, Hk = (case[x] for x in ("batch", "q_len", "k_len", "heads", "kv_heads"))
        if Lq == Lk and H == Hk and case["start"] == 0:
            # the rotated qkv of a QKV projection: q, k and v are column blocks of its rows
            qkv = rnd(B, Lq, 3, H, 64)
            s["q"], s["k"], s["v"] = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        else:
            s["q"], s["k"], s["v"] = rnd(B, Lq, H, 64), rnd(B, Lk, Hk, 64), rnd(B, Lk, Hk, 64)
        starts, lens = _positions(case)
        s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=DEV) if case["kv"] else None
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        # activations: a few channels carry most of the range, tokens differ in size
        x = torch.randn(m, k, generator=g, device=DEV)
        x *= torch.exp(0.8 * torch.randn(k, generator=g, device=DEV))[None, :]
        x *= torch.exp(0.3 * torch.randn(m, generator=g, device=DEV))[:, None]
        w = torch.randn(n, k, generator=g, device=DEV) * 0.02 * torch.exp(0.3 * torch.randn(n, generator=g, device=DEV))[:, None]
        ws = w.abs().amax(1) / 127
        s["w"], s["ws"] = torch.round(w / ws[:, None]).to(torch.int8), ws
        if case["x"] == "int8":
            xs = x.abs().amax(1) / 127
            s["x"], s["xs"] = torch.round(x / xs[:, None]).to(torch.int8), xs
        else:
            s["x"] = x.to(dt)
        s["b"] = rnd(n, scale=0.1) if case["bias"] else None
        if case["epi"] == "rope":
            s["cos"], s["sin"] = _rope_tables(max(1, min(case["length"], m)))
        if case["epi"] == "accumulate":
            s["res"] = torch.randn(m, n, generator=g, device=DEV)
    else:
        r, c = case["rows"], case["c"]
        nw = -(-r // case["length"])
        s["x"] = rnd(r, c, scale=4.0, dtype=DT[case["stream"]])
        s["y"] = rnd(r, c, scale=2.0) + rnd(r, 1)
        s["gate"] = {"none": None, "layer": rnd(c, scale=0.3), "window": rnd(nw, c, scale=0.3)}[case["gate"]]
        s["post_w"] = None if case["post"] == "none" else 1 + rnd(c, scale=0.1)
        s["post_b"] = rnd(c, scale=0.1) if case["post"] == "layer" else None
        s["w"] = 1 + rnd(c, scale=0.1)
        s["b"] = rnd(c, scale=0.1) if case["pre"] == "layer" else None
        s["scale"], s["shift"] = (rnd(nw, c, scale=0.2), rnd(nw, c, scale=0.2)) if case["mod"] else (None, None)
        s["x_out"] = torch.empty_like(s["x"])
    return s


def _rope_tables(length):
    f = torch.outer(torch.arange(length, dtype=torch.float32), 10000.0 ** (-torch.arange(32, dtype=torch.float32) / 32))
    f = torch.cat([f, f], -1)
    return f.cos().contiguous().to(DEV), f.sin().contiguous().to(DEV)


# ---------------------------------------------------------------- one pass


def run(s):
    return {"window": _window, "linear": _linear, "norm": _norm}[s["op"]](s)


def _window(s):
    c = s["case"]
    if own:
        import fastdialoguesidon_b200 as F

        return F.window_attention(s["q"], s["k"], s["v"], c["left"], c["right"], c["sinks"], q_start=s["q_start"],
                                  kv_len=s["kv_len"])
    return _plain_window(s["q"], s["k"], s["v"], c["left"], c["right"], c["sinks"], s["q_start"], s["kv_len"])


def _plain_window(q, k, v, left, right, sinks, q_start, kv_len):
    """Queries in blocks of T; each block against its stretch of keys and the sinks."""
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    left, right, sinks = min(left, Lk), min(right, Lk), min(sinks, Lk)
    T = min(128, Lq)
    nb = -(-Lq // T)
    dev = q.device
    qf = torch.zeros(B, nb * T, H, D, device=dev)
    qf[:, :Lq] = q.float()
    qf = qf.view(B, nb, T, Hk, H // Hk, D).permute(0, 1, 3, 4, 2, 5).reshape(B, nb, Hk, H // Hk * T, D)
    pos = q_start.long()[:, None, None] + torch.arange(nb * T, device=dev).view(1, nb, T)     # [B, nb, T]
    n_valid = kv_len.long() if kv_len is not None else torch.full((B,), Lk, device=dev)
    near = pos[:, :, :1] - left + torch.arange(T + left + right, device=dev)                 # [B, nb, T + left + right]
    first = torch.arange(sinks, device=dev).expand(B, nb, sinks)
    j = torch.cat([near, first], -1)[:, :, None, :]                                          # key positions
    p = pos[..., None]
    in_near = torch.arange(j.shape[-1], device=dev) < T + left + right
    seen = torch.where(in_near, (j >= p - left) & (j <= p + right), j < p - left)
    seen = seen & (j >= 0) & (j < n_valid[:, None, None, None])                              # [B, nb, T, keys]
    rows = torch.arange(B, device=dev)[:, None, None]
    jc = j[:, :, 0].clamp(0, Lk - 1)
    kb = k[rows, jc].float().permute(0, 1, 3, 2, 4)                                          # [B, nb, Hk, keys, D]
    vb = v[rows, jc].float().permute(0, 1, 3, 2, 4)
    seen = seen[:, :, None, None].expand(B, nb, Hk, H // Hk, T, j.shape[-1]).reshape(B, nb, Hk, -1, j.shape[-1])
    a = torch.where(seen, qf @ kb.transpose(-1, -2) / math.sqrt(D), -torch.inf)
    m = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(torch.isfinite(m), m, 0))
    o = (e @ vb) / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.view(B, nb, Hk, H // Hk, T, D).permute(0, 1, 4, 2, 3, 5).reshape(B, nb * T, H, D)
    return o[:, :Lq].to(q.dtype)


def _linear(s):
    c = s["case"]
    dt = DT[c["dtype"]]
    if own:
        import fastdialoguesidon_b200 as F

        x, xs = (s["x"], s["xs"]) if c["x"] == "int8" else F.quantize_rows(s["x"])
        if c["epi"] == "rope":
            return F.linear_int8_rope(x, xs, s["w"], s["ws"], s["b"], s["cos"], s["sin"], c["length"], c["n"] // 192,
                                      dtype=dt)
        if c["epi"] == "accumulate":
            F.accumulate_int8(s["res"], x, xs, s["w"], s["ws"], s["b"])
            return s["res"]
        return F.linear_int8(x, xs, s["w"], s["ws"], s["b"], dtype=dt)
    x = s["x"].float()
    if c["x"] == "int8":
        xs = s["xs"]
    else:
        big = x.abs().amax(1)
        xs = big / 127
        x = torch.round(x * (torch.full_like(big, 127) / big)[:, None])  # (a number / tensor is its reciprocal times it)
    y = (x @ s["w"].float().t()) * (xs[:, None] * s["ws"][None, :])
    if s["b"] is not None:
        y = y + s["b"].float()
    if c["epi"] == "accumulate":
        s["res"].add_(y)
        return s["res"]
    if c["epi"] == "rope":
        t = torch.arange(c["rows"], device=y.device) % c["length"]
        cos, sin = s["cos"][t, None, :32], s["sin"][t, None, :32]
        n3 = c["n"] // 3
        h = y[:, :2 * n3].reshape(c["rows"], -1, 2, 32)
        a, b = h[:, :, 0], h[:, :, 1]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], 2).reshape(c["rows"], 2 * n3)
        y = torch.cat([rot, y[:, 2 * n3:]], 1)
    return y.to(dt)


def _norm(s):
    c = s["case"]
    if own:
        import fastdialoguesidon_b200 as F

        x, h = F.residual_norm(s["x"], s["y"], gate=s["gate"], residual_scale=c["alpha"], post=c["post"],
                               post_weight=s["post_w"], post_bias=s["post_b"], norm=c["pre"], weight=s["w"], bias=s["b"],
                               scale=s["scale"], shift=s["shift"], length=c["length"], residual_out=s["x_out"])
        return {"x": x, "h": h}
    win = torch.arange(c["rows"], device=s["x"].device) // c["length"]
    y = s["y"].float()
    if c["post"] != "none":
        y = _unit(y, c["post"]) * s["post_w"].float()
        if s["post_b"] is not None:
            y = y + s["post_b"].float()
    if c["gate"] == "window":
        y = y * s["gate"].float()[win]
    elif c["gate"] == "layer":
        y = y * s["gate"].float()
    x = s["x"].float() * c["alpha"] + y
    h = _unit(x, c["pre"]) * s["w"].float()
    if s["b"] is not None:
        h = h + s["b"].float()
    if c["mod"]:
        h = h * (1 + s["scale"].float()[win]) + s["shift"].float()[win]
    s["x_out"].copy_(x)
    return {"x": s["x_out"], "h": h.to(DT[c["dtype"]])}


def _unit(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "window":
        B, Lq, Lk, H, Hk = (case[x] for x in ("batch", "q_len", "k_len", "heads", "kv_heads"))
        starts, lens = _positions(case)
        pairs = keys = 0
        for s0, n in zip(starts, lens):
            p = np.arange(s0, s0 + Lq)
            hi = np.minimum(p + case["right"] + 1, n)
            lo = np.maximum(p - case["left"], 0)
            pairs += int(np.maximum(hi - lo, 0).sum() + np.minimum(np.minimum(case["sinks"], lo), np.maximum(hi, 0)).sum())
            keys += int(max(0, hi[-1] - lo[0]) + min(case["sinks"], lo[0], n))
        return {"bytes": 2 * 64 * (2 * B * Lq * H + 2 * keys * Hk), "flops": 4 * 64 * H * pairs}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        x = m * k * 2 if case["x"] == "16bit" else m * k + 4 * m
        out = 8 * m * n if case["epi"] == "accumulate" else 2 * m * n
        rope = 2 * 4 * 32 * min(case["length"], m) if case["epi"] == "rope" else 0
        return {"bytes": x + n * k + 4 * n + (2 * n if case["bias"] else 0) + out + rope, "flops": 2 * m * n * k}
    r, c = case["rows"], case["c"]
    nw = -(-r // case["length"])
    stream = 4 if case["stream"] == "fp32" else 2
    vec = (1 + (case["pre"] == "layer") + (case["post"] != "none") + (case["post"] == "layer") + (case["gate"] == "layer")
           + nw * (case["gate"] == "window") + 2 * nw * case["mod"])
    return {"bytes": r * c * (2 * stream + 4) + 2 * c * vec, "flops": 14 * r * c}


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "linear": _exact_linear, "norm": _exact_norm}[case["op"]](case, s)


def _exact_window(case, s):
    starts, lens = _positions(case)
    B, Lq, H = case["batch"], case["q_len"], case["heads"]
    G = H // case["kv_heads"]
    out = torch.zeros(B, Lq, H, 64, dtype=torch.float64, device=DEV)
    step = 512
    for b in range(B):
        for i0 in range(0, Lq, step):
            i1 = min(Lq, i0 + step)
            p = torch.arange(starts[b] + i0, starts[b] + i1, device=DEV)
            lo, hi = max(0, starts[b] + i0 - case["left"]), min(lens[b], starts[b] + i1 + case["right"])
            sinks = min(case["sinks"], lo, lens[b])
            ids = torch.cat([torch.arange(sinks, device=DEV), torch.arange(lo, max(lo, hi), device=DEV)])
            if ids.numel() == 0:
                continue
            ok = (ids[None] <= p[:, None] + case["right"]) & ((ids[None] >= p[:, None] - case["left"])
                                                                     | (ids[None] < case["sinks"]))
            for h in range(H):
                z = s["q"][b, i0:i1, h].double() @ s["k"][b, ids, h // G].double().t() / 8.0
                z.masked_fill_(~ok, -math.inf)
                a = torch.softmax(z, -1)
                a[~ok.any(1)] = 0.0
                out[b, i0:i1, h] = a @ s["v"][b, ids, h // G].double()
    return out


def _exact_linear(case, s):
    x = s["x"].double()
    if case["x"] == "int8":
        xs = s["xs"].double()
    else:
        big = s["x"].float().abs().amax(1, keepdim=True)
        x = torch.round(s["x"].float() * (torch.full_like(big, 127) / big)).double()
        xs = big[:, 0].double() / 127
    y = torch.einsum("mk,nk->mn", x, s["w"].double()).mul_(xs[:, None]).mul_(s["ws"].double()[None])
    if s["b"] is not None:
        y += s["b"].double()
    if case["epi"] == "accumulate":
        return s["res"].double() + y
    if case["epi"] == "rope":
        hid = case["n"] // 3
        t = torch.arange(case["rows"], device=DEV).remainder(case["length"])
        ang_c, ang_s = s["cos"].double()[t], s["sin"].double()[t]
        for col in range(0, 2 * hid, 64):
            u = y[:, col:col + 64].clone()
            y[:, col:col + 64] = u * ang_c + torch.cat([-u[:, 32:], u[:, :32]], 1) * ang_s
    return y


def _exact_norm(case, s):
    def normed(t, kind, w, b):
        if kind == "layer":
            mu = t.mean(1, keepdim=True)
            t = (t - mu) / torch.sqrt(((t - mu) ** 2).mean(1, keepdim=True) + 1e-5)
        else:
            t = t / torch.sqrt((t ** 2).mean(1, keepdim=True) + 1e-5)
        t = t * w.double()
        return t if b is None else t + b.double()

    of = torch.div(torch.arange(case["rows"], device=DEV), case["length"], rounding_mode="floor")
    z = s["y"].double()
    if case["post"] != "none":
        z = normed(z, case["post"], s["post_w"], s["post_b"])
    if case["gate"] != "none":
        z = z * (s["gate"].double() if case["gate"] == "layer" else s["gate"].double()[of])
    x = case["alpha"] * s["x"].double() + z
    h = normed(x, case["pre"], s["w"], s["b"])
    if case["mod"]:
        h = h * (1.0 + s["scale"].double()[of]) + s["shift"].double()[of]
    return {"x": x, "h": h}
