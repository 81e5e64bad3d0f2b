"""streaming — the time-axis attention of one layer, frame by frame.

The separator's time axis attends over a whole 8 to 11 s chunk.  `StreamingTimeAttention` runs the same kind of layer
(q|k|v projection, per-head norms, rotary positions over time and band, gated attention, output projection, residual)
over a sliding window instead: a first piece goes through `prompt`, later frames through `step` one or a few at a time,
with the keys and values kept in rolling caches of 16 or 4 bits.  Tokens lie as everywhere in the library, [frame][band],
and are read along the time axis in place.

Command line (random weights and input; compares the frame-by-frame result with one pass and times a frame):
    python mbr-cuda-tile_b200/streaming.py --bands 60 --dim 384 --heads 8 --seconds 2 --bits 4
"""
from __future__ import annotations

import argparse

import numpy as np

import cudasep


class StreamingTimeAttention:
    """One layer for `bands` sequences.

    w_qkv [3 * heads * dim_head, dim], w_gate [heads, dim], w_out [dim, heads * dim_head], gamma_q / gamma_k [dim_head]
    fp32; the matrices in fp16 or bf16, on one GPU.  A frame sees itself, `left` frames before it and the first `sinks`
    frames of the stream; `bits` 0 keeps the cache in the matrices' type, 4 in 4 bits.  A stream has up to `max_frames`
    frames (the angle tables are made for as many; 65536 are 10 min 55 s): `prompt` and `step` refuse more and leave the
    stream as it is."""

    def __init__(self, w_qkv, w_gate, w_out, gamma_q, gamma_k, bands, heads, left, sinks=4, bits=0, max_frames=1 << 16):
        import torch

        self.w_qkv, self.w_gate, self.w_out, self.gamma_q, self.gamma_k = w_qkv, w_gate, w_out, gamma_q, gamma_k
        self.bands, self.heads, self.left, self.sinks = bands, heads, left, sinks
        self.dim_head = w_qkv.shape[0] // (3 * heads)
        self.device, self.dtype = w_qkv.device, w_qkv.dtype
        # the first half of each head's pairs turns with the frame, the second with the band
        half = self.dim_head // 2
        self.pairs = [half - half // 2, half // 2]
        self.max_frames = max_frames
        c, s = cudasep.rope_tables(max(max_frames, bands), self.dim_head)
        self.cos, self.sin = (torch.from_numpy(t).to(self.device) for t in (c, s))
        self.band = torch.arange(bands, dtype=torch.int32, device=self.device)
        # a step of n frames needs left + n of them in the ring; 64 is a generous n
        self.cache = cudasep.KVCache.empty(bands, heads, sinks + left + 64, self.dim_head, self.dtype, sinks=sinks,
                                           bits=bits, device=self.device)
        self.frames = 0

    def _project(self, x):
        """x [n, bands, dim] -> q, k, v as [bands, n, heads, dim_head] (q and k normed and rotated), gates
        [bands, n, heads]."""
        import torch

        n, nb, dim = x.shape
        if self.frames + n > self.max_frames:  # positions past the tables would be NaN, in the cache too
            raise ValueError(f"a stream takes up to max_frames = {self.max_frames} frames, got {self.frames} + {n}")
        H, D = self.heads, self.dim_head
        flat = x.reshape(n * nb, dim)
        qkv = cudasep.op_linear(flat, self.w_qkv).view(n, nb, 3 * H, D).transpose(0, 1)
        gates = torch.sigmoid(cudasep.op_linear(flat, self.w_gate).float()).view(n, nb, H).transpose(0, 1).contiguous()
        time = torch.arange(self.frames, self.frames + n, dtype=torch.int32, device=x.device)
        pos = torch.stack([time.expand(nb, n), self.band[:, None].expand(nb, n)], -1)
        q, k = cudasep.op_qk_norm_rope(qkv[:, :, :H], qkv[:, :, H:2 * H], self.gamma_q, self.gamma_k, self.cos, self.sin,
                                       pos, self.pairs)
        return q, k, qkv[:, :, 2 * H:], gates

    def _append(self, k, v):
        import torch

        start = torch.full((self.bands,), self.frames, dtype=torch.int32, device=k.device)
        cudasep.op_cache_append(self.cache, k, v, start)
        self.frames += k.shape[1]

    def attend_prompt(self, x):
        """Heads' outputs [n, bands, heads * dim_head] of the stream's first n frames x [n, bands, dim]."""
        import torch

        if self.frames:
            raise ValueError("prompt is for the start of a stream; use step")
        q, k, v, gates = self._project(x)
        n, nb = x.shape[:2]
        out = torch.empty((n, nb, self.heads, self.dim_head), dtype=x.dtype, device=x.device)
        cudasep.op_window_attention(q, k, v, left=self.left, right=0, sinks=self.sinks, gates=gates,
                                    out=out.transpose(0, 1))
        self._append(k, v)
        return out.view(n, nb, -1)

    def attend_step(self, x):
        """Heads' outputs of the next n frames (n up to 64)."""
        import torch

        n, nb = x.shape[:2]
        if n > self.cache.ring - self.left:
            raise ValueError(f"a step takes up to {self.cache.ring - self.left} frames, got {n}")
        q, k, v, gates = self._project(x)
        self._append(k, v)
        length = torch.full((nb,), self.frames, dtype=torch.int32, device=x.device)
        out = torch.empty((n, nb, self.heads, self.dim_head), dtype=x.dtype, device=x.device)
        cudasep.op_cache_attention(q, self.cache, length, left=self.left, gates=gates, out=out.transpose(0, 1))
        return out.view(n, nb, -1)

    def _finish(self, heads, x):
        y = cudasep.op_linear(heads.reshape(-1, heads.shape[-1]), self.w_out)
        return cudasep.op_add(y, x.reshape(y.shape)).view(x.shape)

    def prompt(self, x):
        """The layer's output for the stream's first frames x [n, bands, dim]."""
        return self._finish(self.attend_prompt(x), x)

    def step(self, x):
        """The layer's output for the next frames."""
        return self._finish(self.attend_step(x), x)


def random_layer(bands, dim, heads, dim_head=64, left=100, sinks=4, bits=0, dtype="bf16", seed=0, device="cuda",
                 max_frames=1 << 16):
    """A layer with seeded random weights."""
    import torch

    rng = np.random.default_rng(seed)
    dt = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]

    def w(*shape, scale):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * scale).to(device)

    inner = heads * dim_head
    return StreamingTimeAttention(w(3 * inner, dim, scale=dim ** -0.5).to(dt), w(heads, dim, scale=dim ** -0.5).to(dt),
                                  w(dim, inner, scale=inner ** -0.5).to(dt), 1 + w(dim_head, scale=0.1),
                                  1 + w(dim_head, scale=0.1), bands, heads, left, sinks, bits,
                                  max_frames)


def main(argv=None):
    import torch

    ap = argparse.ArgumentParser(description="Frame-by-frame time-axis attention of one random layer")
    ap.add_argument("--bands", type=int, default=60)
    ap.add_argument("--dim", type=int, default=384)
    ap.add_argument("--heads", type=int, default=8)
    ap.add_argument("--seconds", type=float, default=2.0, help="100 frames a second")
    ap.add_argument("--left", type=int, default=100, help="frames of history")
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--bits", type=int, default=0, choices=(0, 4))
    ap.add_argument("--dtype", default="bf16", choices=("fp16", "bf16"))
    a = ap.parse_args(argv)
    n = max(2, int(round(100 * a.seconds)))
    x = torch.randn((n, a.bands, a.dim), generator=torch.Generator().manual_seed(1)).cuda()
    make = dict(bands=a.bands, dim=a.dim, heads=a.heads, left=a.left, sinks=a.sinks, bits=a.bits, dtype=a.dtype,
                max_frames=n)
    whole = random_layer(**make)
    x = x.to(whole.dtype)
    want = whole.prompt(x)
    live = random_layer(**make)
    first = n // 2
    got = [live.prompt(x[:first]), live.step(x[first:first + 1])]  # the first step loads the kernels
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got += [live.step(x[i:i + 1]) for i in range(first + 1, n)]
    end.record()
    end.synchronize()
    err = (torch.cat(got).float() - want.float()).abs().max().item()
    print(f"{n} frames, {first} at once and the rest one by one: largest difference from one pass {err:.3e} "
          f"(largest value {want.abs().max().item():.2f}), {start.elapsed_time(end) / max(1, n - first - 1):.3f} ms a frame")


if __name__ == "__main__":
    main()
