"""64-bit CPU references of the streaming-attention operators and the error bounds of their tests.

Bounds.  u is half a unit in the last place relative to the value (fp32 2^-24, fp16 2^-11, bf16 2^-8).
 - Norm and rotation: about ten fp32 operations on values bounded by |y0| + |y1| and one rounding of the result:
   (16 * 2^-24) (|y0| + |y1|) + u |z|.
 - Attention: a score carries at most (D + 8) 2^-24 S (S = scale sum |q_d k_d|) of rounding; that changes weights by
   twice as much, relatively; each weight and the running sums carry (N + 64) 2^-24 over N keys; a 16-bit weight
   carries u; the result is rounded once.  With A = sum_j w_j |v_j|:
   ((2 (D + 8) S + N + 64) 2^-24 + (u where weights are 16-bit)) A + u |out|, fp16 weights below its normal range
   adding at most 2^-25 each, N 2^-25 max |v|.
"""
import numpy as np
import torch

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rotate(x, gamma, cos, sin, pos, pairs, eps):
    """(result, bound) of the norm and rotation of x [S, N, H, D] in 64 bits."""
    S, N, H, D = x.shape
    xd = x.double()
    y = xd / (xd.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if gamma is not None:
        y = y * gamma.double()
    z = y.clone()
    size = y.abs()
    at = 0
    for a, n in enumerate(pairs):
        for i in range(at, at + n):
            p = pos[..., a].long()
            ok = (p >= 0) & (p < cos.shape[0])
            c = torch.where(ok, cos.double()[p.clamp(0, cos.shape[0] - 1), i], torch.nan)[..., None]
            s = torch.where(ok, sin.double()[p.clamp(0, cos.shape[0] - 1), i], torch.nan)[..., None]
            y0, y1 = y[..., 2 * i], y[..., 2 * i + 1]
            z[..., 2 * i], z[..., 2 * i + 1] = y0 * c - y1 * s, y0 * s + y1 * c
            size[..., 2 * i] = size[..., 2 * i + 1] = y0.abs() + y1.abs()
        at += n
    u = HALF_ULP[x.dtype]
    return z, (D / 2 + 16) * 2.0 ** -24 * size + u * 1.01 * z.abs() + TINY[x.dtype]


def attention(q, k, v, see, scale, gates):
    """(result, bound) for one sequence: q [N, H, D], k, v [M, G, D], see [N, M] truth values, gates [N, H] or None.
    Keys that a query does not see take no part."""
    N, H, D = q.shape
    M, G = k.shape[0], k.shape[1]
    out, bound = torch.zeros(N, H, D, dtype=torch.float64), torch.zeros(N, H, D, dtype=torch.float64)
    u = HALF_ULP[q.dtype]
    soft = 0.0 if q.dtype == torch.float32 else u
    for h in range(H):
        kd, vd = k[:, h * G // H].double(), v[:, h * G // H].double()
        for i in range(N):
            js = torch.nonzero(see[i]).flatten()
            if not len(js):
                continue
            qd = q[i, h].double()
            kk, vv = kd[js], vd[js]
            s = scale * (kk @ qd)
            size = scale * (kk.abs() @ qd.abs()).max()
            w = torch.softmax(s, 0)
            g = 1.0 if gates is None else float(gates[i, h])
            o, A = w @ vv, w @ vv.abs()
            n = len(js)
            b = ((2 * (D + 8) * size + n + 64) * 2.0 ** -24 + soft) * A
            if q.dtype == torch.float16:
                b = b + n * 2.0 ** -25 * vv.abs().max()
            out[i, h] = g * o
            bound[i, h] = abs(g) * (b + u * o.abs()) * 1.01 + TINY[q.dtype]
    return out, bound


def visible(p, m, left, right, sinks, held_from=0):
    """[len(p), m] truth values: which keys 0..m-1 queries at positions p see."""
    p = np.asarray(p, np.int64).reshape(-1, 1)
    j = np.arange(m, dtype=np.int64).reshape(1, -1)
    see = np.ones((p.shape[0], m), bool)
    if right >= 0:
        see &= j <= p + right
    if left >= 0:
        see &= (j >= p - left) | (j < sinks)
    see &= (j < sinks) | (j >= held_from)
    return torch.from_numpy(see)


def four_bits(x):
    """(codes, step, offset, values) of x [..., D] in 4 bits per 32 channels, by numpy in fp32 with the roundings of the
    definition."""
    T = x.dtype
    g = x.float().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((hi - lo) * np.float32(1.0 / 15.0)).to(T).float()
    mid = (lo + 8 * step).to(T).float()
    inv = torch.where(step > 0, 1.0 / step, torch.zeros_like(step))
    code = (torch.round((g - mid) * inv) + 8).clamp(0, 15)
    values = (mid + step * (code - 8)).to(T).flatten(-2)
    bad = ~(torch.isfinite(g).all(-1, keepdim=True) & torch.isfinite(hi - lo)).expand_as(g).flatten(-2)
    values[bad] = torch.nan
    return code.flatten(-2), step[..., 0], mid[..., 0], values
