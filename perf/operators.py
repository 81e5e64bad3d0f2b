"""Cases for the streaming-attention operators: inputs, plain forms, 64-bit definitions and work counts.

Four operators, each reached through the Python binding of the library:

  rotate   queries and keys normalised per head and rotated by their positions on several axes
  append   new keys and values written to a rolling cache (first positions kept, the rest in a ring) and read back
  prompt   attention with a sliding window and visible first tokens, many queries at once
  step     the same attention for the newest one or few tokens over the rolling cache

Sizes are those of the separation model: 60 bands, each a sequence of frames at 100 frames a second; 8 or 16 heads of
64 (8 of 32 in the fp32 configuration); 801, 1101 or 1301 frames in a chunk, 6001 in a minute.
"""
import math
import os
import sys

import torch

own = False  # set by the measuring program: False runs the plain forms, True the library's operators

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
GROUP = 32  # channels that share a step and an offset in a 4-bit cache


def listed():
    return [
        # one new frame of one stream (60 bands): what runs per layer and frame while audio comes in
        dict(name="rotate_frame_bf16", op="rotate", dtype="bf16", seqs=60, tokens=1, heads=8, kv_heads=8, dim=64,
             axes=1, packed=True),
        # a whole 8 s chunk, read in place from the packed q|k|v of the projection, time and band axes
        dict(name="rotate_chunk_fp16", op="rotate", dtype="fp16", seqs=60, tokens=801, heads=8, kv_heads=8, dim=64,
             axes=2, packed=True),
        # the fp32 configuration with fewer key heads, an odd length and a third axis (channel)
        dict(name="rotate_odd_fp32", op="rotate", dtype="fp32", seqs=60, tokens=333, heads=8, kv_heads=2, dim=32,
             axes=3, packed=False),
        # one new frame into a 16-bit cache of about 10 s
        dict(name="append_frame_fp16", op="append", dtype="fp16", bits=16, seqs=60, tokens=1, kv_heads=8, dim=64,
             sinks=4, ring=1020, seen=1777),
        # the chunk that a stream starts with, into 4-bit caches that keep its last 5 s
        dict(name="append_chunk_4bit_bf16", op="append", dtype="bf16", bits=4, seqs=60, tokens=801, kv_heads=8, dim=64,
             sinks=4, ring=500, seen=0),
        # a short first piece of one channel in fp32: the smallest prompt
        dict(name="prompt_short_fp32", op="prompt", dtype="fp32", seqs=4, q_tokens=50, kv_tokens=50, heads=8,
             kv_heads=8, dim=32, left=-1, right=2, sinks=1, ragged=False),
        # an 8 s chunk, each frame seeing 2.5 s back and 0.2 s ahead: the ordinary prompt
        dict(name="prompt_chunk_fp16", op="prompt", dtype="fp16", seqs=60, q_tokens=801, kv_tokens=801, heads=8,
             kv_heads=8, dim=64, left=250, right=20, sinks=4, ragged=False),
        # pieces of different lengths (none and one among them) continued after what was seen before, shared key heads
        dict(name="prompt_ragged_bf16", op="prompt", dtype="bf16", seqs=12, q_tokens=777, kv_tokens=1301, heads=16,
             kv_heads=4, dim=128, left=400, right=0, sinks=7, ragged=True),
        # a minute of audio in one pass, 10 s of history: the long prompt
        dict(name="prompt_minute_bf16", op="prompt", dtype="bf16", seqs=4, q_tokens=6001, kv_tokens=6001, heads=8,
             kv_heads=8, dim=64, left=1023, right=0, sinks=16, ragged=False),
        # one frame of one stream over about 10 s of cache: what bounds the delay of a live stream
        dict(name="step_frame_fp16", op="step", dtype="fp16", bits=16, seqs=60, tokens=1, heads=8, kv_heads=8, dim=64,
             sinks=4, ring=1020, seen=1777, left=1000, ragged=False),
        # sixteen live streams on one GPU with 4-bit caches, at different times of their tracks
        dict(name="step_streams_4bit_bf16", op="step", dtype="bf16", bits=4, seqs=960, tokens=1, heads=8, kv_heads=8,
             dim=64, sinks=4, ring=1500, seen=2222, left=-1, ragged=True),
        # three frames at once over an 11 min recording kept whole, few sequences, shared key heads
        dict(name="step_long_bf16", op="step", dtype="bf16", bits=16, seqs=2, tokens=3, heads=16, kv_heads=4, dim=64,
             sinks=0, ring=66001, seen=66001, left=-1, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fits(case):
    """No more work than the largest listed case of the kind, in the operator and in its plain form."""
    w = work(case)
    flops = 4.6e10 if case["dtype"] != "fp32" else 4e9
    scores = case["seqs"] * case["heads"] * case["q_tokens"] * case["kv_tokens"] if case["op"] == "prompt" else 0
    slots = case["seqs"] * case["kv_heads"] * case["ring"] * case["dim"] if case["op"] == "step" else 0
    return w["flops"] <= flops and w["bytes"] <= 6.1e8 and scores <= 1.15e9 and slots <= 7.3e8


def draw(rng):
    op = rng.choice(["rotate", "append", "prompt", "step"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dim = rng.choice([32, 64, 64, 128])
    bits = rng.choice([16, 4])
    dtype = rng.choice(["fp16", "bf16"] if op in ("append", "step") else ["fp32", "fp16", "bf16"])
    if op == "rotate":
        case = dict(op=op, dtype=dtype, seqs=_log(rng, 1, 60), tokens=_log(rng, 1, 1301), heads=heads,
                    kv_heads=kv_heads, dim=rng.choice([32, 64]), axes=rng.choice([1, 2, 3]),
                    packed=rng.choice([False, True]))
    elif op == "append":
        case = dict(op=op, dtype=dtype, bits=bits, seqs=_log(rng, 1, 60), tokens=_log(rng, 1, 801), kv_heads=kv_heads,
                    dim=rng.choice([32, 64]), sinks=rng.choice([0, 1, 4, 17]), ring=_log(rng, 65, 1500),
                    seen=_log(rng, 1, 5000) - 1)
    elif op == "prompt":
        q_tokens = _log(rng, 1, 6001)
        case = dict(op=op, dtype=dtype, seqs=_log(rng, 1, 60), q_tokens=q_tokens,
                    kv_tokens=q_tokens + rng.choice([0, 1]) * rng.randrange(0, 1000), heads=heads, kv_heads=kv_heads,
                    dim=rng.choice([32, 64]) if dtype == "fp32" else dim, left=rng.choice([-1, _log(rng, 1, 1500)]),
                    right=rng.choice([0, 0, _log(rng, 1, 60), -1]), sinks=rng.choice([0, 1, 4, 17, 70]),
                    ragged=rng.choice([False, True]))
    else:
        ring = _log(rng, 100, 66001)
        case = dict(op=op, dtype=dtype, bits=bits, seqs=_log(rng, 1, 960), tokens=rng.choice([1, 1, 2, 5, 16]),
                    heads=heads, kv_heads=kv_heads, dim=dim, sinks=rng.choice([0, 1, 4, 17]), ring=ring,
                    seen=_log(rng, 20, 2 * ring), left=rng.choice([-1, _log(rng, 1, 2000)]),
                    ragged=rng.choice([False, True]))
    while not _fits(case):
        if case["seqs"] > 1:
            case["seqs"] = case["seqs"] * 3 // 4
        else:
            for name in ("tokens", "q_tokens", "kv_tokens"):
                if name in case:
                    case[name] = max(1, case[name] * 3 // 4)
    return case


# ---------------------------------------------------------------------------
# lengths (part of the case, the same for every seed)
# ---------------------------------------------------------------------------
def _share(i):
    """0, 1 and values between, in an order without a pattern."""
    return ((i * 67 + 100) % 101) / 100.0


def _prompt_lengths(case):
    """(queries, keys) of each sequence: keys end with the queries' own tokens."""
    n, m = case["q_tokens"], case["kv_tokens"]
    if not case["ragged"]:
        return [(n, m)] * case["seqs"]
    out = []
    for i in range(case["seqs"]):
        q = (n, 0, 1)[i] if i < 3 else int(round(n * _share(i)))
        out.append((q, min(m, q + int(round((m - n) * _share(i + 5))))))
    return out


def _seen(case, i):
    """Tokens that sequence i had before this call."""
    if not case.get("ragged"):
        return case["seen"]
    return (case["seen"], 0)[i] if i < 2 else int(round(case["seen"] * _share(i)))


def _pairs(dim, axes):
    """Rotated pairs on each axis: all on one, or half on the first and the rest shared by the others (what does not
    divide stays unrotated)."""
    half = dim // 2
    if axes == 1:
        return [half]
    rest = half // 2
    first = half - rest
    each = [rest // (axes - 1)] * (axes - 1)
    return [first] + each


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rand(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _qk_like(gen, shape, dtype):
    """Normed queries or keys: unit mean square with a few strong channels."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    x[..., :2] *= 2.0
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000 + int(seed))
    dt = DTYPES[case["dtype"]]
    s = dict(case=dict(case))
    S, D = case["seqs"], case["dim"]
    if case["op"] == "rotate":
        N, H, G = case["tokens"], case["heads"], case["kv_heads"]
        if case["packed"]:  # the projection's q|k|v rows, token-major over (frame, band)
            x = _rand(gen, (N, S, H + 2 * G, D), dt, 1.5).transpose(0, 1)
            s["q"], s["k"] = x[:, :, :H], x[:, :, H:H + G]
        else:
            s["q"], s["k"] = _rand(gen, (S, N, H, D), dt, 1.5), _rand(gen, (S, N, G, D), dt, 1.5)
        s["gamma_q"] = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
        s["gamma_k"] = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
        rows = 2048
        inv = 10000.0 ** (-2.0 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
        ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        start = torch.randint(0, rows - N, (1,), generator=gen, device="cuda")
        time = (start + torch.arange(N, device="cuda"))[None, :].expand(S, N)
        band = torch.arange(S, device="cuda")[:, None].expand(S, N)
        s["pos"] = torch.stack([time, band, band % 2][:case["axes"]], dim=-1).to(torch.int32).contiguous()
        s["pairs"] = _pairs(D, case["axes"])
        s["axis"] = torch.tensor([a for a, n in enumerate(s["pairs"]) for _ in range(n)] +
                                 [0] * (D // 2 - sum(s["pairs"])), device="cuda")  # the axis of each pair
        return s
    if case["op"] == "prompt":
        N, M, H, G = case["q_tokens"], case["kv_tokens"], case["heads"], case["kv_heads"]
        s["q"] = _qk_like(gen, (S, N, H, D), dt)
        s["k"] = _qk_like(gen, (S, M, G, D), dt)
        s["v"] = _rand(gen, (S, M, G, D), dt)
        s["gates"] = torch.rand((S, N, H), generator=gen, device="cuda")
        s["q_len"] = s["kv_len"] = None
        if case["ragged"]:
            n = torch.tensor(_prompt_lengths(case), dtype=torch.int32, device="cuda")
            s["q_len"], s["kv_len"] = n[:, 0].contiguous(), n[:, 1].contiguous()
        return s
    # the cache: what earlier calls left there
    G, slots = case["kv_heads"], case["sinks"] + case["ring"]
    if case["bits"] == 16:
        s["ck"], s["cv"] = _qk_like(gen, (S, G, slots, D), dt), _rand(gen, (S, G, slots, D), dt)
        s["ck_scale"] = s["cv_scale"] = None
    else:
        for name in ("ck", "cv"):
            s[name] = torch.randint(0, 256, (S, G, slots, D // 2), generator=gen, device="cuda", dtype=torch.uint8)
            step = 0.2 + 0.15 * torch.rand((S, G, slots, D // GROUP, 1), generator=gen, device="cuda")
            mid = 0.3 * torch.randn((S, G, slots, D // GROUP, 1), generator=gen, device="cuda")
            s[name + "_scale"] = torch.cat([step, mid], dim=-1).to(dt)
    N = case["tokens"]
    seen = [_seen(case, i) for i in range(S)]
    if case["op"] == "append":
        s["k"], s["v"] = _qk_like(gen, (S, N, G, D), dt), _rand(gen, (S, N, G, D), dt)
        s["pos"] = torch.tensor(seen, dtype=torch.int32, device="cuda")
    else:
        s["q"] = _qk_like(gen, (S, N, case["heads"], D), dt)
        s["gates"] = torch.rand((S, N, case["heads"]), generator=gen, device="cuda")
        s["length"] = torch.tensor([n + N for n in seen], dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------
# the library's operators
# ---------------------------------------------------------------------------
def _lib():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mbr-cuda-tile_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import cudasep

    return cudasep


def _run_own(s):
    lib, case = sys.modules.get("cudasep") or _lib(), s["case"]
    if case["op"] == "rotate":
        q, k = lib.op_qk_norm_rope(s["q"], s["k"], s["gamma_q"], s["gamma_k"], s["cos"], s["sin"], s["pos"], s["pairs"],
                                   eps=EPS)
        return {"q": q, "k": k}
    if case["op"] == "prompt":
        return {"out": lib.op_window_attention(s["q"], s["k"], s["v"], left=case["left"], right=case["right"],
                                               sinks=case["sinks"], q_len=s["q_len"], kv_len=s["kv_len"],
                                               gates=s["gates"])}
    cache = lib.KVCache(s["ck"], s["cv"], s["ck_scale"], s["cv_scale"], sinks=case["sinks"])
    if case["op"] == "append":
        lib.op_cache_append(cache, s["k"], s["v"], s["pos"])
        k, v = lib.op_cache_read(cache, s["pos"], case["tokens"])
        return {"k": k, "v": v}
    return {"out": lib.op_cache_attention(s["q"], cache, s["length"], left=case["left"], right=0, gates=s["gates"])}


# ---------------------------------------------------------------------------
# plain forms (fp32, elementary torch operations)
# ---------------------------------------------------------------------------
def _plain_rotate_one(x, gamma, cos, sin, rotated):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma
    y0, y1 = y[..., 0::2], y[..., 1::2]
    z0, z1 = y0 * cos - y1 * sin, y0 * sin + y1 * cos
    z = torch.stack([torch.where(rotated, z0, y0), torch.where(rotated, z1, y1)], dim=-1)
    return z.flatten(-2).to(x.dtype)


def _plain_rotate(s):
    D, pairs = s["case"]["dim"], s["pairs"]
    col = torch.arange(D // 2, device="cuda")
    p = s["pos"].long()[..., s["axis"]]  # [S, N, D/2]
    cos, sin = s["cos"][p, col][:, :, None], s["sin"][p, col][:, :, None]
    rotated = col < sum(pairs)
    return {"q": _plain_rotate_one(s["q"], s["gamma_q"], cos, sin, rotated),
            "k": _plain_rotate_one(s["k"], s["gamma_k"], cos, sin, rotated)}


def _plain_attend(q, k, v, visible, gates, dtype):
    """q [S,N,H,D], k and v [S,G,M,D] in 32 bits, visible [S or 1,N,M]."""
    S, N, H, D = q.shape
    G, M = k.shape[1], k.shape[2]
    q = q.reshape(S, N, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(S, G, (H // G) * N, D)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(S, G, H // G, N, M)
    score.masked_fill_(~visible[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True) if M else score.new_zeros((S, G, H // G, N, 1))
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = score.sub_(top).exp_()
    den = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(S, G, (H // G) * N, M), v).view(S, G, H // G, N, D)
    out = out / torch.where(den > 0, den, torch.ones_like(den))
    out = out.permute(0, 3, 1, 2, 4).reshape(S, N, H, D)
    return (out * gates[..., None]).to(dtype)


def _visible(p, j, held, left, right, sinks):
    """p [S,N,1] positions of the queries, j [1,1,M] of the keys, held [S,1,M]."""
    see = held & (j >= 0)
    if right >= 0:
        see = see & (j <= p + right)
    if left >= 0:
        see = see & ((j >= p - left) | (j < sinks))
    return see


def _plain_prompt(s):
    case = s["case"]
    S, N, M = case["seqs"], case["q_tokens"], case["kv_tokens"]
    if s["q_len"] is None:
        q_len = torch.full((S, 1, 1), N, device="cuda")
        kv_len = torch.full((S, 1, 1), M, device="cuda")
    else:
        q_len, kv_len = s["q_len"].long().view(S, 1, 1), s["kv_len"].long().view(S, 1, 1)
    i = torch.arange(N, device="cuda").view(1, N, 1)
    j = torch.arange(M, device="cuda").view(1, 1, M)
    see = _visible(kv_len - q_len + i, j, j < kv_len, case["left"], case["right"], case["sinks"]) & (i < q_len)
    return {"out": _plain_attend(s["q"].float(), s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2), see,
                                 s["gates"], s["q"].dtype)}


def _plain_values(codes, scale):
    """4-bit rows as the values they stand for: middle + step * (code - 8), in the cache's type."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    f = scale.float()
    return (f[..., 1:] + f[..., :1] * (c - 8)).flatten(-2).to(scale.dtype)


def _plain_four_bits(x):
    """x [..., D] rounded to 4 bits per group of 32 and back."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((hi - lo) * (1.0 / 15.0)).to(x.dtype).float()
    mid = (lo + 8 * step).to(x.dtype).float()
    inv = torch.where(step > 0, step.reciprocal(), torch.zeros_like(step))
    c = (((g - mid) * inv).round() + 8).clamp(0, 15)
    return (mid + step * (c - 8)).flatten(-2).to(x.dtype)


def _plain_append(s):
    case = s["case"]
    p = s["pos"].long()[:, None] + torch.arange(case["tokens"], device="cuda")
    last = s["pos"].long()[:, None] + case["tokens"] - 1
    kept = ((p < case["sinks"]) | (p > last - case["ring"]))[:, :, None, None]
    out = {}
    for name in ("k", "v"):
        x = s[name] if case["bits"] == 16 else _plain_four_bits(s[name])
        out[name] = torch.where(kept, x, torch.zeros_like(x))
    return out


def _plain_step(s):
    case = s["case"]
    S, N, sinks, ring = case["seqs"], case["tokens"], case["sinks"], case["ring"]
    length = s["length"].long().view(S, 1, 1)
    slot = torch.arange(sinks + ring, device="cuda").view(1, 1, -1)
    # the newest position that a ring slot can hold; a slot of the first positions holds its own
    j = torch.where(slot < sinks, slot, length - 1 - (length - 1 - slot) % ring)
    held = (j < length) & ((slot < sinks) | (j >= sinks))
    p = length - N + torch.arange(N, device="cuda").view(1, N, 1)
    see = held & (j <= p) & (p >= 0)
    if case["left"] >= 0:
        see = see & ((j >= p - case["left"]) | (slot < sinks))
    k, v = s["ck"], s["cv"]
    if case["bits"] == 4:
        k, v = _plain_values(k, s["ck_scale"]), _plain_values(v, s["cv_scale"])
    return {"out": _plain_attend(s["q"].float(), k.float(), v.float(), see, s["gates"], s["q"].dtype)}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "rotate":
        return _plain_rotate(state)
    if op == "append":
        return _plain_append(state)
    return _plain_prompt(state) if op == "prompt" else _plain_step(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotate(s):
    D, out = s["case"]["dim"], {}
    for name in ("q", "k"):
        x = s[name].double()
        norm = x.pow(2).sum(-1, keepdim=True).div(D).add(EPS).sqrt()
        y = torch.view_as_complex((x / norm * s["gamma_" + name].double()).unflatten(-1, (D // 2, 2)).contiguous())
        at, parts = 0, []
        for a, n in enumerate(s["pairs"]):
            p = s["pos"][..., a].long()
            turn = torch.complex(s["cos"].double()[:, at:at + n], s["sin"].double()[:, at:at + n])[p]
            parts.append(y[..., at:at + n] * turn[:, :, None])
            at += n
        parts.append(y[..., at:])
        out[name] = torch.view_as_real(torch.cat(parts, -1)).flatten(-2)
    return out


def _exact_attend(q, k, v, bias, gates):
    """q [S,N,H,D]; k, v [S,M,G,D] in 64 bits; bias [S or 1,N,M]: 0 or -inf. One query head after the other."""
    S, N, H, D = q.shape
    G, out = k.shape[2], torch.zeros_like(q)
    for h in range(H):
        kh, vh = k[:, :, h * G // H], v[:, :, h * G // H]
        score = torch.einsum("snd,smd->snm", q[:, :, h], kh) * D ** -0.5 + bias
        out[:, :, h] = torch.nan_to_num(torch.softmax(score, -1), nan=0.0) @ vh
    return out * gates.double()[..., None]


def _exact_prompt(s):
    case = s["case"]
    N, M = case["q_tokens"], case["kv_tokens"]
    bias = torch.full((case["seqs"] if case["ragged"] else 1, N, M), -math.inf, dtype=torch.float64, device="cuda")
    key = torch.arange(M, device="cuda")[None]
    for b, (n, m) in enumerate(_prompt_lengths(case)[:bias.shape[0]]):
        at = torch.arange(m - n, m, device="cuda")[:, None]
        first = at - case["left"] if case["left"] >= 0 else torch.zeros_like(at)
        last = torch.clamp(at + case["right"], max=m - 1) if case["right"] >= 0 else torch.full_like(at, m - 1)
        see = ((key >= first) & (key <= last)) | ((key < case["sinks"]) & (key <= last))
        bias[b, :n][see] = 0.0
    return {"out": _exact_attend(s["q"].double(), s["k"].double(), s["v"].double(), bias, s["gates"])}


def _exact_append(s):
    case, out = s["case"], {}
    N = case["tokens"]
    for name in ("k", "v"):
        x = s[name].double()
        if case["bits"] == 4:
            T, rounded = s[name].dtype, []
            for g in x.split(GROUP, dim=-1):
                lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
                step = ((hi - lo) / 15).to(T).double()
                mid = (lo + 8 * step).to(T).double()
                code = torch.where(step > 0, torch.round((g - mid) / step), 0 * g).clamp(-8, 7)
                rounded.append((mid + code * step).to(T).double())
            x = torch.cat(rounded, -1)
        for b in range(case["seqs"]):
            first = _seen(case, b)
            gone = [i for i in range(N) if case["sinks"] <= first + i < first + N - case["ring"]]
            if gone:
                x[b, gone[0]:gone[-1] + 1] = 0
        out[name] = x
    return out


def _exact_step(s):
    case = s["case"]
    S, N, sinks, ring, D = case["seqs"], case["tokens"], case["sinks"], case["ring"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(S):
        length = _seen(case, b) + N
        j = torch.arange(length, device="cuda")
        j = j[(j < sinks) | (j >= length - ring)]
        slot = torch.where(j < sinks, j, sinks + (j - sinks) % ring)
        kv = []
        for name in ("ck", "cv"):
            x = s[name][b][:, slot]
            if case["bits"] == 4:
                f = s[name + "_scale"][b][:, slot].double()
                code = torch.empty(x.shape[:-1] + (D,), dtype=torch.float64, device="cuda")
                code[..., 0::2], code[..., 1::2] = (x % 16).double(), (x // 16).double()
                step, mid = (f[..., n].repeat_interleave(GROUP, -1) for n in (0, 1))
                x = (mid + step * (code - 8)).to(s["q"].dtype)
            kv.append(x.double().transpose(0, 1)[None])
        p = torch.arange(length - N, length, device="cuda")[:, None]
        see = j[None] <= p
        if case["left"] >= 0:
            see &= (j[None] >= p - case["left"]) | (j[None] < sinks)
        bias = torch.where(see, 0.0, -math.inf).double()[None]
        out[b:b + 1] = _exact_attend(s["q"][b:b + 1].double(), *kv, bias, s["gates"][b:b + 1])
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "prompt": _exact_prompt,
            "step": _exact_step}[case["op"]](s)


# ---------------------------------------------------------------------------
# work: each input read once, each output written once; products and sums of the visible pairs
# ---------------------------------------------------------------------------
def _row_bytes(case, es):
    """Bytes of one cached key or value of one head."""
    return case["dim"] * es if case["bits"] == 16 else case["dim"] // 2 + case["dim"] // GROUP * 2 * es


def work(case):
    S, D = case["seqs"], case["dim"]
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotate":
        n = S * case["tokens"] * (case["heads"] + case["kv_heads"]) * D
        return {"bytes": 2 * n * es + 4 * S * case["tokens"] * case["axes"], "flops": 9 * n}
    if case["op"] == "append":
        kept = 0
        for i in range(S):
            first, end = _seen(case, i), _seen(case, i) + case["tokens"]
            low = max(first, end - case["ring"], case["sinks"])
            kept += max(0, end - low) + max(0, min(end, case["sinks"]) - first)
        rows = kept * case["kv_heads"] * 2
        back = S * case["tokens"] * case["kv_heads"] * 2 * D * es
        return {"bytes": rows * (D * es + 2 * _row_bytes(case, es)) + back,
                "flops": rows * D * (8 if case["bits"] == 4 else 0)}
    H, G = case["heads"], case["kv_heads"]
    pairs = keys = queries = 0
    left = case["left"] if case["left"] >= 0 else 1 << 40
    if case["op"] == "prompt":
        right = case["right"] if case["right"] >= 0 else 1 << 40
        lens, row = _prompt_lengths(case), D * es
    else:
        right, row = 0, _row_bytes(case, es)
        lens = [(case["tokens"], _seen(case, i) + case["tokens"]) for i in range(S)]
    known = {}
    for n, m in lens:
        if (n, m) not in known:
            held = max(0, m - case["ring"]) if case["op"] == "step" else 0
            got, lowest = 0, m
            for p in range(m - n, m):
                end = min(m, p + right + 1)
                low = max(0, p - left, held)
                first = min(case["sinks"], end, low)
                got += max(0, end - low) + max(0, first)
                lowest = min(lowest, low)
            known[n, m] = (got, (m - lowest + min(case["sinks"], lowest)) if n else 0)
        pairs += known[n, m][0]
        keys += known[n, m][1]
        queries += n
    total = S * (case["q_tokens"] if case["op"] == "prompt" else case["tokens"])
    return {"bytes": queries * H * (D * es + 4) + total * H * D * es + 2 * keys * G * row, "flops": 4 * D * H * pairs}
