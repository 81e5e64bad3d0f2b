"""GPU parity of the streaming-attention operators against 64-bit CPU references (tests/stream_ref.py, which derives
the bounds), at the sizes, strides and masks where they can go wrong, and their refusals."""
import math

import pytest

import stream_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _dt(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def _randn(torch, shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _within(got, want, bound, what):
    got = got.double().cpu()
    assert got.shape == want.shape
    nan = want.isnan()
    assert (got.isnan() == nan).all(), f"{what}: NaN in other places"
    err = (got - want).abs()[~nan]
    over = err - bound[~nan]
    assert (over <= 0).all(), f"{what}: error {err.max():.3e}, over its bound by {over.max():.3e}"


# ---------------------------------------------------------------------------
# norm + rotation
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("S,N,H,G,D,pairs", [
    (1, 1, 1, 1, 64, [32]),
    (3, 7, 8, 8, 64, [32]),
    (2, 33, 8, 2, 32, [8, 8]),
    (2, 5, 4, 1, 128, [20, 21, 23]),
    (1, 9, 3, 3, 40, [7, 5]),
    (2, 3, 2, 2, 6, [1, 1, 1]),
    (1, 4, 2, 1, 256, [100, 10, 10, 8]),
    (2, 17, 5, 0, 64, [16, 0, 16]),
    (5, 2, 16, 16, 96, []),
    (2, 70, 8, 8, 64, [3, 29]),
])
def test_qk_norm_rope(torch_cuda, dtype, S, N, H, G, D, pairs):
    torch = torch_cuda
    import cudasep

    dt, rows = _dt(torch, dtype), 50
    q, k = _randn(torch, (S, N, H, D), dt, 1, 2.0), _randn(torch, (S, N, G, D), dt, 2, 0.3)
    gq, gk = _randn(torch, (D,), torch.float32, 3), _randn(torch, (D,), torch.float32, 4)
    ang = _randn(torch, (rows, max(1, D // 2)), torch.float32, 5, 3.0)
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, rows, (S, N, len(pairs)), generator=torch.Generator().manual_seed(6), dtype=torch.int32)
    got = cudasep.op_qk_norm_rope(q.cuda(), k.cuda(), gq.cuda(), gk.cuda(), cos.cuda(), sin.cuda(), pos.cuda(), pairs,
                                  eps=1e-5)
    for x, gamma, y in ((q, gq, got[0]), (k, gk, got[1])):
        _within(y, *ref.rotate(x, gamma, cos, sin, pos, pairs, 1e-5), "qk_norm_rope")


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("S,N,H,G,D,pairs", [
    (60, 101, 8, 2, 32, [8, 4, 4]),  # heads that do not fill a step of the form for many tokens
    (41, 103, 8, 8, 64, [20]),       # some pairs are not turned
    (30, 100, 9, 4, 128, [40, 24]),
])
def test_qk_norm_rope_many_tokens(torch_cuda, dtype, S, N, H, G, D, pairs):
    test_qk_norm_rope(torch_cuda, dtype, S, N, H, G, D, pairs)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("layout", ["packed", "offset", "in_place", "no_gamma"])
def test_qk_norm_rope_layouts(torch_cuda, dtype, layout):
    """Views of the packed q|k|v rows along the time axis, rows that are not 16-byte aligned, results in place, no gain."""
    torch = torch_cuda
    import cudasep

    dt, S, N, H, G, D = _dt(torch, dtype), 3, 11, 4, 2, 64
    pairs = [16, 16]
    odd = 1 if layout == "offset" else 0
    x = _randn(torch, (N, S, H + 2 * G, D + odd), dt, 7)
    xd = x.cuda()
    gq, gk = (None, None) if layout == "no_gamma" else (_randn(torch, (D,), torch.float32, 8),) * 2
    ang = _randn(torch, (2048, D // 2), torch.float32, 9)
    cos, sin = ang.cos(), ang.sin()
    pos = torch.stack([torch.arange(N).expand(S, N) + 1990, torch.arange(S)[:, None].expand(S, N)], -1).int().contiguous()

    def views(t):
        t = t.transpose(0, 1)[..., odd:]
        return t[:, :, :H], t[:, :, H:H + G]

    q, k = views(xd)
    want = [ref.rotate(a, g, cos, sin, pos, pairs, 1e-6) for a, g in zip(views(x), (gq, gk))]
    keep = xd.clone()
    dev = [None if t is None else t.cuda() for t in (gq, gk)]
    out = dict(q_out=q, k_out=k) if layout == "in_place" else {}
    got = cudasep.op_qk_norm_rope(q, k, *dev, cos.cuda(), sin.cuda(), pos.cuda(), pairs, **out)
    for y, w in zip(got, want):
        _within(y, *w, layout)
    if layout == "in_place":  # v is not touched
        assert torch.equal(xd[:, :, H + G:], keep[:, :, H + G:])
        assert got[0].data_ptr() == q.data_ptr()
    else:
        assert torch.equal(xd, keep)


def test_qk_norm_rope_positions_outside_the_tables_are_nan(torch_cuda):
    torch = torch_cuda
    import cudasep

    q = _randn(torch, (1, 4, 2, 64), torch.float16, 1)
    cos = torch.ones(10, 32)
    pos = torch.tensor([[[0, 0], [10, 3], [3, -1], [2 ** 31 - 1, 9]]], dtype=torch.int32)
    want, bound = ref.rotate(q, None, cos, cos, pos, [16, 8], 0.0)
    assert want.isnan().any() and not want.isnan().all()
    got, _ = cudasep.op_qk_norm_rope(q.cuda(), q.cuda(), None, None, cos.cuda(), cos.cuda(), pos.cuda(), [16, 8], eps=0.0)
    _within(got, want, bound, "positions")


def test_qk_norm_rope_zero_rows_and_empty_calls(torch_cuda):
    torch = torch_cuda
    import cudasep

    z = torch.zeros(1, 2, 3, 64, device="cuda")
    q, k = cudasep.op_qk_norm_rope(z, z)
    assert (q == 0).all() and (k == 0).all()
    for shape in ((0, 2, 3, 64), (1, 0, 3, 64)):
        e = torch.zeros(shape, device="cuda")
        q, k = cudasep.op_qk_norm_rope(e, e)
        assert tuple(q.shape) == shape
    # eps 0 and a zero row: 0 / 0
    q, _ = cudasep.op_qk_norm_rope(z, z, eps=0.0)
    assert q.isnan().all()


# ---------------------------------------------------------------------------
# cache
# ---------------------------------------------------------------------------
def _fill(torch, cache, k, v, pos=0):
    """All tokens of k, v [S, N, G, D] appended from position pos on."""
    import cudasep

    p = torch.full((k.shape[0],), pos, dtype=torch.int32, device="cuda")
    cudasep.op_cache_append(cache, k, v, p)


CACHES = [("fp32", 0), ("fp16", 0), ("bf16", 0), ("fp16", 4), ("bf16", 4)]


def _values(x, bits):
    return ref.four_bits(x)[3] if bits else x


def _same(a, b):
    a, b = a.cpu().double(), b.cpu().double()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dtype,bits", CACHES)
@pytest.mark.parametrize("D", [32, 64, 128, 8, 40])
@pytest.mark.parametrize("sinks,ring,steps", [(0, 7, [3, 3, 3]), (4, 9, [1, 1, 20, 2]), (3, 5, [2, 5]), (2, 70, [64, 1, 33]),
                                              (0, 1, [1, 4, 1])])
def test_cache_append_and_read(torch_cuda, dtype, bits, D, sinks, ring, steps):
    """Every position that should be held reads back as what was written (4 bits: exactly the defined values), others as
    zeros, whatever the steps in which they were written."""
    torch = torch_cuda
    import cudasep

    if bits and D % 32:
        pytest.skip("4 bits need a multiple of 32")
    dt, S, G = _dt(torch, dtype), 2, 3
    cache = cudasep.KVCache.empty(S, G, sinks + ring, D, dt, sinks=sinks, bits=bits)
    total = sum(steps)
    k, v = _randn(torch, (S, total, G, D), dt, 11), _randn(torch, (S, total, G, D), dt, 12, 3.0)
    at = 0
    for n in steps:
        start = torch.full((S,), at, dtype=torch.int32, device="cuda")
        cudasep.op_cache_append(cache, k[:, at:at + n].cuda(), v[:, at:at + n].cuda(), start)
        at += n
        zero = torch.zeros(S, dtype=torch.int32, device="cuda")
        gk, gv = cudasep.op_cache_read(cache, zero, at)
        held = torch.arange(at)
        held = ((held < sinks) | (held >= at - ring)).view(1, -1, 1, 1)
        for got, x in ((gk, k), (gv, v)):
            assert _same(got, torch.where(held, _values(x[:, :at], bits), torch.zeros((), dtype=dt)))


@pytest.mark.parametrize("dtype,bits", CACHES)
def test_cache_ragged_counts_negative_positions_and_views(torch_cuda, dtype, bits):
    """Counts below, at and above `tokens`; positions below zero are left out; strided and unaligned views; other
    sequences' and slots' bytes stay."""
    torch = torch_cuda
    import cudasep

    dt, S, G, D, N, sinks, ring = _dt(torch, dtype), 6, 2, 64, 9, 2, 6
    cache = cudasep.KVCache.empty(S, G, sinks + ring, D, dt, sinks=sinks, bits=bits)
    old_k, old_v = _randn(torch, (S, 8, G, D), dt, 1), _randn(torch, (S, 8, G, D), dt, 2)
    _fill(torch, cache, old_k.cuda(), old_v.cuda())
    base = _randn(torch, (N, S, 2 * G, D + 1), dt, 3)
    new = base.cuda().transpose(0, 1)[..., 1:]
    host = base.transpose(0, 1)[..., 1:]
    pos = torch.tensor([8, 8, 8, 5, -3, 2 ** 31 - 4], dtype=torch.int32)
    count = torch.tensor([0, 3, 100, 9, 9, 9], dtype=torch.int32)
    cudasep.op_cache_append(cache, new[:, :, :G], new[:, :, G:], pos.cuda(), count.cuda())
    buf = torch.zeros(S, N, 2 * G, D + 1, dtype=dt, device="cuda")
    rk, rv = cudasep.op_cache_read(cache, pos.cuda(), N, count=count.cuda(), k=buf[:, :, :G, 1:], v=buf[:, :, G:, 1:])
    for got, x in ((rk, host[:, :, :G]), (rv, host[:, :, G:])):
        vals = _values(x.contiguous(), bits)
        want = torch.zeros(S, N, G, D, dtype=dt)
        for s in range(S):
            n, p0 = min(int(count[s]), N), int(pos[s])
            for i in range(n):
                p = p0 + i
                if 0 <= p < 2 ** 31 and (p < sinks or p > p0 + n - 1 - ring):
                    want[s, i] = vals[s, i]
        assert _same(got, want)
    assert (buf[..., 0] == 0).all()
    # the untouched sequence still holds its own
    z = torch.zeros(S, dtype=torch.int32, device="cuda")
    gk, _ = cudasep.op_cache_read(cache, z, 8)
    assert _same(gk[0], _values(old_k, bits)[0])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_four_bit_codes(torch_cuda, dtype):
    """Codes, steps and offsets are the defined ones, at ties, constant groups, subnormal ranges, large offsets and
    values that are not finite."""
    torch = torch_cuda
    import cudasep

    dt, D = _dt(torch, dtype), 64
    x = _randn(torch, (1, 12, 1, D), dt, 5)
    x[0, 0] = 0
    x[0, 1] = 3.25
    x[0, 2, 0, :32] = torch.arange(32) % 16
    x[0, 3] = x[0, 3] * 2.0 ** -14
    x[0, 4] = x[0, 4] + 500
    x[0, 5] = x[0, 5] * 1e4
    x[0, 6, 0, 3] = math.inf
    x[0, 7, 0, 40] = math.nan
    x[0, 8, 0, 0], x[0, 8, 0, 1] = torch.finfo(dt).max, torch.finfo(dt).min
    x[0, 9, 0, ::2] = -0.0
    x[0, 10] = torch.arange(64).view(1, 64) * 0.5
    code, step, mid, values = ref.four_bits(x)
    cache = cudasep.KVCache.empty(1, 1, 16, D, dt, bits=4)
    _fill(torch, cache, x.cuda(), x.cuda())
    finite = ~values.isnan()
    got_codes = torch.stack([cache.k & 15, cache.k >> 4], -1).flatten(-2)[0, 0, :12].cpu().double()
    assert torch.equal(got_codes[finite[0, :, 0]], code[0, :, 0].double()[finite[0, :, 0]])
    ok = finite.unflatten(-1, (2, 32)).all(-1)[0, :, 0]
    assert torch.equal(cache.k_scale[0, 0, :12, :, 0].cpu().float()[ok], step[0, :, 0][ok])
    assert torch.equal(cache.k_scale[0, 0, :12, :, 1].cpu().float()[ok], mid[0, :, 0][ok])
    assert cache.k_scale[0, 0, :12].cpu()[~ok].isnan().all()
    k, v = cudasep.op_cache_read(cache, torch.zeros(1, dtype=torch.int32, device="cuda"), 12)
    assert _same(k, values) and _same(v, values)


# ---------------------------------------------------------------------------
# windowed attention, prompt form
# ---------------------------------------------------------------------------
def _window_case(torch, dtype, S, N, M, H, G, D, left, right, sinks, q_len=None, kv_len=None, gates=True, scale=0.0,
                 size=1.0, make=None, layout="plain"):
    import cudasep

    dt = _dt(torch, dtype)
    q = _randn(torch, (S, N, H, D), dt, 21, size)
    k, v = _randn(torch, (S, M, G, D), dt, 22, size), _randn(torch, (S, M, G, D), dt, 23)
    gt = torch.rand(S, N, H, generator=torch.Generator().manual_seed(24)) if gates else None
    if make:
        make(q, k, v)
    ql = None if q_len is None else torch.tensor(q_len, dtype=torch.int32)
    kl = None if kv_len is None else torch.tensor(kv_len, dtype=torch.int32)
    want, bound = torch.zeros(S, N, H, D, dtype=torch.float64), torch.zeros(S, N, H, D, dtype=torch.float64)
    for s in range(S):
        n = N if q_len is None else min(max(q_len[s], 0), N)
        m = M if kv_len is None else min(max(kv_len[s], 0), M)
        see = ref.visible(range(m - n, m), m, left, right, sinks)
        want[s, :n], bound[s, :n] = ref.attention(q[s, :n], k[s, :m], v[s, :m], see, scale or D ** -0.5,
                                                  None if gt is None else gt[s, :n])
    if layout == "plain":
        dq, dk, dv, out = q.cuda(), k.cuda(), v.cuda(), None
    else:  # token-major packed rows; "odd": rows that are not 16-byte aligned
        odd = 1 if layout == "odd" else 0
        x = torch.zeros(max(N, M), S, H + 2 * G, D + odd, dtype=dt, device="cuda").transpose(0, 1)[..., odd:]
        dq, dk, dv = x[:, :N, :H], x[:, :M, H:H + G], x[:, :M, H + G:]
        for d, t in ((dq, q), (dk, k), (dv, v)):
            d.copy_(t)
        out = torch.full((S, H, N, D + odd), 7.0, dtype=dt, device="cuda").transpose(1, 2)[..., odd:]
    dev = [None if t is None else t.cuda() for t in (ql, kl, gt)]
    got = cudasep.op_window_attention(dq, dk, dv, left=left, right=right, sinks=sinks, scale=scale, q_len=dev[0],
                                      kv_len=dev[1], gates=dev[2], out=out)
    torch.cuda.synchronize()
    _within(got, want, bound, "window_attention")
    return got


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("S,N,M,H,G,D,left,right,sinks", [
    (1, 1, 1, 1, 1, 64, -1, -1, 0),
    (2, 1, 40, 2, 1, 64, 10, 0, 2),
    (1, 130, 130, 2, 2, 64, -1, 0, 0),
    (1, 129, 129, 1, 1, 64, -1, -1, 0),
    (2, 200, 200, 2, 2, 64, 30, 5, 3),
    (1, 257, 257, 1, 1, 64, 63, 0, 70),
    (1, 100, 300, 4, 2, 64, 64, 64, 1),
    (1, 150, 150, 2, 1, 32, 20, 0, 4),
    (1, 140, 260, 2, 1, 128, 90, 0, 130),
    (1, 66, 66, 3, 1, 40, 0, 0, 0),
    (1, 65, 70, 2, 2, 96, -1, 3, 5),
    (1, 64, 128, 8, 1, 64, 0, 0, 1),
    (2, 63, 65, 2, 2, 8, 7, 0, 0),
    (1, 300, 300, 1, 1, 64, 2 ** 31 - 1, 2 ** 31 - 1, 2),
])
def test_window_attention(torch_cuda, dtype, S, N, M, H, G, D, left, right, sinks):
    _window_case(torch_cuda, dtype, S, N, M, H, G, D, left, right, sinks)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("S,N,M,H,G,D,left,right,sinks", [
    (30, 130, 150, 8, 8, 64, 70, 3, 2),   # several tiles a CTA, the latest queries first
    (30, 140, 140, 8, 8, 32, 70, -1, 0),  # in order
    (20, 130, 140, 8, 8, 128, -1, 0, 0),
    (40, 150, 100, 8, 2, 64, 20, 0, 1),   # more queries than keys: the first see nothing
    (1, 16, 90, 2, 1, 64, 30, 0, 1),      # two row tiles of the form for few queries
    (1, 25, 300, 1, 1, 128, -1, 0, 0),
    (100, 20, 70, 2, 2, 64, 33, 2, 0),    # as many rows, but many sequences
])
def test_window_attention_many_tiles(torch_cuda, dtype, S, N, M, H, G, D, left, right, sinks):
    _window_case(torch_cuda, dtype, S, N, M, H, G, D, left, right, sinks)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (20, 3, 2), (-1, -1, 0), (5, 40, 0)])
def test_window_attention_ragged(torch_cuda, dtype, left, right, sinks):
    """No queries, no keys, one of each, more queries than keys (the first see nothing or only what lies ahead),
    lengths beyond the buffers."""
    q_len = [0, 5, 1, 130, 140, 9, 200, -4]
    kv_len = [50, 0, 1, 130, 100, 140, 1000, 30]
    _window_case(torch_cuda, dtype, 8, 140, 140, 2, 1, 64, left, right, sinks, q_len, kv_len)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_window_attention_strides(torch_cuda, dtype, layout):
    _window_case(torch_cuda, dtype, 3, 90, 150, 4, 2, 64, 50, 2, 3, layout=layout)
    _window_case(torch_cuda, dtype, 2, 70, 70, 2, 2, 128, -1, 0, 0, layout=layout, gates=False, scale=0.3)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_window_attention_large_scores(torch_cuda, dtype):
    """Scores that grow along the keys (the running maximum rises in every block), that fall, and that are all far
    below zero."""
    torch = torch_cuda

    def rising(q, k, v):
        q.fill_(0.5)
        k.copy_((torch.arange(k.shape[1]) * 0.5).view(1, -1, 1, 1).expand_as(k))

    def falling(q, k, v):
        q.fill_(0.5)
        k.copy_((torch.arange(k.shape[1]) * -0.5).view(1, -1, 1, 1).expand_as(k))

    def low(q, k, v):
        q.fill_(4.0)
        k.sub_(20.0)

    for make in (rising, falling, low):
        for left, sinks in ((-1, 0), (100, 2)):
            _window_case(torch, dtype, 1, 200, 330, 1, 1, 64, left, 0, sinks, make=make)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, "max", "min"])
def test_window_attention_hidden_keys_have_no_effect(torch_cuda, dtype, bad):
    """What a query does not see may hold anything: keys past the length, behind the window, and keys that only other
    queries of the same tile see.  Queries that do see them get what the formula gives."""
    torch = torch_cuda
    import cudasep

    dt, S, N, M, H, D = _dt(torch, dtype), 2, 150, 200, 2, 64
    left, sinks = 20, 3
    value = {"max": torch.finfo(dt).max, "min": torch.finfo(dt).min}.get(bad, bad)
    q, k, v = (_randn(torch, (S, n, H, D), dt, i) for i, n in ((1, N), (2, M), (3, M)))
    kl = [150, 170]
    clean = [ref.attention(q[s], k[s, :kl[s]], v[s, :kl[s]],
                           ref.visible(range(kl[s] - N, kl[s]), kl[s], left, 0, sinks), D ** -0.5, None)
             for s in range(S)]
    hit = 90
    for s in range(S):
        for t in (k, v):
            t[s, kl[s]:] = value  # past the end
            t[s, hit] = value     # seen by the queries at positions hit .. hit + left only
            t[s, sinks:max(sinks, kl[s] - N - left)] = value  # behind every window
    got = cudasep.op_window_attention(q.cuda(), k.cuda(), v.cuda(), left=left, right=0, sinks=sinks,
                                      kv_len=torch.tensor(kl, dtype=torch.int32, device="cuda"))
    for s in range(S):
        p = torch.arange(N) + kl[s] - N
        sees = (p >= hit) & (p <= hit + left)
        _within(got[s, ~sees], clean[s][0][~sees], clean[s][1][~sees], "rows that do not see it")
        if bad is math.nan:
            assert got[s, sees].isnan().all()


def test_window_attention_all_scores_minus_infinity_is_nan(torch_cuda):
    torch = torch_cuda
    import cudasep

    for dt in (torch.float32, torch.float16, torch.bfloat16):
        q = torch.ones(1, 3, 1, 64, dtype=dt, device="cuda")
        k = torch.full((1, 3, 1, 64), -math.inf, dtype=dt, device="cuda")
        out = cudasep.op_window_attention(q, k, q, right=0)
        assert out.isnan().all()


def test_window_attention_empty_calls(torch_cuda):
    torch = torch_cuda
    import cudasep

    for S, N, M, H in ((0, 3, 3, 2), (2, 0, 3, 2), (2, 3, 3, 0)):
        q = torch.zeros(S, N, H, 64, dtype=torch.float16, device="cuda")
        k = torch.zeros(S, M, H, 64, dtype=torch.float16, device="cuda")
        assert cudasep.op_window_attention(q, k, k).shape == q.shape
    for dt in (torch.float32, torch.bfloat16):
        q = torch.ones(2, 3, 2, 64, dtype=dt, device="cuda")
        k = torch.ones(2, 0, 2, 64, dtype=dt, device="cuda")
        assert (cudasep.op_window_attention(q, k, k) == 0).all()


# ---------------------------------------------------------------------------
# attention over the cache
# ---------------------------------------------------------------------------
def _cache_case(torch, dtype, bits, S, N, H, G, D, sinks, ring, lengths, left, right=0, gates=True, garbage=None):
    """Caches filled by appends to the given lengths; each sequence against the reference on the values it holds."""
    import cudasep

    dt = _dt(torch, dtype)
    top = max(max(lengths), 1)
    k, v = _randn(torch, (S, top, G, D), dt, 31), _randn(torch, (S, top, G, D), dt, 32)
    cache = cudasep.KVCache.empty(S, G, sinks + ring, D, dt, sinks=sinks, bits=bits)
    if garbage is not None:  # what unused slots hold
        for t in ((cache.k, cache.v) if not bits else (cache.k_scale, cache.v_scale)):
            t.fill_(garbage)
    cnt = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    zero = torch.zeros(S, dtype=torch.int32, device="cuda")
    cudasep.op_cache_append(cache, k.cuda(), v.cuda(), zero, count=cnt)
    kv, vv = _values(k, bits), _values(v, bits)
    q = _randn(torch, (S, N, H, D), dt, 33)
    gt = torch.rand(S, N, H, generator=torch.Generator().manual_seed(34)) if gates else None
    want, bound = torch.zeros(S, N, H, D, dtype=torch.float64), torch.zeros(S, N, H, D, dtype=torch.float64)
    for s in range(S):
        m = lengths[s]
        rows = [i for i in range(N) if m - N + i >= 0]
        if rows and m:
            see = ref.visible([m - N + i for i in rows], m, left, right, sinks, held_from=m - ring)
            w = ref.attention(q[s, rows], kv[s, :m], vv[s, :m], see, D ** -0.5, None if gt is None else gt[s, rows])
            want[s, rows], bound[s, rows] = w
    got = cudasep.op_cache_attention(q.cuda(), cache, cnt, left=left, right=right, gates=None if gt is None else gt.cuda())
    torch.cuda.synchronize()
    _within(got, want, bound, "cache_attention")


@pytest.mark.parametrize("dtype,bits", CACHES)
@pytest.mark.parametrize("S,N,H,G,D,sinks,ring,lengths,left", [
    (1, 1, 1, 1, 64, 0, 16, [1], -1),
    (4, 1, 8, 8, 64, 4, 60, [1, 64, 65, 200], -1),
    (4, 1, 2, 2, 64, 4, 100, [3, 4, 5, 333], 17),
    (2, 3, 4, 1, 64, 0, 300, [300, 299], -1),
    (2, 5, 8, 2, 64, 2, 130, [7, 500], 40),
    (2, 16, 4, 2, 128, 17, 90, [100, 1000], -1),
    (3, 2, 2, 2, 32, 1, 33, [2, 34, 77], 8),
    (2, 20, 4, 1, 64, 3, 257, [600, 21], 200),
    (2, 1, 16, 1, 64, 0, 700, [650, 1500], -1),
    (1, 1, 3, 3, 96, 5, 40, [300], -1),
    (1, 2, 2, 1, 40, 5, 40, [300], 12),
    (1, 1, 1, 1, 64, 0, 1, [9], -1),
])
def test_cache_attention(torch_cuda, dtype, bits, S, N, H, G, D, sinks, ring, lengths, left):
    if bits and D % 32:
        pytest.skip("4 bits need a multiple of 32")
    _cache_case(torch_cuda, dtype, bits, S, N, H, G, D, sinks, ring, lengths, left)


@pytest.mark.parametrize("dtype,bits", CACHES)
def test_cache_attention_short_and_empty_sequences(torch_cuda, dtype, bits):
    """Fewer tokens than queries: rows of negative position are zeros; unused slots hold NaN; keys ahead are seen."""
    torch = torch_cuda
    _cache_case(torch, dtype, bits, 5, 4, 2, 1, 64, 2, 30, [0, 1, 3, 4, 31], -1, garbage=math.nan)
    _cache_case(torch, dtype, bits, 3, 6, 4, 2, 64, 0, 50, [6, 20, 100], 9, right=2, garbage=math.inf)
    _cache_case(torch, dtype, bits, 2, 3, 2, 2, 32, 3, 50, [60, 20], 5, right=-1, gates=False)


@pytest.mark.parametrize("dtype,bits", CACHES)
def test_cache_attention_long(torch_cuda, dtype, bits):
    """A long axis that is split and joined, few rows."""
    _cache_case(torch_cuda, dtype, bits, 1, 1, 2, 1, 64, 4, 6000, [7001], -1)
    _cache_case(torch_cuda, dtype, bits, 2, 2, 2, 1, 64, 4, 3000, [2999, 5], 1999)


@pytest.mark.parametrize("dtype,bits", CACHES)
def test_cache_attention_hidden_values_have_no_effect(torch_cuda, dtype, bits):
    """A NaN key that only some rows of a step see stays with those rows."""
    torch = torch_cuda
    import cudasep

    dt, S, N, G, D, ring = _dt(torch, dtype), 1, 4, 2, 64, 100
    k, v = _randn(torch, (S, 90, G, D), dt, 1), _randn(torch, (S, 90, G, D), dt, 2)
    q = _randn(torch, (S, N, G, D), dt, 3).cuda()
    length = torch.tensor([90], dtype=torch.int32, device="cuda")
    want, bound = ref.attention(q[0].cpu(), _values(k, bits)[0], _values(v, bits)[0], ref.visible(range(86, 90), 90, 20, 0, 0),
                                D ** -0.5, None)
    k[0, 89, 1], v[0, 88, 0], v[0, 40] = math.nan, math.inf, math.nan
    cache = cudasep.KVCache.empty(S, G, ring, D, dt, bits=bits)
    _fill(torch, cache, k.cuda(), v.cuda())
    got = cudasep.op_cache_attention(q, cache, length, left=20).cpu()[0]
    _within(got[:3, 1], want[:3, 1], bound[:3, 1], "rows that do not see it")
    _within(got[:2, 0], want[:2, 0], bound[:2, 0], "rows that do not see it")
    assert got[3, 1].isnan().all() and not torch.isfinite(got[2:, 0]).any()


def test_cache_attention_empty_calls(torch_cuda):
    torch = torch_cuda
    import cudasep

    cache = cudasep.KVCache.empty(2, 2, 8, 64, torch.float16)
    length = torch.zeros(2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 0, 2, 64, dtype=torch.float16, device="cuda")
    assert cudasep.op_cache_attention(q, cache, length).shape == q.shape
    q = torch.ones(2, 1, 2, 64, dtype=torch.float16, device="cuda")
    assert (cudasep.op_cache_attention(q, cache, length - 5) == 0).all()


# ---------------------------------------------------------------------------
# streams, graphs, repeatability
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bits", [("fp16", 0), ("bf16", 4), ("fp32", 0)])
def test_streams_graphs_and_repeats(torch_cuda, dtype, bits):
    """The calls run on the given stream, can be captured, and give the same bits every time."""
    torch = torch_cuda
    import cudasep

    dt, S, N, H, D = _dt(torch, dtype), 3, 150, 2, 64
    q, k, v = (_randn(torch, (S, N, H, D), dt, i).cuda() for i in range(3))
    pos = torch.zeros(S, dtype=torch.int32, device="cuda")
    length = torch.full((S,), N, dtype=torch.int32, device="cuda")
    cache = cudasep.KVCache.empty(S, H, 120, D, dt, sinks=4, bits=bits)
    outs = [torch.empty_like(q), torch.empty_like(q), torch.empty(S, 2, H, D, dtype=dt, device="cuda")]
    kk = torch.empty_like(k)

    def chain():
        cudasep.op_qk_norm_rope(q, k, q_out=outs[0], k_out=kk)
        cudasep.op_window_attention(outs[0], kk, v, left=40, right=0, sinks=4, out=outs[1])
        cudasep.op_cache_append(cache, kk, v, pos)
        cudasep.op_cache_attention(outs[0][:, -2:], cache, length, out=outs[2])

    chain()
    torch.cuda.synchronize()
    want = [t.clone() for t in outs]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for t in outs + [kk]:
            t.zero_()
        chain()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for _ in range(3):
        for t in outs + [kk, cache.k, cache.v]:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals_of_the_binding(torch_cuda):
    torch = torch_cuda
    import cudasep

    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device="cuda")
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = cudasep.KVCache.empty(2, 4, 8, 64, torch.float16)
    bad = [
        lambda: cudasep.op_qk_norm_rope(q, q.float()),
        lambda: cudasep.op_qk_norm_rope(q, q[:, :2]),
        lambda: cudasep.op_qk_norm_rope(q, q, pairs=[32]),
        lambda: cudasep.op_qk_norm_rope(q, q, gamma_q=torch.ones(64, device="cuda", dtype=torch.float16)),
        lambda: cudasep.op_qk_norm_rope(q.cpu(), q.cpu()),
        lambda: cudasep.op_qk_norm_rope(q[..., ::2], q[..., ::2]),
        lambda: cudasep.op_window_attention(q, q.bfloat16(), q),
        lambda: cudasep.op_window_attention(q, q[:1], q),
        lambda: cudasep.op_window_attention(q, q, q, q_len=i32.long()),
        lambda: cudasep.op_window_attention(q, q, q, gates=torch.ones(2, 3, device="cuda")),
        lambda: cudasep.op_window_attention(q, q, q, out=q[:, :1]),
        lambda: cudasep.op_cache_append(cache, q[:, :, :2], q[:, :, :2], i32),
        lambda: cudasep.op_cache_append(cache, q, q, i32[:1]),
        lambda: cudasep.op_cache_append(cache, q.float(), q.float(), i32),
        lambda: cudasep.op_cache_read(cache, i32.long(), 3),
        lambda: cudasep.op_cache_attention(q[:1], cache, i32),
        lambda: cudasep.op_cache_attention(q, cache, None),
        lambda: cudasep.KVCache(cache.k, cache.v[:, :, :4]),
        lambda: cudasep.KVCache(cache.k, cache.v, sinks=8),
        lambda: cudasep.KVCache(cache.k.view(torch.uint8), cache.v.view(torch.uint8)),
        lambda: cudasep.KVCache.empty(2, 4, 8, 64, torch.float16, bits=8),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted:", n)


def test_refusals_of_the_library(torch_cuda):
    """The checks behind the C entry points (code MBR_ERR_INVALID), which launch nothing."""
    torch = torch_cuda
    import cudasep

    def z(*shape, dt=torch.float16):
        return torch.zeros(shape, dtype=dt, device="cuda")

    q = z(2, 3, 4, 64)
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = z(5, 32, dt=torch.float32)
    pos = torch.zeros(2, 3, 2, dtype=torch.int32, device="cuda")
    calls = [
        (lambda: cudasep.op_qk_norm_rope(z(1, 1, 1, 63), z(1, 1, 1, 63)), "dim_head"),
        (lambda: cudasep.op_qk_norm_rope(z(1, 1, 1, 258), z(1, 1, 1, 258)), "dim_head"),
        (lambda: cudasep.op_qk_norm_rope(q, q, None, None, table, table, pos, [20, 13]), "sections"),
        (lambda: cudasep.op_qk_norm_rope(q, q, None, None, table, table, pos, [-1, 3]), "sections"),
        (lambda: cudasep.op_qk_norm_rope(q, q, eps=-1.0), "eps"),
        (lambda: cudasep.op_window_attention(z(1, 2, 3, 64), z(1, 2, 2, 64), z(1, 2, 2, 64)), "multiple of kv_heads"),
        (lambda: cudasep.op_window_attention(z(1, 2, 2, 136), z(1, 2, 2, 136), z(1, 2, 2, 136)), "dim_head"),
        (lambda: cudasep.op_window_attention(z(1, 2, 2, 12), z(1, 2, 2, 12), z(1, 2, 2, 12)), "dim_head"),
        (lambda: cudasep.op_window_attention(q, q, q, sinks=-1), "sinks"),
        (lambda: cudasep.op_window_attention(q, q, q, scale=math.inf), "scale"),
        (lambda: cudasep.op_cache_append(cudasep.KVCache.empty(2, 4, 8, 136, torch.float16), z(2, 3, 4, 136),
                                         z(2, 3, 4, 136), i32), "dim_head"),
        (lambda: cudasep.op_cache_attention(z(2, 1, 3, 64), cudasep.KVCache.empty(2, 2, 8, 64, torch.float16), i32),
         "multiple of kv_heads"),
    ]
    for call, text in calls:
        with pytest.raises(cudasep.MBRError) as e:
            call()
        assert e.value.code == 1 and text in str(e.value), (text, str(e.value))
