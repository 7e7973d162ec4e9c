"""Operators around an int8 K/V cache on the device, against plain 64-bit implementations.

Tolerances.  u = 2^-24 is half a step of fp32, 2^-8 of bfloat16 (finfo.eps / 2).
  qk_norm_rope_seq   a sum of up to 256 squares, 8 in a lane and then pairs: 13 roundings at most, so 13 u of it, 6.5 u of
                     its root; the mean, eps, root and reciprocal 4 u, the two products and 1 + w 3 u: 14 u of a normalised element,
                     taken as 16.  A rotated one is x cos - y sin: the angle in turns, at most half a one, is rounded to
                     fp32 once (2^-25 of a turn, 3.2 u of a radian), sine and cosine are off by up to 2 u more, products and
                     the sum by 2 u: (16 + 8) u (|x| + |y|).  bfloat16: rounded once more.
  kv_cache_*         the quotient and the scale are IEEE divisions and everything else is exact: equal bits.
  attention_seq_i8   an element of q is off by half a unit, 1 / 2 of its row's largest over 32639 (bfloat16) or 8355711 (fp32),
                     a score so by that times |scale| sum |k|; the sum itself is exact, its conversions and the products with the
                     row's unit (itself three roundings) and K's scale take 10 u of the score.  The largest of
                     a row's errors counts twice, in the numerator and in the sum.  exp2 and its argument, sums over n keys
                     and their joins (16 + sqrt(n)) u, V's scale u, of sum p |v|; bfloat16: P in two parts, 2^-16 of it, in the form for few
                     rows and rounded once, 2^-8, in the one for prompts, and the output rounded once more.  A part of P below 2^-126, the smallest normal number, may count as 0 in the matrix instruction: each of
                     at most three parts of n keys then takes up to 2^-126 times a code of 128 from a sum that is divided by
                     at least 1 (the largest probability's term): n 3 2^-119 in all, whatever the output's size.
"""
import math
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = 2.0 ** -8


def gen(torch, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def starts(lens):
    return [0] + np.cumsum(lens).tolist()


# ------------------------------------------------------------------ norms and rotation

def rope_oracle(torch, x, w, pos, rot, theta=1e7, eps=1e-6):
    """float64 on the CPU: (out, bound)."""
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (1.0 + w.double())
    half, out, tol = rot // 2, y.clone(), 16 * U * y.abs()
    if half:
        ang = pos.double()[:, None] * torch.tensor([theta ** (-2.0 * i / rot) for i in range(half)], dtype=torch.float64)
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        a, b = y[..., :half], y[..., half:rot]
        out[..., :half], out[..., half:rot] = a * c - b * s, b * c + a * s
        both = 24 * U * (a.abs() + b.abs())
        tol[..., :half], tol[..., half:rot] = both, both
    return out, tol


def rope_check(torch, got, want, bf16):
    wo, tol = want
    err = (got.cpu().double() - wo).abs()
    lim = tol + (BF * (wo.abs() + tol) if bf16 else U * wo.abs())
    assert (err <= lim).all(), (err.max().item(), (err / lim.clamp(min=1e-30)).max().item())


ROPE = [  # tokens, heads, kv heads, dim, rotated
    (1, 8, 2, 256, 64), (1, 1, 1, 128, 128), (2, 3, 1, 256, 256), (5, 6, 2, 128, 32), (7, 16, 4, 128, 16), (33, 8, 2, 256, 0),
    (64, 32, 1, 256, 64), (65, 2, 2, 128, 64), (300, 8, 8, 128, 96), (1000, 8, 2, 256, 48), (3, 1, 40, 256, 240),
    (1801, 3, 1, 128, 64), (2000, 5, 2, 256, 48), (4097, 2, 3, 128, 16), (4096, 1, 1, 256, 32),   # another number of waves a token
]


@pytest.mark.parametrize("tokens,h,kvh,d,rot", ROPE)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_norm_rope(q, torch_cuda, tokens, h, kvh, d, rot, bf16):
    torch = torch_cuda
    g, dt = gen(torch, tokens + h + rot), torch.bfloat16 if bf16 else torch.float32
    qk = (torch.randn(tokens, h, 2 * d, generator=g) * 3).to(dt)      # query and gate halves
    kk = (torch.randn(tokens, kvh, d, generator=g) * 0.2).to(dt)
    qw, kw = torch.randn(d, generator=g) * 0.3, torch.randn(d, generator=g) * 0.3
    pos = torch.randint(0, 131072, (tokens,), generator=g, dtype=torch.int32)
    pos[0] = 0 if tokens > 1 else 131071
    wide = torch.full((tokens + 1, (h + kvh) * d + 16), 7.0, dtype=dt, device="cuda")
    qo, ko = wide[:tokens, :h * d].view(tokens, h, d), wide[:tokens, h * d:(h + kvh) * d].view(tokens, kvh, d)
    dev = [qk.cuda()[:, :, :d], kk.cuda(), qw.cuda(), kw.cuda(), pos.cuda()]
    q.qk_norm_rope_seq(qo, ko, *dev, rot)
    rope_check(torch, qo, rope_oracle(torch, qk[:, :, :d], qw, pos, rot), bf16)
    rope_check(torch, ko, rope_oracle(torch, kk, kw, pos, rot), bf16)
    assert (wide[tokens:] == 7).all() and (wide[:, (h + kvh) * d:] == 7).all()
    # head-major, and in place: the same bits
    q2, k2 = dev[0].transpose(0, 1).contiguous().transpose(0, 1), kk.cuda()
    q.qk_norm_rope_seq(q2, k2, q2, k2, *dev[2:], rot)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    # in place in the rows of one projection, queries and keys beside each other and beside others' columns
    row = torch.full((tokens, (h + kvh) * d + 16), 7.0, dtype=dt, device="cuda")
    q3, k3 = row[:, :h * d].view(tokens, h, d), row[:, h * d:(h + kvh) * d].view(tokens, kvh, d)
    q3.copy_(qk[:, :, :d]), k3.copy_(kk)          # (dev[0] may have been q2)
    q.qk_norm_rope_seq(q3, k3, q3, k3, *dev[2:], rot)
    assert torch.equal(q3, qo) and torch.equal(k3, ko) and (row[:, (h + kvh) * d:] == 7).all()


def test_norm_rope_is_the_one_token_ops(q, torch_cuda):
    """rmsnorm, rope_cos_sin and apply_rope of each head, near enough: their angles are rounded to fp32, so positions are small."""
    torch = torch_cuda
    g, d = gen(torch, 1), 256
    x, kk, w = torch.randn(4, 2, d, generator=g).cuda(), torch.randn(4, 1, d, generator=g).cuda(), torch.randn(d, generator=g).cuda()
    pos = torch.tensor([0, 1, 7, 40], dtype=torch.int32)
    qo, ko = torch.empty_like(x), torch.empty_like(kk)
    q.qk_norm_rope_seq(qo, ko, x, kk, w, w, pos.cuda())
    c, s, y = torch.empty(64, device="cuda"), torch.empty(64, device="cuda"), torch.empty(d, device="cuda")
    for t in range(4):
        q.rope_cos_sin(int(pos[t]), c, s)
        for got, src in ((qo[t, 0], x[t, 0]), (qo[t, 1], x[t, 1]), (ko[t, 0], kk[t, 0])):
            q.rmsnorm(y, src.contiguous(), w, d)
            q.apply_rope(y, c, s)
            # 24 u (|x| + |y|) on either side, and the angle's rounding: 2 u of 40
            assert (got - y).abs().max().item() <= (48 + 80) * U * 2 * y.abs().max().item()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_norm_rope_far_positions_and_bases(q, torch_cuda, bf16):
    torch = torch_cuda
    g, d, dt = gen(torch, 2), 128, torch.bfloat16 if bf16 else torch.float32
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 1 << 20, 131071, 99999999], dtype=torch.int32)
    x, kk = torch.randn(8, 2, d, generator=g).to(dt), torch.randn(8, 1, d, generator=g).to(dt)
    w = torch.zeros(d)
    for theta, rot, eps in ((1e7, 128, 1e-6), (1e4, 64, 1e-5), (2.0, 16, 0.0), (1.0, 32, 1.0), (5e8, 64, 1e-6)):
        qo, ko = torch.empty_like(x, device="cuda"), torch.empty_like(kk, device="cuda")
        q.qk_norm_rope_seq(qo, ko, x.cuda(), kk.cuda(), w.cuda(), w.cuda(), pos.cuda(), rot, theta, eps)
        # positions of 2^31 turn 2^31 / (2 pi) times at most: what 64 bits leave of that, 2^-53 2^29 of a turn, four times over
        far = 4 * 2.0 ** -24 * 2 * math.pi * 2
        for got, src in ((qo, x), (ko, kk)):
            wo, tol = rope_oracle(torch, src, w, pos, rot, theta, eps)
            rope_check(torch, got, (wo, tol + far * src.double().abs().amax(-1, keepdim=True) / torch.sqrt(src.double().square().mean(-1, keepdim=True) + eps)), bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_norm_rope_rows_on_their_own(q, torch_cuda, bf16):
    """A row of zeros stays one, a row with a NaN or an infinity is its own affair."""
    torch = torch_cuda
    g, dt = gen(torch, 3), torch.bfloat16 if bf16 else torch.float32
    x, kk = torch.randn(6, 3, 256, generator=g).to(dt).cuda(), torch.randn(6, 2, 256, generator=g).to(dt).cuda()
    w, pos = torch.randn(256, generator=g).cuda(), torch.arange(6, dtype=torch.int32, device="cuda")
    run = lambda: (lambda a, b: (q.qk_norm_rope_seq(a, b, x, kk, w, w, pos), a, b)[1:])(torch.empty_like(x), torch.empty_like(kk))
    a0, b0 = run()
    x[1, 0] = 0
    x[2, 1, 5], kk[3, 1, 200] = math.nan, math.inf
    a, b = run()
    assert (a[1, 0] == 0).all() and torch.isnan(a[2, 1]).all() and torch.isnan(b[3, 1, 200])
    a[1, 0], a[2, 1], b[3, 1] = a0[1, 0], a0[2, 1], b0[3, 1]
    assert torch.equal(a, a0) and torch.equal(b, b0)


# ------------------------------------------------------------------ the cache

def code_oracle(torch, x):
    """(codes, scales) of rows, by fp32 divisions on the CPU, as quant_rows defines them."""
    x = x.float()
    top = x.abs().amax(-1)
    s = torch.where(top > 0, top / 127.0, 1.0)
    s = torch.where((top > 0) & (s == 0), torch.tensor(2.0 ** -149), s)
    ok = torch.isfinite(x).all(-1)
    c = torch.where(ok[..., None], torch.clamp(torch.round(x / s[..., None]), -127, 127), 0.0).to(torch.int8)
    return c, torch.where(ok, s, math.nan)


def same(torch, a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def cache_new(torch, rows, kvh, d, layout):
    """(kq, ks, vq, vs) filled with what no call writes."""
    i8 = dict(dtype=torch.int8, device="cuda")
    if layout == "rows":
        kq, vq = torch.full((rows, kvh, d), -128, **i8), torch.full((rows, kvh, d), -128, **i8)
        ks, vs = torch.full((rows, kvh), -5.0, device="cuda"), torch.full((rows, kvh), -5.0, device="cuda")
    elif layout == "heads":          # head-major, scales as well
        kq, vq = (torch.full((kvh, rows, d), -128, **i8).transpose(0, 1) for _ in range(2))
        ks, vs = (torch.full((kvh, rows), -5.0, device="cuda").t() for _ in range(2))
    else:                            # keys and values of a row side by side, scales in odd places
        both = torch.full((rows, 2, kvh, d + 16), -128, **i8)
        kq, vq = both[:, 0, :, :d], both[:, 1, :, :d]
        sc = torch.full((rows, 2 * kvh + 3), -5.0, device="cuda")
        ks, vs = sc[:, 1:1 + kvh], sc[:, 2 + kvh:2 + 2 * kvh]
    return kq, ks, vq, vs


CACHE = [  # tokens, rows, kv heads, dim
    (1, 1, 1, 128), (1, 40, 2, 256), (3, 9, 1, 256), (15, 16, 3, 128), (16, 33, 8, 128), (17, 1000, 2, 256), (129, 200, 5, 128),
    (700, 900, 2, 256), (5, 4000, 40, 256),
    (3000, 3333, 3, 128), (1700, 2000, 5, 256), (8200, 9000, 1, 128),      # four rows of a token at a time
]


@pytest.mark.parametrize("tokens,rows,kvh,d", CACHE)
@pytest.mark.parametrize("layout", ["rows", "heads", "side"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_cache_write_and_read(q, torch_cuda, tokens, rows, kvh, d, layout, bf16):
    torch = torch_cuda
    g, dt = gen(torch, tokens * 3 + rows + kvh), torch.bfloat16 if bf16 else torch.float32
    row = (torch.randn(tokens, 2 * kvh * d + 32, generator=g) * torch.exp(torch.randn(tokens, 1, generator=g) * 4)).to(dt)
    kv = [row[:, a:a + kvh * d].view(tokens, kvh, d) for a in (0, kvh * d + 16)]
    dev = [row.cuda()[:, a:a + kvh * d].view(tokens, kvh, d) for a in (0, kvh * d + 16)]
    slot = torch.randperm(rows, generator=g)[:tokens].to(torch.int64)
    for i, s in ((1, -1), (4, rows), (6, 2 ** 63 - 1), (8, -2 ** 63), (10, rows + 7)):     # no places of the cache
        if i < tokens:
            slot[i] = s
    there = (slot >= 0) & (slot < rows)
    c = cache_new(torch, rows, kvh, d, layout)
    q.kv_cache_write_i8(*c, *dev, slot.cuda())
    out = [torch.full((tokens + 1, kvh, d + 16), 7.0, dtype=dt, device="cuda") for _ in range(2)]
    o = [x[:tokens, :, :d] for x in out]
    q.kv_cache_read_i8(*o, *c, slot.cuda())
    for x, cq, cs, got, full in zip(kv, c[::2], c[1::2], o, out):
        codes, sc = code_oracle(torch, x)
        wq, wsc = torch.full((rows, kvh, d), -128, dtype=torch.int8), torch.full((rows, kvh), -5.0)
        wq[slot[there]], wsc[slot[there]] = codes[there], sc[there]
        assert torch.equal(cq.cpu(), wq) and torch.equal(cs.cpu(), wsc)
        want = (codes.float() * sc[..., None]).to(dt)
        want[~there] = 7.0
        assert torch.equal(got.cpu(), want) and (full[tokens:] == 7).all() and (full[:, :, d:] == 7).all()
        # the same codes as the packer's operator gives
        if layout == "rows" and not bf16:
            pq, ps = torch.empty(tokens * kvh, d, dtype=torch.int8, device="cuda"), torch.empty(tokens * kvh, device="cuda")
            q.quant_rows(pq, ps, x.reshape(-1, d).contiguous().cuda(), tokens * kvh, d)
            assert torch.equal(pq.cpu().view(tokens, kvh, d), codes) and torch.equal(ps.cpu().view(tokens, kvh), sc)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_cache_odd_rows(q, torch_cuda, bf16, d):
    """Zeros, halves between two codes, the smallest and the largest numbers, what is not finite."""
    torch = torch_cuda
    dt = torch.bfloat16 if bf16 else torch.float32
    g = gen(torch, d)
    x = torch.randn(14, 2, d, generator=g)
    x[0] = 0.0
    x[1] = torch.arange(d) - 126.5
    x[1, :, 0] = 127.0                               # scale 1: ties go to the even code
    x[2] = torch.sign(x[2]) * 2.0 ** -149
    x[3] *= 2.0 ** -140
    x[4] *= 2.0 ** -127
    x[5] *= 1e-36
    x[6] = torch.sign(x[6]) * 3.3895314e38           # the largest bfloat16
    x[7] *= 1e30
    x[8, 0, 3], x[9, 1, d - 1], x[10, 0, 64] = math.nan, math.inf, -math.inf
    x[11] = -0.0
    x[12, :, 1:] = 0.0
    x[13] = 5.0
    x = x.to(dt)
    c = cache_new(torch, 14, 2, d, "rows")
    slot = torch.arange(14).cuda()
    q.kv_cache_write_i8(*c, x.cuda(), x.flip(0).cuda(), slot)
    for src, cq, cs in ((x, c[0], c[1]), (x.flip(0), c[2], c[3])):
        codes, sc = code_oracle(torch, src)
        assert torch.equal(cq.cpu(), codes) and same(torch, cs.cpu(), sc)
    o = [torch.empty(14, 2, d, dtype=dt, device="cuda") for _ in range(2)]
    q.kv_cache_read_i8(*o, *c, slot)
    codes, sc = code_oracle(torch, x)
    assert same(torch, o[0].cpu(), (codes.float() * sc[..., None]).to(dt))


def test_cache_read_any_codes_many_times(q, torch_cuda):
    """All codes, -128 among them, and one row named by every token."""
    torch = torch_cuda
    g = gen(torch, 4)
    kq, vq = (torch.randint(-128, 128, (50, 2, 128), generator=g, dtype=torch.int8) for _ in range(2))
    ks, vs = torch.randn(50, 2, generator=g), torch.rand(50, 2, generator=g)
    slot = torch.randint(0, 50, (400,), generator=g)
    slot[:100] = 17
    for dt in (torch.float32, torch.bfloat16):
        o = [torch.empty(400, 2, 128, dtype=dt, device="cuda") for _ in range(2)]
        q.kv_cache_read_i8(*o, kq.cuda(), ks.cuda(), vq.cuda(), vs.cuda(), slot.cuda())
        assert torch.equal(o[0].cpu(), (kq[slot].float() * ks[slot][..., None]).to(dt))
        assert torch.equal(o[1].cpu(), (vq[slot].float() * vs[slot][..., None]).to(dt))


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_cache_rows_far_apart(q, torch_cuda, bf16):
    """Rows of the cache 16 MB apart, the last behind 2^32 bytes, and a token's rows far from the next."""
    torch = torch_cuda
    g, dt, rows, ld = gen(torch, 6), torch.bfloat16 if bf16 else torch.float32, 300, 1 << 24
    far = torch.zeros((rows - 1) * ld + 512, dtype=torch.int8, device="cuda").as_strided((rows, 2, 256), (ld, 256, 1))
    vq = torch.zeros(rows, 2, 256, dtype=torch.int8, device="cuda")
    ks, vs = torch.zeros(rows, 2, device="cuda"), torch.zeros((rows - 1) * (1 << 22) + 2, device="cuda").as_strided((rows, 2), (1 << 22, 1))
    x = torch.randn(40, 2, 256, generator=g).to(dt)
    xf = torch.empty(39 * (1 << 26) + 512, dtype=dt, device="cuda").as_strided((40, 2, 256), (1 << 26, 256, 1))
    xf.copy_(x)
    slot = torch.randperm(rows, generator=g)[:40]
    slot[0] = rows - 1
    q.kv_cache_write_i8(far, ks, vq, vs, xf, xf, slot.cuda())
    codes, sc = code_oracle(torch, x)
    for cq, cs in ((far, ks), (vq, vs)):
        assert torch.equal(cq[slot.cuda()].cpu(), codes) and torch.equal(cs[slot.cuda()].cpu(), sc)
    o = torch.empty(40, 2, 256, dtype=dt, device="cuda")
    xf.zero_()
    q.kv_cache_read_i8(o, xf, far, ks, vq, vs, slot.cuda())
    want = (codes.float() * sc[..., None]).to(dt)
    assert torch.equal(o.cpu(), want) and torch.equal(xf.contiguous().cpu(), want)


# ------------------------------------------------------------------ attention over the cache

TOP = {False: 8355704.0, True: 32639.0}      # a query row's largest element, in units
MAX_Q = None                                 # the bound that a call is given; None: the longest sequence
LARGE = 1 << 26                              # a bound that asks for the form for prompts


def p_rounding(lens, G, bf16):
    """What P's rounding may take: from 128 rows a kv head on, the form for prompts may run."""
    return 0.0 if not bf16 else BF if max(lens + [0] if MAX_Q is None else [MAX_Q]) * G >= 128 else 2.0 ** -16


def attn_oracle(torch, qq, kq, ks, vq, vs, lens, ctx, at_k, scale, bf16):
    """float64 on the CPU: (out, the bound without the output's rounding)."""
    h, kvh = qq.shape[1], kq.shape[1]
    out, tol, at = torch.zeros(qq.shape, dtype=torch.float64), torch.zeros(qq.shape, dtype=torch.float64), 0
    for n, m, k0 in zip(lens, ctx, at_k):
        for hh in range(h if n and m else 0):
            c = hh // (h // kvh)
            a = qq[at:at + n, hh].double()
            b, v = (x[k0:k0 + m, c].double() * s[k0:k0 + m, c, None].double() for x, s in ((kq, ks), (vq, vs)))
            s = a @ b.t() * scale
            es = abs(scale) * a.abs().amax(-1, keepdim=True) / (2 * TOP[bf16]) * b.abs().sum(-1)[None, :] + 10 * U * s.abs()
            hide = torch.arange(m)[None, :] > torch.arange(n)[:, None] + (m - n)
            es = es.masked_fill(hide, 0.0).amax(-1, keepdim=True)
            none = hide.all(-1, keepdim=True)
            p = torch.softmax(s.masked_fill(hide, -math.inf).masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
            out[at:at + n, hh] = p @ v
            tol[at:at + n, hh] = (2 * es + (17 + math.sqrt(m)) * U + p_rounding(lens, h // kvh, bf16)) * (p @ v.abs()) + 3 * m * 2.0 ** -119
        at += n
    return out, tol


def attn_inputs(torch, seed, lens, ctx, h, kvh, d, bf16, gap=0, qscale=2.0):
    """(q, kq, ks, vq, vs) and where each sequence's keys begin."""
    g = gen(torch, seed)
    at_k, rows = [], 0
    for m in ctx:
        rows += gap
        at_k.append(rows)
        rows += m
    rows += gap
    qq = (torch.randn(sum(lens), h, d, generator=g) * qscale).to(torch.bfloat16 if bf16 else torch.float32)
    sides = []
    for _ in range(2):
        x = torch.randn(rows, kvh, d, generator=g) * torch.exp(torch.randn(rows, kvh, 1, generator=g) * 0.3)
        sides += code_oracle(torch, x) if rows else (torch.zeros(0, kvh, d, dtype=torch.int8), torch.zeros(0, kvh))
    return (qq, *sides), at_k


def attn_run(q, torch, dev, lens, ctx, at_k, scale=None, max_q=None, max_k=None, out=None):
    qq, kq = dev[:2]
    t, h, d = qq.shape
    if out is None:
        out = torch.full((t, h, d), 7.0, dtype=qq.dtype, device="cuda")
    mq = max_q if max_q is not None else MAX_Q if MAX_Q is not None else max(lens + [0])
    mk = max(ctx + [0]) if max_k is None else max_k
    nb = q.attention_seq_i8_workspace(t, len(lens), mq, mk, h, kq.shape[1], d, q.BF16 if qq.dtype is torch.bfloat16 else q.F32)
    ws = torch.full((nb,), 0xFF, dtype=torch.uint8, device="cuda")          # NaN bits
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q.attention_seq_i8(out, *dev, i32(starts(lens)), torch.tensor(at_k, dtype=torch.int64, device="cuda"), i32(ctx), ws, mq, mk, scale)
    return out


def attn_check(torch, got, want, bf16):
    wo, tol = want
    err = (got.cpu().double()[:wo.shape[0]] - wo).abs()
    lim = tol + (BF * (wo.abs() + tol) if bf16 else U * wo.abs())
    assert (err <= lim).all(), (err.max().item(), (err / lim.clamp(min=1e-30)).max().item())


def both(torch, inp, at, lens, ctx, scale, bf16):
    return [x.cuda() for x in inp], attn_oracle(torch, *inp, lens, ctx, at, scale, bf16)


def short(x):
    return str(x)[:40]


ATTN = [  # lens, keys, heads, kv heads, dim
    ([1], [1], 1, 1, 128), ([1], [1], 8, 2, 256), ([1, 1, 1], [7, 300, 1], 8, 2, 256), ([1, 1], [2500, 15], 4, 4, 128),
    ([1], [5000], 8, 2, 256), ([2, 3], [33, 64], 6, 2, 128), ([4], [1000], 16, 1, 128), ([1], [777], 32, 1, 256), ([1], [31], 2, 1, 128),
    ([1], [32], 2, 1, 256), ([1], [129], 2, 1, 128), ([15, 16, 17], [15, 16, 17], 2, 1, 128), ([64], [64], 2, 2, 256),
    ([63, 0, 65], [63, 5, 70], 4, 2, 128), ([127, 1], [127, 129], 8, 2, 256), ([129], [400], 2, 1, 256), ([200, 90], [200, 90], 3, 3, 128),
    ([300], [300], 8, 2, 256), ([33], [2000], 2, 1, 128), ([260], [261], 1, 1, 256), ([520], [520], 4, 1, 128), ([5], [5], 3, 1, 256),
    ([200, 1], [1400, 900], 8, 2, 256), ([1] * 70, [1500 - 20 * i for i in range(70)], 4, 1, 128), ([100, 7], [3000, 100], 4, 2, 128),
    ([1] * 135, [10 + i for i in range(134)] + [6000], 4, 2, 128), ([90, 600], [90, 5000], 2, 1, 128),
]


@pytest.mark.parametrize("lens,ctx,h,kvh,d", ATTN, ids=short)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention(q, torch_cuda, lens, ctx, h, kvh, d, bf16):
    torch = torch_cuda
    inp, at = attn_inputs(torch, sum(lens) + sum(ctx) + h, lens, ctx, h, kvh, d, bf16, gap=3)
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(d), bf16)
    t = sum(lens)
    out = torch.full((t + 2, h, d), 7.0, dtype=dev[0].dtype, device="cuda")
    dev[0] = torch.cat([dev[0], dev[0][:1], dev[0][:1]])            # two rows behind the last sequence
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at, out=out), want, bf16)
    assert (out[t:] == 7).all()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_rows_without_keys(q, torch_cuda, bf16, d):
    """More rows than keys: the first rows see none and come out as 0; no key at all."""
    torch = torch_cuda
    for lens, ctx in (([70, 3], [9, 0]), ([200], [1]), ([5, 1], [2, 0]), ([2], [0])):
        inp, at = attn_inputs(torch, 1, lens, ctx, 4, 2, d, bf16, gap=1)
        dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(d), bf16)
        got = attn_run(q, torch, dev, lens, ctx, at)
        attn_check(torch, got, want, bf16)
        assert (got[:lens[0] - ctx[0]] == 0).all()


def test_attention_without_a_cache(q, torch_cuda):
    torch = torch_cuda
    inp, _ = attn_inputs(torch, 1, [3], [0], 2, 1, 128, False)
    assert (attn_run(q, torch, [x.cuda() for x in inp], [3], [0], [0]) == 0).all()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("n,m", [(1, 200), (5, 300), (100, 100), (150, 260), (90, 1200)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38], ids=str)
def test_attention_hidden_keys_have_no_influence(q, torch_cuda, bf16, d, n, m, bad):
    """What stands behind a row's keys (the next tokens, rows of the cache not yet written, another sequence's) may be
    anything; a scale that is not finite reaches the rows that see it, in the heads that share it."""
    torch = torch_cuda
    lens, ctx = [n, 2], [m, 2]
    inp, at = attn_inputs(torch, 2, lens, ctx, 4, 2, d, bf16, gap=40)
    clean = attn_run(q, torch, [x.cuda() for x in inp], lens, ctx, at)
    for codes, sc in (inp[1:3], inp[3:5]):
        for r in (slice(0, at[0]), slice(at[0] + m, at[1]), slice(at[1] + 2, None)):
            codes[r], sc[r] = 127, bad
    hit = at[0] + m - max(n // 3, 1)      # a key that the first rows do not see, and the last ones do
    finite = math.isfinite(bad)
    if n > 1 and not finite:
        inp[2][hit, 0], inp[4][hit, 1] = bad, bad
    got = attn_run(q, torch, [x.cuda() for x in inp], lens, ctx, at)
    free = n if n == 1 or finite else n - max(n // 3, 1)
    assert torch.equal(got[:free], clean[:free]) and torch.equal(got[n:], clean[n:])
    if free < n:
        # V's scale: infinity times a code is one, or NaN where the code is 0, and a kernel's parts may make it NaN everywhere
        assert not torch.isfinite(got[free:n, 2:]).any() and (math.isinf(bad) or torch.isnan(got[free:n, 2:]).all())
        assert math.isinf(bad) or torch.isnan(got[free:n, :2]).all()   # K's


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention_strides(q, torch_cuda, bf16):
    """Queries inside a query and gate projection, a cache of slots with keys and values side by side, head-major ones,
    an output inside wider rows, one row of queries for all (stride 0)."""
    torch = torch_cuda
    lens, ctx, h, kvh, d = [40, 1, 70], [40, 90, 71], 4, 2, 128
    inp, _ = attn_inputs(torch, 5, lens, ctx, h, kvh, d, bf16)
    src, at, t = starts(ctx), [240, 0, 120], sum(lens)
    c = cache_new(torch, 360, kvh, d, "side")
    hm = cache_new(torch, 360, kvh, d, "heads")
    for i, m in enumerate(ctx):
        for x, a, b in zip(inp[1:], c, hm):
            a[at[i]:at[i] + m] = x[src[i]:src[i] + m].cuda()
            b[at[i]:at[i] + m] = x[src[i]:src[i] + m].cuda()
    want = attn_oracle(torch, inp[0], *[x.cpu() for x in c], lens, ctx, at, 1 / math.sqrt(d), bf16)
    gate = torch.full((t, h, 2 * d), 9.0, dtype=inp[0].dtype, device="cuda")
    gate[:, :, :d] = inp[0].cuda()
    wide = torch.full((t, h * d + 64), 7.0, dtype=inp[0].dtype, device="cuda")
    out = wide[:, 32:32 + h * d].view(t, h, d)
    attn_run(q, torch, [gate[:, :, :d], *c], lens, ctx, at, out=out)
    attn_check(torch, out, want, bf16)
    assert (wide[:, :32] == 7).all() and (wide[:, 32 + h * d:] == 7).all()
    o2 = torch.empty(h, t, d, dtype=inp[0].dtype, device="cuda").transpose(0, 1)
    attn_run(q, torch, [inp[0].transpose(0, 1).contiguous().cuda().transpose(0, 1), *hm], lens, ctx, at, out=o2)
    assert torch.equal(o2, out)
    one = inp[0][:1].expand(t, h, d)
    want = attn_oracle(torch, one, *[x.cpu() for x in c], lens, ctx, at, 1 / math.sqrt(d), bf16)
    attn_check(torch, attn_run(q, torch, [inp[0][:1].cuda().expand(t, h, d), *c], lens, ctx, at), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention_bounds_too_small_or_large(q, torch_cuda, monkeypatch, bf16):
    """max_q and max_k choose the form: any value gives the same within tolerance."""
    torch = torch_cuda
    monkeypatch.setattr(sys.modules[__name__], "MAX_Q", LARGE)      # (the bound of the form for prompts)
    lens, ctx = [1, 90, 3], [900, 90, 500]
    inp, at = attn_inputs(torch, 6, lens, ctx, 4, 2, 128, bf16)
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(128), bf16)
    for mq in (0, 1, 4, 90, 5000, LARGE):
        for mk in (0, 100, 900, 100000):
            attn_check(torch, attn_run(q, torch, dev, lens, ctx, at, max_q=mq, max_k=mk), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention_large_scores(q, torch_cuda, bf16):
    """Scores far apart (one key takes all), equal scores, a scale of 0 (the mean of the keys), a negative one, and
    scores of 2^40 (whose rounding is more than a power of two holds)."""
    torch = torch_cuda
    for scale in (4.0, 0.0, -0.3, 1e10):
        inp, at = attn_inputs(torch, 7, [20, 1], [30, 400], 2, 1, 128, bf16)
        dev, want = both(torch, inp, at, [20, 1], [30, 400], scale, bf16)
        attn_check(torch, attn_run(q, torch, dev, [20, 1], [30, 400], at, scale=scale), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -120, 2.0 ** -64, 2.0 ** -62, 1e-3, 1e30])
def test_attention_queries_of_any_size(q, torch_cuda, bf16, size):
    """Rows of very small and very large elements beside ordinary ones, rows of zeros, single elements; K's scales make up for it."""
    torch = torch_cuda
    lens, ctx, d = [30, 1], [50, 300], 256
    inp, at = attn_inputs(torch, 8, lens, ctx, 2, 1, d, bf16)
    inp = list(inp)
    inp[0] = inp[0] * size
    inp[0][3] = 0.0
    inp[0][4, :, 1:] = 0.0
    inp[0][5] = torch.sign(inp[0][5]) * size
    inp[2] = inp[2] * min(max(1.0 / size, 1e-30), 1e30)
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(d), bf16)
    wo, tol = want
    if size < 2.0 ** -125:     # the row's unit has steps of 2^-149: up to 2^-150 off, times sums of 256 codes of 128 and 30 (scales up to 1e30)
        tol = tol + 1e-6 * inp[4].abs().max().double() * 127
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at), (wo, tol), bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, LARGE])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_keys_near_the_end_of_the_range(q, torch_cuda, monkeypatch, bf16, max_q, d):
    """Scales of K near 2^106: a sum of digits times codes (2^23 and more) times the scale is beyond a float, the score is not."""
    torch = torch_cuda
    monkeypatch.setattr(sys.modules[__name__], "MAX_Q", max_q)      # (the bound of the form)
    lens, ctx = [70, 1], [150, 300]
    inp, at = attn_inputs(torch, 16, lens, ctx, 2, 1, d, bf16)
    inp = list(inp)
    inp[0] = inp[0] * 2.0 ** -105
    inp[2] = inp[2] * 2.0 ** 111
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(d), bf16)
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at, max_q=max_q), want, bf16)
    inp[2][40:] = inp[2][40:] * 2.0 ** -111     # these scales among ordinary ones: stages with and without them
    inp[0] = inp[0] * 2.0 ** 100
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(d), bf16)
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at, max_q=max_q), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention_any_codes(q, torch_cuda, bf16):
    """All codes, -128 among them, and the largest sums that there are."""
    torch = torch_cuda
    g = gen(torch, 9)
    for d in (128, 256):
        inp, at = attn_inputs(torch, 9, [40], [70], 2, 1, d, bf16)
        kq, vq = (torch.randint(-128, 128, inp[1].shape, generator=g, dtype=torch.int8) for _ in range(2))
        kq[7], kq[8], vq[9] = -128, 127, -128
        inp = (inp[0], kq, torch.full((70, 1), 1e-3), vq, inp[4])
        inp[0][5] = -2.0
        inp[0][6] = 2.0
        dev, want = both(torch, inp, at, [40], [70], 0.1, bf16)
        attn_check(torch, attn_run(q, torch, dev, [40], [70], at, scale=0.1), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=str)
def test_attention_query_rows_on_their_own(q, torch_cuda, bf16, bad):
    torch = torch_cuda
    lens, ctx = [70, 1], [90, 300]
    inp, at = attn_inputs(torch, 10, lens, ctx, 4, 2, 128, bf16)
    clean = attn_run(q, torch, [x.cuda() for x in inp], lens, ctx, at)
    for r, h, e in ((0, 1, 5), (33, 3, 127), (70, 0, 0)):
        inp[0][r, h, e] = bad
    got = attn_run(q, torch, [x.cuda() for x in inp], lens, ctx, at)
    for r, h in ((0, 1), (33, 3), (70, 0)):
        assert torch.isnan(got[r, h]).all()
        got[r, h] = clean[r, h]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,m", [(1, 40), (30, 40), (90, 600)])
def test_attention_bad_ranges(q, torch_cuda, bf16, n, m):
    """Key ranges outside the array give NaN in that sequence's rows; row bounds out of order leave rows alone."""
    torch = torch_cuda
    lens, ctx = [n, n, n], [m, m, m]
    inp, at = attn_inputs(torch, 8, lens, ctx, 2, 1, 128, bf16)
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(128), bf16)
    part = lambda a, b: (want[0][a:b], want[1][a:b])
    for start, length in ((-1, m), (2 * m + 1, m), (m, -1), (1 << 40, m), (0, 3 * m + 1)):
        k2, c2 = list(at), list(ctx)
        k2[1], c2[1] = start, length
        got = attn_run(q, torch, dev, lens, c2, k2, max_k=m)
        assert torch.isnan(got[n:2 * n]).all()
        attn_check(torch, got[:n], part(0, n), bf16)
        attn_check(torch, got[2 * n:], part(2 * n, 3 * n), bf16)
    out = torch.full((3 * n, 2, 128), 7.0, dtype=dev[0].dtype, device="cuda")
    ws = torch.empty(q.attention_seq_i8_workspace(3 * n, 3, n, m, 2, 1, 128), dtype=torch.uint8, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q.attention_seq_i8(out, *dev, i32([0, n, 3 * n + 1, 3 * n]), torch.tensor(at, dtype=torch.int64, device="cuda"), i32(ctx), ws, n, m)
    attn_check(torch, out[:n], part(0, n), bf16)
    assert (out[n:] == 7).all()


# The form for prompts, whatever the lengths.

@pytest.fixture
def prompts(monkeypatch):
    monkeypatch.setattr(sys.modules[__name__], "MAX_Q", LARGE)


@pytest.mark.parametrize("lens,ctx,h,kvh,d", ATTN + [
    ([700], [3000], 8, 2, 256), ([130, 1], [4100, 2000], 2, 2, 128), ([40], [9000], 4, 4, 128), ([1023, 0, 513], [1023, 4, 800], 4, 1, 256),
    ([257], [700], 12, 4, 256)], ids=short)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_form(prompts, q, torch_cuda, lens, ctx, h, kvh, d, bf16):
    test_attention(q, torch_cuda, lens, ctx, h, kvh, d, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_prompt_form_rows_without_keys(prompts, q, torch_cuda, bf16, d):
    test_attention_rows_without_keys(q, torch_cuda, bf16, d)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,m", [(1, 200), (5, 300), (100, 100), (150, 260), (90, 1200)])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 3e38], ids=str)
def test_prompt_form_hidden_keys_have_no_influence(prompts, q, torch_cuda, bf16, d, n, m, bad):
    test_attention_hidden_keys_have_no_influence(q, torch_cuda, bf16, d, n, m, bad)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_form_strides(prompts, q, torch_cuda, bf16):
    test_attention_strides(q, torch_cuda, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_form_large_scores_and_any_codes(prompts, q, torch_cuda, bf16):
    test_attention_large_scores(q, torch_cuda, bf16)
    test_attention_any_codes(q, torch_cuda, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -64, 1e30])
def test_prompt_form_queries_of_any_size(prompts, q, torch_cuda, bf16, size):
    test_attention_queries_of_any_size(q, torch_cuda, bf16, size)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=str)
def test_prompt_form_query_rows_on_their_own(prompts, q, torch_cuda, bf16, bad):
    test_attention_query_rows_on_their_own(q, torch_cuda, bf16, bad)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,m", [(30, 40), (90, 600)])
def test_prompt_form_bad_ranges(prompts, q, torch_cuda, bf16, n, m):
    test_attention_bad_ranges(q, torch_cuda, bf16, n, m)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_k", [129, 300, 700, 20000])
def test_prompt_form_places_in_the_workspace(q, torch_cuda, prompts, bf16, max_k):
    """max_k is a bound on what the workspace holds, not on the keys: what finds no place there is not split."""
    torch = torch_cuda
    lens, ctx = [70, 3, 0, 129, 64, 1, 70, 2, 300], [900, 3, 10, 1500, 64, 2500, 400, 2, 3000]
    inp, at = attn_inputs(torch, 15, lens, ctx, 4, 2, 128, bf16)
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(128), bf16)
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at, max_q=LARGE, max_k=max_k), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, LARGE])
def test_attention_of_many_sequences(q, torch_cuda, monkeypatch, bf16, max_q):
    """More than the 64 sequences that a wave looks at together; long ones among empty and short ones."""
    torch = torch_cuda
    monkeypatch.setattr(sys.modules[__name__], "MAX_Q", max_q)
    lens = [(5 * i) % 9 for i in range(150)]
    ctx = [n + (7 * i) % 40 for i, n in enumerate(lens)]
    for i, n, m in ((3, 140, 900), (64, 1, 1500), (149, 70, 70)):
        lens[i], ctx[i] = n, m
    inp, at = attn_inputs(torch, 10, lens, ctx, 4, 2, 128, bf16)
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(128), bf16)
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at, max_q=max_q), want, bf16)


@pytest.mark.parametrize("ld", [1 << 22, (1 << 24) - 16])
@pytest.mark.parametrize("max_q", [1, LARGE])
def test_attention_rows_far_apart(q, torch_cuda, monkeypatch, ld, max_q):
    """Rows of codes 4 and 16 MB apart (the largest stride), the last ones behind 2^32 bytes; scales 1 MB apart."""
    torch = torch_cuda
    monkeypatch.setattr(sys.modules[__name__], "MAX_Q", max_q)
    rows = 1100 if ld == 1 << 22 else 300
    lens, ctx, at = [40, 1, 200], [rows, 250, rows - 60], [0, rows - 250, 60]
    inp, _ = attn_inputs(torch, 13, lens, [rows], 4, 2, 128, True)
    want = attn_oracle(torch, *inp, lens, ctx, at, 1 / math.sqrt(128), True)
    dev = [inp[0].cuda()]
    for x in inp[1:]:
        step = ld if x.dtype is torch.int8 else 1 << 18
        far = torch.empty((rows - 1) * step + x[0].numel(), dtype=x.dtype, device="cuda").as_strided(x.shape, (step, *x.stride()[1:]))
        far.copy_(x)
        dev.append(far)
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at, max_q=max_q), want, True)


# ------------------------------------------------------------------ calls that cannot be answered

def test_refused_tensors(q, torch_cuda, monkeypatch):
    """Other types, shapes and strides; operands in host memory or on another device, each of them; parameters are tensors
    like others."""
    torch = torch_cuda
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")
    i8, i32, i64 = torch.int8, torch.int32, torch.int64
    cache = lambda: [z(9, 1, 128, dt=i8), z(9, 1), z(9, 1, 128, dt=i8), z(9, 1)]
    rope = [z(4, 2, 128), z(4, 1, 128), z(4, 2, 128), z(4, 1, 128), z(128), z(128), z(4, dt=i32)]
    write = [*cache(), z(4, 1, 128), z(4, 1, 128), torch.arange(4, device="cuda")]
    read = [z(4, 1, 128), z(4, 1, 128), *cache(), torch.arange(4, device="cuda")]
    attn = [z(4, 2, 128), z(4, 2, 128), *cache(), z(2, dt=i32), z(1, dt=i64), z(1, dt=i32), None, 4, 9]
    calls = [(q.qk_norm_rope_seq, rope, 7), (q.kv_cache_write_i8, write, 7), (q.kv_cache_read_i8, read, 7), (q.attention_seq_i8, attn, 9)]
    for f, ops, n in calls:
        f(*ops)
        f(*[torch.nn.Parameter(x, requires_grad=False) if k < n else x for k, x in enumerate(ops)])
        for i in range(n):
            put = lambda x: [x if k == i else y for k, y in enumerate(ops)]
            with pytest.raises(TypeError):
                f(*put(ops[i].cpu()))
            with pytest.raises(TypeError):
                f(*put(ops[i].half() if ops[i].is_floating_point() else ops[i].to(torch.int16)))
            with pytest.raises(ValueError):
                f(*put(z(*[s + 1 for s in ops[i].shape], dt=ops[i].dtype)))
            if ops[i].shape[-1] == 128:
                with pytest.raises(ValueError):
                    f(*put(z(*ops[i].shape[:-1], 256, dt=ops[i].dtype)[..., ::2]))
    for f, ops, _ in calls[1:3]:
        with pytest.raises(q.QHError):
            f(*[z(9, 1, 136, dt=i8)[..., 8:] if x.dtype is i8 else x for x in ops])      # 8 bytes off
    with pytest.raises(q.QHError):
        q.kv_cache_write_i8(*[z(1, 1, 128, dt=i8).expand(9, 1, 128) if k == 0 else x for k, x in enumerate(write)])   # one row for all
    with pytest.raises(q.QHError):
        q.kv_cache_write_i8(*[write[2] if k == 0 else x for k, x in enumerate(write)])   # keys and values in one place
    with pytest.raises(q.QHError):
        q.qk_norm_rope_seq(*rope, 24)
    with pytest.raises(q.QHError):
        q.qk_norm_rope_seq(*[x[..., :64].contiguous() if x.shape[-1] == 128 else x for x in rope])
    with pytest.raises(TypeError):
        q.attention_seq_i8(*attn[:9], torch.empty(64, dtype=torch.uint8), 4, 9)
    with pytest.raises(q.QHError):
        q.attention_seq_i8(*attn[:9], torch.empty(256, dtype=torch.uint8, device="cuda"), 4, 1000)
    with pytest.raises(q.QHError):
        q.attention_seq_i8(*attn[:10], 4, 1 << 40)
    far = torch.empty(8 * (1 << 24) + 128, dtype=i8, device="cuda").as_strided((9, 1, 128), (1 << 24, 128, 1))
    with pytest.raises(q.QHError):
        q.attention_seq_i8(*[far if k == 2 else x for k, x in enumerate(attn)])
    monkeypatch.setattr(q._Short, "device", lambda: 1)
    for f, ops, _ in calls:
        with pytest.raises(ValueError):
            f(*ops)


# ------------------------------------------------------------------ streams, graphs, together

def test_two_streams(q, torch_cuda):
    """Calls beside one another on two streams, each with operands and a workspace of its own, over one cache that both read."""
    torch = torch_cuda
    lens, ctx = [80, 5], [80, 900]
    inp, at = attn_inputs(torch, 12, lens, ctx, 8, 2, 256, True)
    dev, want = both(torch, inp, at, lens, ctx, 1 / 16, True)
    slot = torch.arange(980, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    res = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                c = cache_new(torch, 980, 2, 256, "rows")
                o = [torch.empty(980, 2, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
                q.kv_cache_read_i8(*o, *dev[1:], slot)
                q.kv_cache_write_i8(*c, *o, slot)
                res.append((attn_run(q, torch, dev, lens, ctx, at), attn_run(q, torch, dev, lens, ctx, at, max_q=LARGE), o, c))
    torch.cuda.synchronize()
    for a, b, o, c in res:
        attn_check(torch, a, want, True)
        attn_check(torch, b, want, True)
        assert torch.equal(a, res[0][0]) and torch.equal(b, res[0][1])
        assert torch.equal(o[0].cpu(), (inp[1].float() * inp[2][..., None]).bfloat16())
        assert torch.equal(c[0].cpu(), code_oracle(torch, o[0].cpu())[0])


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [4, LARGE])
def test_attention_replayed(q, torch_cuda, monkeypatch, bf16, max_q):
    """A call whose keys are split (a second kernel joins them), captured once and replayed with other lengths and ranges on the
    device, eager work between: the eager call's bits each time, rows behind the last sequence as they were."""
    torch = torch_cuda
    monkeypatch.setattr(sys.modules[__name__], "MAX_Q", max_q)      # (the bound of the form)
    h, kvh, d, rows, t, n, max_k = 4, 2, 128, 6000, 12, 4, 6000
    inp, _ = attn_inputs(torch, 17, [t], [rows], h, kvh, d, bf16)
    dev = [x.cuda() for x in inp]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cu, at, kl = i32([0] * (n + 1)), torch.zeros(n, dtype=torch.int64, device="cuda"), i32([0] * n)
    out = torch.empty(t, h, d, dtype=dev[0].dtype, device="cuda")
    nb = q.attention_seq_i8_workspace(t, n, max_q, max_k, h, kvh, d, q.BF16 if bf16 else q.F32)
    assert nb > 0
    ws = [torch.full((nb,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]     # the graph's own, and one for eager calls
    call = lambda w: q.attention_seq_i8(out, *dev, cu, at, kl, w, max_q, max_k)
    call(ws[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(ws[0])
    for lens, ctx, k0 in (([1, 1, 1, 1], [5000, 3, 600, 4000], [0, 17, 5400, 2000]), ([4, 0, 3, 1], [6000, 9, 2, 1], [0, 5, 5998, 3]),
                          ([0, 0, 0, 2], [0, 0, 0, 3100], [0, 0, 0, 2900]), ([4, 4, 4, 0], [900, 800, 700, 0], [1, 2000, 5300, 0])):
        cu.copy_(i32(starts(lens))), at.copy_(torch.tensor(k0)), kl.copy_(i32(ctx))
        got = []
        for run in (lambda: call(ws[1]), graph.replay, graph.replay):
            out.fill_(7.0)
            run()
            torch.cuda.synchronize()
            got.append(out.clone())
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and (got[0][sum(lens):] == 7).all()
        want = attn_oracle(torch, inp[0][:sum(lens)], *inp[1:], lens, ctx, k0, 1 / math.sqrt(d), bf16)
        attn_check(torch, got[0], want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_layer_over_the_cache(q, torch_cuda, bf16):
    """The operators as a layer chains them: one projection's queries, keys and values normalised, rotated, written into
    slots of the cache and attended to; prompts of several sequences first, then single tokens from a graph that is replayed with
    other positions, slots and lengths on the device (some places of the batch unused), eager work between.  Every replay gives the
    eager call's bits, and each stage its bound against 64 bits on its own inputs."""
    torch = torch_cuda
    h, kvh, d, room, n_seq, dt = 8, 2, 128, 200, 4, torch.bfloat16 if bf16 else torch.float32
    g = gen(torch, 21)
    lens = [90, 1, 0, 33]
    qw, kw = (torch.randn(d, generator=g) * 0.2 for _ in range(2))
    c = cache_new(torch, n_seq * room, kvh, d, "side")
    for x in c[1::2]:
        x.fill_(math.nan)                          # rows that were never written hold anything
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    k_start = torch.arange(n_seq, device="cuda") * room

    def stage_check(row, pos, out, qn, kn, vv, cu, ctx):
        rope_check(torch, qn, rope_oracle(torch, row[:, :h].cpu(), qw, pos, 64), bf16)
        rope_check(torch, kn, rope_oracle(torch, row[:, h:h + kvh].cpu(), kw, pos, 64), bf16)
        ln = [b - a for a, b in zip(cu, cu[1:])]
        n = cu[-1]
        host = [x.cpu() for x in c]
        for x in host[1::2]:
            x[x.isnan()] = 0.0
        attn_check(torch, out[:n], attn_oracle(torch, qn[:n].cpu(), *host, ln, ctx, k_start.tolist(), 1 / math.sqrt(d), bf16), bf16)

    def step(row, pos, slot, cu, kl, out, ws, mq):
        t = row.shape[0]
        qn, kn = torch.empty(t, h, d, dtype=dt, device="cuda"), torch.empty(t, kvh, d, dtype=dt, device="cuda")
        q.qk_norm_rope_seq(qn, kn, row[:, :h], row[:, h:h + kvh], qw_d, kw_d, pos)
        q.kv_cache_write_i8(*c, kn, row[:, h + kvh:], slot)
        q.attention_seq_i8(out, qn, *c, cu, k_start, kl, ws, mq, room)
        return qn, kn

    qw_d, kw_d = qw.cuda(), kw.cuda()
    t = sum(lens)
    row = torch.randn(t, h + 2 * kvh, d, generator=g).to(dt).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32)
    slot = pos.long() + torch.tensor(sum([[i] * n for i, n in enumerate(lens)], [])) * room
    out = torch.full((t, h, d), 7.0, dtype=dt, device="cuda")
    ws = torch.empty(q.attention_seq_i8_workspace(t, n_seq, max(lens), room, h, kvh, d), dtype=torch.uint8, device="cuda")
    qn, kn = step(row, pos.cuda(), slot.cuda(), i32(starts(lens)), i32(lens), out, ws, max(lens))
    stage_check(row, pos, out, qn, kn, None, starts(lens), lens)
    codes, sc = code_oracle(torch, kn.cpu())
    assert torch.equal(c[0][slot.cuda()].cpu(), codes) and torch.equal(c[1][slot.cuda()].cpu(), sc)

    # single tokens
    row1, pos1, slot1 = torch.zeros(n_seq, h + 2 * kvh, d, dtype=dt, device="cuda"), i32([0] * n_seq), torch.full((n_seq,), -1, device="cuda")
    cu1, kl1, out1 = i32([0] * (n_seq + 1)), i32([0] * n_seq), torch.empty(n_seq, h, d, dtype=dt, device="cuda")
    ws1 = torch.empty(q.attention_seq_i8_workspace(n_seq, n_seq, 1, room, h, kvh, d), dtype=torch.uint8, device="cuda")
    args = (row1, pos1, slot1, cu1, kl1, out1, ws1, 1)
    step(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qn1, kn1 = step(*args)
    held = list(lens)
    for it in range(6):
        live = [i for i in range(n_seq) if (it + i) % 3 != 0]       # the sequences with a token now, at the batch's first places
        new = torch.randn(n_seq, h + 2 * kvh, d, generator=g).to(dt)
        row1.copy_(new)
        p = [held[i] for i in live] + [0] * (n_seq - len(live))
        pos1.copy_(i32(p))
        slot1.copy_(torch.tensor([i * room + held[i] for i in live] + [-1] * (n_seq - len(live)), device="cuda"))
        for i in live:
            held[i] += 1
        cu = [0]
        for i in range(n_seq):
            cu.append(cu[-1] + (i in live))
        cu1.copy_(i32(cu)), kl1.copy_(i32(held))
        before = [x.clone() for x in c]
        res = []
        for run in (lambda: step(*args), lambda: (graph.replay(), (qn1, kn1))[1], lambda: (graph.replay(), (qn1, kn1))[1]):
            for x, b in zip(c, before):
                x.copy_(b)
            out1.fill_(7.0)
            got = run()
            torch.cuda.synchronize()
            res.append([x.clone() for x in (out1, *got, *c)])
        for r in res[1:]:
            assert all(same(torch, a, b) for a, b in zip(r, res[0]))
        assert (out1[len(live):] == 7).all()
        stage_check(row1, pos1.cpu(), out1, res[0][1], res[0][2], None, cu, held)


# ------------------------------------------------------------------ rows of a wave are their own affair

@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, LARGE])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_large_scores_of_other_rows(q, torch_cuda, bf16, max_q, d):
    """Scores of 2^18 to 2^20 whose keys differ by a few powers of two, where a product rounded before it is subtracted and one
    that is not give different probabilities; a key behind a row takes the rows that see it past 2^20.  The rows that do not
    keep their bits."""
    torch = torch_cuda
    g, n, h, kvh, hit, u = gen(torch, 22), 100, 4, 2, 67, 16
    k0 = torch.randint(20, 128, (kvh, d), generator=g) * (1 - 2 * torch.randint(0, 2, (kvh, d), generator=g))
    kq = k0.expand(n, kvh, d).clone()
    kq[..., :u] = torch.randint(-127, 128, (n, kvh, u), generator=g)
    qq = torch.sign(k0).float().repeat_interleave(h // kvh, 0) * (0.5 + 0.5 * torch.rand(n, h, d, generator=g))
    qq[..., :u] = torch.randn(n, h, u, generator=g) * 2.0 ** -13 * d / 128
    ks, vs = torch.full((n, kvh), 2.0 ** -7), torch.rand(n, kvh, generator=g) + 0.5
    vq = torch.randint(-127, 128, (n, kvh, d), generator=g)
    inp = [qq.to(torch.bfloat16 if bf16 else torch.float32), kq.to(torch.int8), ks, vq.to(torch.int8), vs]
    dots = torch.einsum("thd,mhd->htm", inp[0].double(), kq.repeat_interleave(h // kvh, 1).double()) * 2.0 ** -7
    scale = 0.95 * 2.0 ** 20 / math.log2(math.e) / dots.max().item()
    p = torch.softmax((dots * scale)[:, hit - 3:hit, :hit - 3], -1).amax(-1)
    assert dots.min() * scale * math.log2(math.e) > 2.0 ** 18 and p.median() < 0.7      # several keys have a part in a row
    clean = attn_run(q, torch, [x.cuda() for x in inp], [n], [n], [0], scale=scale, max_q=max_q)
    inp[2][hit] *= 16
    got = attn_run(q, torch, [x.cuda() for x in inp], [n], [n], [0], scale=scale, max_q=max_q)
    assert torch.equal(got[:hit], clean[:hit])


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, LARGE])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("bad_q", [math.nan, math.inf], ids=str)
@pytest.mark.parametrize("bad_k", [math.nan, math.inf, 2.0 ** 97], ids=str)
def test_attention_bad_queries_beside_bad_scales(q, torch_cuda, bf16, max_q, d, bad_q, bad_k):
    """Query rows that are not finite, one before and one behind a key of the same 32 whose scale is large or not finite:
    both are NaN, and the rows that do not see the key keep their bits."""
    torch = torch_cuda
    lens, ctx = [70, 1], [90, 300]
    inp, at = attn_inputs(torch, 23, lens, ctx, 4, 2, d, bf16)
    clean = attn_run(q, torch, [x.cuda() for x in inp], lens, ctx, at, max_q=max_q)
    inp[2][at[0] + 28, 0] = bad_k                  # the tokens from 8 on see it
    inp[0][3, 1, 5], inp[0][50, 0, d - 1] = bad_q, bad_q
    got = attn_run(q, torch, [x.cuda() for x in inp], lens, ctx, at, max_q=max_q)
    assert torch.isnan(got[3, 1]).all() and torch.isnan(got[50, 0]).all()
    got[3, 1] = clean[3, 1]
    assert torch.equal(got[:8], clean[:8]) and torch.equal(got[:, 2:], clean[:, 2:]) and torch.equal(got[70:], clean[70:])


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, LARGE])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("bad", [2.0 ** 97, 3e38, math.inf, math.nan], ids=str)
def test_attention_small_scales_beside_hidden_large_ones(q, torch_cuda, bf16, max_q, d, bad):
    """Queries near 2^100 and scales of K near 2^-104, where a scale moved down by 2^32 would lose bits: a large scale of a key
    behind them has no influence; and queries near 2^115, whose unit times 2^32 is beyond a float."""
    torch = torch_cuda
    lens, ctx = [70, 1], [90, 300]
    inp, at = attn_inputs(torch, 24, lens, ctx, 4, 2, d, bf16)
    inp = list(inp)
    for up in (100, 115):
        now = list(inp)
        now[0], now[2] = inp[0] * 2.0 ** up, inp[2] * 2.0 ** -(up + 4)
        clean = attn_run(q, torch, [x.cuda() for x in now], lens, ctx, at, max_q=max_q)
        attn_check(torch, clean, attn_oracle(torch, *now, lens, ctx, at, 1 / math.sqrt(d), bf16), bf16)
        now[2] = now[2].clone()
        now[2][at[0] + 28] = bad                        # the tokens from 8 on see it
        got = attn_run(q, torch, [x.cuda() for x in now], lens, ctx, at, max_q=max_q)
        assert torch.equal(got[:8], clean[:8]) and torch.equal(got[70:], clean[70:])


@pytest.mark.parametrize("single,keys,part", [(31, 6000, 300), (60, 6000, 300), (8, 4000, 20)])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_single_tokens_beside_a_part_of_a_prompt(q, torch_cuda, d, single, keys, part):
    """bfloat16: single tokens keep the two parts of P (2^-16) beside a part of a prompt, as on their own.  Queries of 0 take the mean
    of the values: three of four keys hold c x and the fourth -3 c x, so that what rounding leaves of c and of 3 c is all there is."""
    torch = torch_cuda
    lens, ctx, h, kvh = [1] * single + [part], [keys - 4 * i for i in range(single)] + [part], 8, 2
    inp, at = attn_inputs(torch, 25, lens, ctx, h, kvh, d, True)
    g = gen(torch, 26)
    inp[0][:single] = 0.0
    for i in range(single):
        r = slice(at[i], at[i] + ctx[i])
        x, c = inp[3][at[i]].clone(), torch.rand(kvh, generator=g) + 0.5
        inp[3][r], inp[4][r] = x, c
        inp[3][at[i] + 3:at[i] + ctx[i]:4], inp[4][at[i] + 3:at[i] + ctx[i]:4] = -x, 3 * c
    got = attn_run(q, torch, [x.cuda() for x in inp], lens, ctx, at)
    want = attn_oracle(torch, inp[0][:single], *inp[1:], lens[:single], ctx[:single], at[:single], 1 / math.sqrt(d), True)   # (its max_q is 1)
    attn_check(torch, got[:single], want, True)


@pytest.fixture
def two_parts(monkeypatch):
    """The bound of the form for few rows: P in two parts whatever the number of rows."""
    monkeypatch.setattr(sys.modules[__name__], "p_rounding", lambda lens, G, bf16: 2.0 ** -16 if bf16 else 0.0)


@pytest.mark.parametrize("lens,ctx,h,kvh,d", ATTN, ids=short)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_few_rows_keep_two_parts(two_parts, q, torch_cuda, lens, ctx, h, kvh, d, bf16):
    """All of these take the form for few rows by their own lengths.  Queries are small, so that their own rounding does not hide P's."""
    torch = torch_cuda
    inp, at = attn_inputs(torch, sum(lens) + sum(ctx) + h, lens, ctx, h, kvh, d, bf16, gap=3, qscale=0.02)
    dev, want = both(torch, inp, at, lens, ctx, 1 / math.sqrt(d), bf16)
    attn_check(torch, attn_run(q, torch, dev, lens, ctx, at), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,past,h,kvh,d", [
    (2200, 0, 8, 8, 128), (500, 1490, 8, 2, 256),                                 # few rows, the last before the form changes
    (2300, 0, 8, 2, 256), (512, 3500, 8, 2, 256), (2900, 0, 8, 8, 128),           # prompts in bfloat16 (and in fp32 behind a prefix)
])
def test_attention_on_both_sides_of_the_form(q, torch_cuda, monkeypatch, n, past, h, kvh, d, bf16):
    """The form that a call takes by its own sizes, at the bound of that form."""
    torch = torch_cuda
    if n <= 500 or n == 2200:
        monkeypatch.setattr(sys.modules[__name__], "p_rounding", lambda lens, G, bf16: 2.0 ** -16 if bf16 else 0.0)
    inp, at = attn_inputs(torch, n, [n], [n + past], h, kvh, d, bf16, gap=5, qscale=0.02)
    dev, want = both(torch, inp, at, [n], [n + past], 1 / math.sqrt(d), bf16)
    attn_check(torch, attn_run(q, torch, dev, [n], [n + past], at), want, bf16)


@pytest.mark.parametrize("d", [128, 256])
def test_cache_rows_are_quant_rows_at_any_size(q, torch_cuda, d):
    """The packer's operator and the cache's agree bit for bit from the smallest rows whose scale is not 0 in fp32 on."""
    torch = torch_cuda
    g, n = gen(torch, d + 1), 260
    x = torch.randn(n, 1, d, generator=g) * (2.0 ** (torch.arange(n).double() - 142)).float()[:, None, None]
    x = torch.where(torch.isfinite(x), x, 1.0)
    assert (x.abs().amax(-1) / 127 > 0).all()
    c = cache_new(torch, n, 1, d, "rows")
    q.kv_cache_write_i8(*c, x.cuda(), x.cuda(), torch.arange(n, device="cuda"))
    pq, ps = torch.empty(n, d, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    q.quant_rows(pq, ps, x.reshape(n, d).cuda(), n, d)
    for codes, sc in ((c[0], c[1]), (c[2], c[3])):
        assert torch.equal(codes[:, 0], pq) and torch.equal(sc[:, 0], ps)


@pytest.mark.parametrize("tokens,h,kvh,d,rot", [
    (1, 1, 1, 256, 64), (513, 2, 2, 128, 32), (2, 3, 1, 128, 128), (5000, 1, 1, 256, 64),       # a wave whose rows it takes at once
    (1900, 32, 8, 128, 64), (1800, 20, 1, 256, 96), (4100, 8, 2, 256, 64), (4097, 4, 1, 256, 16)], ids=str)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_norm_rope_numbers_of_waves(q, torch_cuda, tokens, h, kvh, d, rot, bf16):
    test_norm_rope(q, torch_cuda, tokens, h, kvh, d, rot, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, LARGE])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_inputs_that_repeat(q, torch_cuda, bf16, max_q, d):
    """Strides of 0: one scale for all rows or for all heads, one row of codes for all, one head of keys for two; the first
    sequence behind rows of none; sequences whose keys are the same rows."""
    torch = torch_cuda
    lens, ctx, h, kvh, rows = [40, 1, 70], [150, 400, 290], 4, 2, 420
    at = [20, 20, 100]
    inp, _ = attn_inputs(torch, 31, lens, [rows], h, kvh, d, bf16)
    qq, kq, ks, vq, vs = inp
    for host in ((kq, ks[:1].expand(rows, kvh), vq, vs[:, :1].expand(rows, kvh)), (kq[:, :1].expand(rows, kvh, d), ks, vq[5:6].expand(rows, kvh, d), vs),
                 (kq[7:8].expand(rows, kvh, d), ks[3:4, :1].expand(rows, kvh), vq, vs)):
        dev = [qq.cuda()]
        for x in host:      # the same strides on the device
            base = x[tuple(slice(0, 1) if s == 0 else slice(None) for s in x.stride())].contiguous().cuda()
            dev.append(base.expand(x.shape))
            assert 0 in dev[-1].stride() or 0 not in x.stride()
        want = attn_oracle(torch, qq, *host, lens, ctx, at, 1 / math.sqrt(d), bf16)
        pre = 3
        out = torch.full((pre + sum(lens), h, d), 7.0, dtype=qq.dtype, device="cuda")
        dev[0] = torch.cat([dev[0][:pre], dev[0]])
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        ws = torch.empty(q.attention_seq_i8_workspace(out.shape[0], 3, max_q, rows, h, kvh, d), dtype=torch.uint8, device="cuda")
        q.attention_seq_i8(out, *dev, i32([pre + x for x in starts(lens)]), torch.tensor(at, dtype=torch.int64, device="cuda"), i32(ctx), ws, max_q, rows)
        assert (out[:pre] == 7).all()
        attn_check(torch, out[pre:], want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_norms_and_cache_inputs_that_repeat(q, torch_cuda, bf16):
    """Strides of 0 in what is read: one row of queries for all tokens, one head of keys for all, one row of new values for all tokens,
    one scale for the cache's rows."""
    torch = torch_cuda
    g, dt = gen(torch, 32), torch.bfloat16 if bf16 else torch.float32
    x, y = torch.randn(1, 4, 128, generator=g).to(dt), torch.randn(30, 1, 128, generator=g).to(dt)
    w, pos = torch.randn(128, generator=g), torch.arange(30, dtype=torch.int32)
    qo, ko = torch.empty(30, 4, 128, dtype=dt, device="cuda"), torch.empty(30, 2, 128, dtype=dt, device="cuda")
    q.qk_norm_rope_seq(qo, ko, x.cuda().expand(30, 4, 128), y.cuda().expand(30, 2, 128), w.cuda(), w.cuda(), pos.cuda())
    rope_check(torch, qo, rope_oracle(torch, x.expand(30, 4, 128), w, pos, 64), bf16)
    rope_check(torch, ko, rope_oracle(torch, y.expand(30, 2, 128), w, pos, 64), bf16)
    c = cache_new(torch, 40, 2, 128, "rows")
    slot = torch.randperm(40, generator=g)[:30]
    q.kv_cache_write_i8(*c, y.cuda().expand(30, 2, 128), x[:, :2].cuda().expand(30, 2, 128), slot.cuda())
    for src, cq, cs in ((y.expand(30, 2, 128), c[0], c[1]), (x[:, :2].expand(30, 2, 128), c[2], c[3])):
        codes, sc = code_oracle(torch, src)
        assert torch.equal(cq[slot.cuda()].cpu(), codes) and torch.equal(cs[slot.cuda()].cpu(), sc)
    one = torch.rand(1, 2, generator=g)
    o = [torch.empty(30, 2, 128, dtype=dt, device="cuda") for _ in range(2)]
    q.kv_cache_read_i8(*o, c[0][:1].expand(40, 2, 128), one.cuda().expand(40, 2), c[2], one.cuda().expand(40, 2), slot.cuda())
    assert torch.equal(o[0].cpu(), (c[0][:1].cpu().float() * one[..., None]).expand(30, 2, 128).to(dt))
    assert torch.equal(o[1].cpu(), (c[2].cpu()[slot].float() * one[..., None]).to(dt))
