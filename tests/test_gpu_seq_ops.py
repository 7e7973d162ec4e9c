"""Operators over packed sequences on the device, against plain 64-bit implementations.

Tolerances.  u = 2^-24 is half a step of fp32, 2^-8 of bfloat16 (finfo.eps / 2).
  gemm_i8_w8a8    int32 sums are exact and the two products are rounded as written: equal bits.
  attention_seq   a score is a sum of `dim` products: its error is a random walk of dim roundings, each at most
                  u times a partial sum, taken as 6 sqrt(dim) u |scale| sqrt(sum (q_i k_i)^2) (six deviations), and
                  the softmax's argument adds two roundings of its size; a probability is then off by that much
                  relatively, exp2 and its argument by 8u; sums over n keys add (8 + sqrt(n)) u.  All relative to
                  sum p |v|.  bfloat16: probabilities are rounded to bfloat16 for the product with V, 2^-8 of
                  sum p |v|, and the output once more, 2^-8 of itself.
  delta_rule_seq  a token's delta and output are sums of 128 products with the state: 6 sqrt(128) u of
                  |S| |k| in norms, and a rounding of the update; k, q have norm at most 1 and beta, exp(g) are
                  at most 1, so no step enlarges an earlier error, and n steps add up to n of them at most:
                  (n + 1) (6 sqrt(128) + 8) u times the largest state (or v) norm of a column.  bfloat16: the
                  output rounded once more.
"""
import functools
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


# ------------------------------------------------------------------ int8 matrix product

# one and many tokens, rows at and off every tile's edge, the smallest and ragged depths (one 16-byte piece up
# to more than a pass of any tile), a vocabulary's height
GEMM = [(1, 512, 1024), (1, 1, 16), (2, 17, 48), (5, 1021, 3584), (15, 100, 80), (16, 256, 64), (17, 255, 144), (31, 129, 1040),
        (33, 512, 2048), (63, 64, 3584), (64, 640, 128), (65, 1000, 272), (127, 257, 1024), (129, 384, 1024), (255, 130, 4096),
        (257, 1024, 192), (300, 2049, 1024), (1024, 96, 16), (4, 20011, 1024)]


@pytest.mark.parametrize("tokens,out,inn", GEMM)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_gemm(q, torch_cuda, tokens, out, inn, bf16):
    torch = torch_cuda
    g = gen(torch, tokens + 7 * out + inn)
    w = torch.randint(-128, 128, (out, inn), generator=g, dtype=torch.int8)
    x = torch.randint(-128, 128, (tokens, inn), generator=g, dtype=torch.int8)
    w[out // 2], x[tokens // 2] = 127, -128          # the largest sums
    sw, sx = torch.rand(out, generator=g) * 1e-2, torch.rand(tokens, generator=g)
    acc = (x.double() @ w.double().t()).to(torch.float32)     # below 2^53: exact, then rounded as float(int32)
    want = (acc * sx[:, None]) * sw[None, :]
    dt = torch.bfloat16 if bf16 else torch.float32
    y = torch.full((tokens + 1, out + 3), 7.0, dtype=dt, device="cuda")   # rows wider than out, odd stride
    q.gemm_i8_w8a8(y[:tokens, :out], w.cuda(), sw.cuda(), x.cuda(), sx.cuda())
    got = y.cpu()
    assert torch.equal(got[:tokens, :out], want.to(dt))
    assert (got[tokens:] == 7).all() and (got[:, out:] == 7).all()


@pytest.mark.parametrize("tokens,out,inn", [
    (9, 16500, 16), (5, 16400, 80), (70, 4200, 48), (130, 2800, 208), (300, 2000, 272), (129, 2800, 336), (600, 1030, 400),
    (16, 16390, 528), (24, 4100, 1008), (66, 2050, 96), (257, 100, 1040)])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_gemm_forms(q, torch_cuda, tokens, out, inn, bf16):
    """Tiles whose inner dimension is shorter than the loads ahead or ends inside a step, few tokens among them; units
    of 16, 32 and 64 tokens of both types."""
    test_gemm(q, torch_cuda, tokens, out, inn, bf16)


def test_gemm_rows_far_apart(q, torch_cuda):
    """Activations' rows 16 MB apart and the last one behind 2^32 bytes."""
    torch = torch_cuda
    g, tokens, out, inn, ld = gen(torch, 5), 300, 2000, 48, 1 << 24
    w = torch.randint(-127, 128, (out, inn), generator=g, dtype=torch.int8).cuda()
    x = torch.randint(-127, 128, (tokens, inn), generator=g, dtype=torch.int8).cuda()
    sw, sx = torch.rand(out, generator=g).cuda(), torch.rand(tokens, generator=g).cuda()
    far = torch.empty((tokens - 1) * ld + inn, dtype=torch.int8, device="cuda").as_strided((tokens, inn), (ld, 1))
    far.copy_(x)
    y, want = torch.empty(tokens, out, device="cuda"), torch.empty(tokens, out, device="cuda")
    q.gemm_i8_w8a8(want, w, sw, x, sx)
    q.gemm_i8_w8a8(y, w, sw, far, sx)
    assert torch.equal(y, want)


def test_gemm_is_the_one_token_op(q, torch_cuda):
    torch = torch_cuda
    g = gen(torch, 3)
    tokens, out, inn = 6, 1000, 1024
    w = torch.randint(-127, 128, (out, inn), generator=g, dtype=torch.int8).cuda()
    sw = torch.rand(out, generator=g).cuda()
    x = torch.randn(tokens, inn, generator=g).cuda()
    wide = torch.zeros(tokens, inn + 64, dtype=torch.int8, device="cuda")     # activations in wider rows
    xq, sx, y = torch.empty(tokens, inn, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda"), torch.empty(tokens, out, device="cuda")
    q.quant_rows(xq, sx, x, tokens, inn)
    wide[:, 32:32 + inn] = xq
    q.gemm_i8_w8a8(y, w, sw, wide[:, 32:32 + inn], sx)
    one, acc = torch.empty(out, device="cuda"), torch.empty(out, dtype=torch.int32, device="cuda")
    for t in range(tokens):
        q.gemv_i8_w8a8(one, acc, w, sw, xq[t], sx[t:t + 1], out, inn)
        assert torch.equal(one, y[t])


# ------------------------------------------------------------------ gated delta rule

def delta_oracle(torch, qq, kk, vv, g, beta, S, lens):
    """float64 on the CPU; returns (out, S, the largest column norm of any state or v)."""
    qq, kk, vv, g, beta, S = (t.double() for t in (qq, kk, vv, g, beta, S))
    rep = vv.shape[1] // kk.shape[1]
    out, S, at, top = torch.zeros_like(vv), S.clone(), 0, 0.0
    for i, n in enumerate(lens):
        s = S[i]
        for t in range(at, at + n):
            k1, q1 = kk[t].repeat_interleave(rep, 0), qq[t].repeat_interleave(rep, 0)
            s = s * torch.exp(g[t])[:, None, None]
            d = (vv[t] - torch.einsum("hkv,hk->hv", s, k1)) * beta[t][:, None]
            s = s + k1[:, :, None] * d[:, None, :]
            out[t] = torch.einsum("hkv,hk->hv", s, q1)
            top = max(top, s.norm(dim=1).max().item(), vv[t].abs().max().item())
        S[i] = s
        top = max(top, s.norm(dim=1).max().item())
        at += n
    return out, S, top


def delta_inputs(torch, seed, lens, kh, h, bf16, decay=1.0, fused=True):
    g = gen(torch, seed)
    t = sum(lens)
    dt = torch.bfloat16 if bf16 else torch.float32
    unit = lambda x: x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)
    qq = (unit(torch.randn(t, kh, 128, generator=g)) / math.sqrt(128)).to(dt)
    kk, vv = unit(torch.randn(t, kh, 128, generator=g)).to(dt), torch.randn(t, h, 128, generator=g).to(dt)
    gg = -decay * torch.rand(t, h, generator=g) ** 3
    beta = torch.rand(t, h, generator=g)
    S = torch.randn(len(lens), h, 128, 128, generator=g) * 0.1
    if fused:   # one row of all heads a token, as the projection leaves it, and rows past the last sequence
        row = torch.zeros(t + 2, (2 * kh + h) * 128 + 16, dtype=dt)
        row[:t, :kh * 128], row[:t, kh * 128:2 * kh * 128] = qq.reshape(t, -1), kk.reshape(t, -1)
        row[:t, 2 * kh * 128:(2 * kh + h) * 128] = vv.reshape(t, -1)
        row = row.cuda()
        dev = [row[:, a * 128:b * 128].view(t + 2, b - a, 128) for a, b in ((0, kh), (kh, 2 * kh), (2 * kh, 2 * kh + h))]
        gb = torch.zeros(t + 2, 2 * h + 1)
        gb[:t, :h], gb[:t, h + 1:] = gg, beta
        gb = gb.cuda()
        dev += [gb[:, :h], gb[:, h + 1:]]
    else:       # head-major
        dev = [x.transpose(0, 1).contiguous().cuda().transpose(0, 1) for x in (qq, kk, vv)] + [gg.cuda(), beta.cuda()]
    return (qq, kk, vv, gg, beta, S), dev


def delta_run(q, torch, dev, S, lens, out=None, max_len=None):
    t, h = dev[2].shape[:2]
    if out is None:
        out = torch.full((t, h, 128), 7.0, dtype=dev[2].dtype, device="cuda")
    cu = torch.tensor(starts(lens), dtype=torch.int32, device="cuda")
    ml = max(lens + [0]) if max_len is None else max_len
    ws = torch.full((q.delta_rule_seq_workspace(t, len(lens), h, ml),), 0x7F, dtype=torch.uint8, device="cuda")   # NaN bits
    ws.fill_(0xFF)
    q.delta_rule_seq(out, *dev, S, cu, ws, ml)
    return out


def delta_check(torch, out, S, want, lens, bf16):
    wo, wS, top = want
    t = sum(lens)
    tol = (max(lens + [0]) + 1) * (6 * math.sqrt(128) + 8) * U * top
    assert (S.cpu().double() - wS).abs().max().item() <= tol
    err = (out[:t].cpu().double() - wo).abs()
    assert (err <= tol + (BF * (wo.abs() + tol) if bf16 else 0.0)).all(), (err.max().item(), tol)


DELTA = [  # lens, key heads, heads
    ([1], 16, 16), ([1, 1, 1], 2, 2), ([1, 0, 2, 1, 4], 2, 4), ([0, 5], 1, 1), ([15, 16, 17], 1, 2), ([31, 33, 32], 2, 2),
    ([70, 1, 0, 130, 64, 5, 66, 20], 8, 16),            # enough heads for two column tiles a workgroup
    ([3, 60, 0] * 22 + [1, 65, 2, 129], 1, 2),          # more sequences than a wave has lanes
    ([63], 1, 1), ([64], 1, 3), ([65], 1, 1), ([127, 128, 129], 1, 1), ([200, 1, 0, 70], 1, 2), ([333], 2, 2), ([700], 1, 1),
]


@pytest.mark.parametrize("lens,kh,h", DELTA, ids=str)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_delta_rule(q, torch_cuda, lens, kh, h, bf16):
    torch = torch_cuda
    host, dev = delta_inputs(torch, 11 * sum(lens) + h, lens, kh, h, bf16)
    S = host[5].cuda()
    out = delta_run(q, torch, dev, S, lens)
    delta_check(torch, out, S, delta_oracle(torch, *host, lens), lens, bf16)
    assert (out[sum(lens):] == 7).all()      # rows behind the last sequence
    for i, n in enumerate(lens):
        if n == 0:
            assert torch.equal(S[i].cpu(), host[5][i])


@pytest.mark.parametrize("decay", [0.0, 0.05, 30.0, 200.0])
def test_delta_decays(q, torch_cuda, decay):
    """No decay at all; none that matters; one that forgets within tokens, and within one."""
    torch = torch_cuda
    lens = [150, 70]
    host, dev = delta_inputs(torch, 5, lens, 1, 2, False, decay=decay, fused=False)
    S = host[5].cuda()
    out = delta_run(q, torch, dev, S, lens)
    delta_check(torch, out, S, delta_oracle(torch, *host, lens), lens, False)


def test_delta_full_resets(q, torch_cuda):
    """A log decay of minus infinity (a new document) empties the state, first, inside and last."""
    torch = torch_cuda
    lens = [140, 3]
    host, _ = delta_inputs(torch, 6, lens, 1, 1, False)
    for t in (0, 40, 41, 64, 100, 139, 141):
        host[3][t] = -math.inf
    dev = [x.cuda() for x in host[:5]]
    S = host[5].cuda()
    out = delta_run(q, torch, dev, S, lens)
    delta_check(torch, out, S, delta_oracle(torch, *host, lens), lens, False)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta", "S"])
@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=str)
def test_delta_non_finite_inputs(q, torch_cuda, bf16, which, bad):
    """A token that is not finite has no influence on those before it, on other heads or on other sequences,
    and a query's none on the state; what comes after it shows it."""
    torch = torch_cuda
    lens, at = [100, 80], 75                      # in the second chunk of the first sequence
    host, _ = delta_inputs(torch, 14, lens, 2, 2, bf16, decay=0.05)
    run = lambda h: (lambda S: (delta_run(q, torch, [x.cuda() for x in h[:5]], S, lens).cpu(), S.cpu()))(h[5].cuda())
    clean, S0 = run(host)
    i = ["q", "k", "v", "g", "beta", "S"].index(which)
    if which == "S":
        host[5][0, 0, :, 9] = bad                 # one column of one head
    elif which in ("g", "beta"):
        host[i][at, 0] = bad
    else:
        host[i][at, 0, 5] = bad
    out, S = run(host)
    first = 0 if which == "S" else at
    ok = lambda x, y: (x.double() - y.double()).abs().max().item() <= 1e-3 * y.double().abs().max().item() + (BF if bf16 else 0)
    assert torch.isfinite(out[:first]).all() and (first == 0 or ok(out[:first], clean[:first]))
    assert torch.equal(out[100:], clean[100:]) and torch.equal(S[1], S0[1])
    assert ok(out[:100, 1], clean[:100, 1]) and ok(S[0, 1], S0[0, 1])       # the other head
    if which == "q":
        assert not torch.isfinite(out[at, 0]).any() and ok(S[0, 0], S0[0, 0])
        assert torch.isfinite(out[at + 1:100, 0]).all()
    elif which == "S":
        assert not torch.isfinite(S[0, 0, :, 9]).any()
        keep = [c for c in range(128) if c != 9]
        assert ok(out[:100, 0][:, keep], clean[:100, 0][:, keep]) and ok(S[0, 0][:, keep], S0[0, 0][:, keep])
    else:
        assert not torch.isfinite(out[at:100, 0]).all() and not torch.isfinite(S[0, 0]).all()


def test_delta_prompt_then_tokens(q, torch_cuda):
    """A prompt in one call, in two, and token by token through the one-token op: the same within tolerance."""
    torch = torch_cuda
    lens = [90]
    host, dev = delta_inputs(torch, 8, lens, 16, 16, False, fused=False)
    want = delta_oracle(torch, *host, lens)
    S1, S2, S3 = (host[5].cuda() for _ in range(3))
    delta_check(torch, delta_run(q, torch, dev, S1, lens), S1, want, lens, False)
    o2 = torch.cat([delta_run(q, torch, [x[a:b] for x in dev], S2, [b - a]) for a, b in ((0, 71), (71, 72), (72, 90))])
    delta_check(torch, o2, S2, want, lens, False)
    o3, flat = torch.empty(90, 16, 128, device="cuda"), [x.contiguous() for x in dev]
    for t in range(90):
        q.delta_rule_layer(*(flat[i][t].reshape(-1) for i in range(5)), S3, o3[t])
    delta_check(torch, o3, S3, want, lens, False)


def test_delta_bound_too_small(q, torch_cuda):
    """A max_len below the lengths costs speed, not results."""
    torch = torch_cuda
    lens = [100, 3, 1]
    host, dev = delta_inputs(torch, 9, lens, 1, 1, False)
    want = delta_oracle(torch, *host, lens)
    for ml in (0, 1, 5, 100, 1000):
        S = host[5].cuda()
        delta_check(torch, delta_run(q, torch, dev, S, lens, max_len=ml), S, want, lens, False)


def test_delta_bad_bounds(q, torch_cuda):
    """Bounds out of order or outside the array: that sequence is taken as empty, the others are computed."""
    torch = torch_cuda
    lens = [20, 30]
    host, dev = delta_inputs(torch, 10, lens, 1, 1, False, fused=False)
    wo, wS, top = delta_oracle(torch, *host, lens)
    for bad in ([0, 20, 50, 10], [0, 20, 50, 51], [0, 20, 50, -3]):
        S = torch.cat([host[5], torch.full((1, 1, 128, 128), 3.0)]).cuda()
        out = torch.full((50, 1, 128), 7.0, device="cuda")
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        ws = torch.empty(q.delta_rule_seq_workspace(50, 3, 1, 50), dtype=torch.uint8, device="cuda")
        q.delta_rule_seq(out, *dev, S, cu, ws, 50)
        assert (S[2] == 3.0).all()
        delta_check(torch, out, S[:2], (wo, wS, top), lens, False)


# ------------------------------------------------------------------ attention

def attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, scale):
    """float64 on the CPU: (out, the tolerance's sums without their rounding of the output)."""
    h, kvh, d = qq.shape[1], kk.shape[1], qq.shape[2]
    out, tol, at = torch.zeros(qq.shape, dtype=torch.float64), torch.zeros(qq.shape, dtype=torch.float64), 0
    for n, m, ks in zip(lens, ctx, at_k):
        for hh in range(h):
            if n == 0 or m == 0:
                continue
            a, b, v = (x.double() for x in (qq[at:at + n, hh], kk[ks:ks + m, hh // (h // kvh)], vv[ks:ks + m, hh // (h // kvh)]))
            s = a @ b.t() * scale
            es = 6 * math.sqrt(d) * U * abs(scale) * torch.sqrt((a * a) @ (b * b).t()) + 2 * U * s.abs()
            hide = torch.arange(m)[None, :] > torch.arange(n)[:, None] + (m - n)
            s = s.masked_fill(hide, -math.inf)
            es = es.masked_fill(hide, 0.0).amax(-1, keepdim=True)
            none = hide.all(-1, keepdim=True)
            p = torch.softmax(s.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
            out[at:at + n, hh] = p @ v
            tol[at:at + n, hh] = (2 * es + (16 + math.sqrt(m)) * U) * (p @ v.abs())
        at += n
    return out, tol


def attn_inputs(torch, seed, lens, ctx, h, kvh, d, bf16, gap=0, qscale=2.0):
    g = gen(torch, seed)
    dt = torch.bfloat16 if bf16 else torch.float32
    at_k, rows = [], 0
    for m in ctx:
        rows += gap
        at_k.append(rows)
        rows += m
    rows += gap
    t = sum(lens)
    qq = (torch.randn(t, h, d, generator=g) * qscale).to(dt)
    kk, vv = torch.randn(rows, kvh, d, generator=g).to(dt), torch.randn(rows, kvh, d, generator=g).to(dt)
    return qq, kk, vv, at_k


def attn_run(q, torch, qq, kk, vv, lens, ctx, at_k, scale=None, max_q=None, max_k=None, out=None):
    t, h, d = qq.shape
    if out is None:
        out = torch.full((t, h, d), 7.0, dtype=qq.dtype, device="cuda")
    mq, mk = max(lens + [0]) if max_q is None else max_q, max(ctx + [0]) if max_k is None else max_k
    ws = torch.full((q.attention_seq_workspace(t, len(lens), mq, mk, h, kk.shape[1], d),), 0xFF, dtype=torch.uint8, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q.attention_seq(out, qq, kk, vv, i32(starts(lens)), torch.tensor(at_k, dtype=torch.int64, device="cuda"), i32(ctx), ws, mq, mk,
                    scale)
    return out


def attn_check(torch, got, want, bf16):
    wo, tol = want
    got = got.cpu().double()[:wo.shape[0]]
    err = (got - wo).abs()
    if bf16:
        # sum p |v| is at most tol / (16 u): the probabilities' rounding, then the output's
        lim = tol + BF * (tol / (16 * U)).clamp(max=8.0) + BF * (wo.abs() + tol)
    else:
        lim = tol + U * wo.abs()
    assert (err <= lim).all(), (err.max().item(), (err / lim.clamp(min=1e-30)).max().item())


ATTN = [  # lens, keys, heads, kv heads, dim
    ([1], [1], 1, 1, 128), ([1], [1], 8, 2, 256), ([1, 1, 1], [7, 300, 1], 8, 2, 256), ([1, 1], [2500, 15], 4, 4, 128),
    ([1], [5000], 8, 2, 256), ([2, 3], [33, 64], 6, 2, 128), ([4], [1000], 16, 1, 128), ([1], [777], 32, 1, 256),
    ([15, 16, 17], [15, 16, 17], 2, 1, 128), ([64], [64], 2, 2, 256), ([63, 0, 65], [63, 5, 70], 4, 2, 128), ([127, 1], [127, 129], 8, 2, 256),
    ([129], [400], 2, 1, 256), ([200, 90], [200, 90], 3, 3, 128), ([300], [300], 8, 2, 256), ([33], [2000], 2, 1, 128), ([260], [261], 1, 1, 256),
    ([520], [520], 4, 1, 128), ([5], [5], 3, 1, 256),
]


@pytest.mark.parametrize("lens,ctx,h,kvh,d", ATTN, ids=str)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention(q, torch_cuda, lens, ctx, h, kvh, d, bf16):
    torch = torch_cuda
    qq, kk, vv, at_k = attn_inputs(torch, sum(lens) + sum(ctx) + h, lens, ctx, h, kvh, d, bf16, gap=3)
    scale = 1 / math.sqrt(d)
    out = torch.full((qq.shape[0] + 2, h, d), 7.0, dtype=qq.dtype, device="cuda")
    pad = torch.cat([qq, qq[:1], qq[:1]]) if qq.shape[0] else qq    # two rows behind the last sequence
    got = attn_run(q, torch, pad.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k, out=out)
    attn_check(torch, got, attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, scale), bf16)
    assert (got[qq.shape[0]:] == 7).all()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_rows_without_keys(q, torch_cuda, bf16, d):
    """More rows than keys: the first rows see none and come out as 0; no key at all."""
    torch = torch_cuda
    for lens, ctx in (([70, 3], [9, 0]), ([200], [1]), ([5, 1], [2, 0])):
        qq, kk, vv, at_k = attn_inputs(torch, 1, lens, ctx, 4, 2, d, bf16, gap=1)
        got = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k)
        attn_check(torch, got, attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(d)), bf16)
        assert (got[:lens[0] - ctx[0]] == 0).all()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,m", [(1, 200), (5, 300), (100, 100), (150, 260)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_attention_hidden_keys_have_no_influence(q, torch_cuda, bf16, n, m, bad):
    """What stands behind a row's keys (the next tokens, rows of the cache not yet written, another sequence)
    may be anything; what a row does see reaches it."""
    torch = torch_cuda
    lens, ctx = [n, 2], [m, 2]
    qq, kk, vv, at_k = attn_inputs(torch, 2, lens, ctx, 4, 2, 128, bf16, gap=40)
    clean = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k)
    for t in (kk, vv):
        t[:at_k[0]] = bad
        t[at_k[0] + m:at_k[1]] = bad
        t[at_k[1] + 2:] = bad
    hit = at_k[0] + m - max(n // 3, 1)      # a key that the first rows do not see, and the last ones do
    if n > 1:
        kk[hit, 0, 5], vv[hit, :, 7] = bad, bad
    got = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k)
    free = n if n == 1 else n - max(n // 3, 1)
    assert torch.equal(got[:free], clean[:free]) and torch.equal(got[n:], clean[n:])
    if n > 1:
        assert not torch.isfinite(got[free:n, :, 7]).any()
        if math.isnan(bad):
            assert torch.isnan(got[free:n, :2]).all()     # heads of the key that scores NaN


def test_attention_infinite_value_reaches_its_element_only(q, torch_cuda):
    torch = torch_cuda
    for bf16 in (False, True):
        for n, m in ((1, 50), (40, 40), (130, 300)):
            qq, kk, vv, at_k = attn_inputs(torch, 4, [n], [m], 2, 1, 128, bf16, qscale=0.2)
            clean = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), [n], [m], at_k)
            vv[m - 1, 0, 3] = math.inf       # the last key: seen by the last row alone
            got = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), [n], [m], at_k)
            assert (got[n - 1, :, 3] == math.inf).all()
            got[n - 1, :, 3] = clean[n - 1, :, 3]
            assert torch.equal(got, clean)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention_strides(q, torch_cuda, bf16):
    """Queries inside a query and gate projection, caches of slots, an output inside wider rows, head-major
    inputs, one row of queries for all (stride 0)."""
    torch = torch_cuda
    lens, ctx, h, kvh, d = [40, 1, 70], [40, 90, 71], 4, 2, 128
    qq, kk, vv, _ = attn_inputs(torch, 5, lens, ctx, h, kvh, d, bf16)
    slots, kp = 120, torch.zeros(3 * 120, kvh, d, dtype=qq.dtype)
    vp, at_k, src = torch.zeros_like(kp), [slots * 2, 0, slots], starts(ctx)
    for i, m in enumerate(ctx):
        kp[at_k[i]:at_k[i] + m], vp[at_k[i]:at_k[i] + m] = kk[src[i]:src[i] + m], vv[src[i]:src[i] + m]
    want = attn_oracle(torch, qq, kp, vp, lens, ctx, at_k, 1 / math.sqrt(d))
    t = sum(lens)
    gate = torch.full((t, h, 2 * d), 9.0, dtype=qq.dtype, device="cuda")
    gate[:, :, :d] = qq.cuda()
    wide = torch.full((t, h * d + 64), 7.0, dtype=qq.dtype, device="cuda")
    out = wide[:, 32:32 + h * d].view(t, h, d)
    attn_run(q, torch, gate[:, :, :d], kp.cuda(), vp.cuda(), lens, ctx, at_k, out=out)
    attn_check(torch, out, want, bf16)
    assert (wide[:, :32] == 7).all() and (wide[:, 32 + h * d:] == 7).all()
    hm = lambda x: x.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    o2 = torch.empty(h, t, d, dtype=qq.dtype, device="cuda").transpose(0, 1)
    attn_run(q, torch, hm(qq), hm(kp), hm(vp), lens, ctx, at_k, out=o2)
    assert torch.equal(o2, out)
    same = qq[:1].cuda().expand(t, h, d)
    want = attn_oracle(torch, qq[:1].expand(t, h, d), kp, vp, lens, ctx, at_k, 1 / math.sqrt(d))
    attn_check(torch, attn_run(q, torch, same, kp.cuda(), vp.cuda(), lens, ctx, at_k), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention_bounds_too_small_or_large(q, torch_cuda, bf16):
    """max_q and max_k choose the form: any value gives the same within tolerance."""
    torch = torch_cuda
    lens, ctx = [1, 90, 3], [900, 90, 500]
    qq, kk, vv, at_k = attn_inputs(torch, 6, lens, ctx, 4, 2, 128, bf16)
    want = attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(128))
    for mq in (0, 1, 4, 90, 5000):
        for mk in (0, 100, 900, 100000):
            attn_check(torch, attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k, max_q=mq, max_k=mk), want, bf16)


def test_attention_large_scores(q, torch_cuda):
    """Scores far apart (one key takes all), equal scores, and a scale of 0 (the mean of the keys)."""
    torch = torch_cuda
    for scale in (40.0, 0.0, -0.3):
        qq, kk, vv, at_k = attn_inputs(torch, 7, [20, 1], [30, 400], 2, 1, 128, False)
        got = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), [20, 1], [30, 400], at_k, scale=scale)
        attn_check(torch, got, attn_oracle(torch, qq, kk, vv, [20, 1], [30, 400], at_k, scale), False)


def test_attention_bad_ranges(q, torch_cuda):
    """Key ranges outside the array give NaN in that sequence's rows; row bounds out of order leave rows alone."""
    torch = torch_cuda
    for n, m in ((1, 40), (30, 40)):
        lens, ctx = [n, n, n], [m, m, m]
        qq, kk, vv, at_k = attn_inputs(torch, 8, lens, ctx, 2, 1, 128, False)
        clean = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k)
        for start, length in ((-1, m), (2 * m + 1, m), (m, -1), (1 << 40, m), (0, 3 * m + 1)):
            k2, c2 = list(at_k), list(ctx)
            k2[1], c2[1] = start, length
            got = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, c2, k2, max_k=m)
            assert torch.isnan(got[n:2 * n]).all()
            assert torch.equal(got[:n], clean[:n]) and torch.equal(got[2 * n:], clean[2 * n:])
        out = torch.full((3 * n, 2, 128), 7.0, device="cuda")
        ws = torch.empty(q.attention_seq_workspace(3 * n, 3, n, m, 2, 1, 128), dtype=torch.uint8, device="cuda")
        cu = torch.tensor([0, n, 3 * n + 1, 3 * n], dtype=torch.int32, device="cuda")
        q.attention_seq(out, qq.cuda(), kk.cuda(), vv.cuda(), cu, torch.tensor(at_k, dtype=torch.int64, device="cuda"),
                        torch.tensor(ctx, dtype=torch.int32, device="cuda"), ws, n, m)
        assert torch.equal(out[:n], clean[:n]) and (out[n:] == 7).all()


def test_attention_prompt_then_tokens(q, torch_cuda):
    """Rows one call at a time over the growing cache see what they see in one call."""
    torch = torch_cuda
    n = 70
    qq, kk, vv, at_k = attn_inputs(torch, 9, [n], [n], 8, 2, 256, False)
    want = attn_oracle(torch, qq, kk, vv, [n], [n], at_k, 1 / 16.0)
    dev = [x.cuda() for x in (qq, kk, vv)]
    attn_check(torch, attn_run(q, torch, *dev, [n], [n], at_k), want, False)
    one = torch.cat([attn_run(q, torch, dev[0][t:t + 1], dev[1], dev[2], [1], [t + 1], [0]) for t in range(n)])
    attn_check(torch, one, want, False)


# The form for prompts, whatever the lengths: max_q is a bound, and a large one asks for it.

@pytest.fixture
def prompts(monkeypatch):
    monkeypatch.setattr(sys.modules[__name__], "attn_run", functools.partial(attn_run, max_q=4096))


@pytest.mark.parametrize("lens,ctx,h,kvh,d", ATTN + [
    ([700], [3000], 8, 2, 256), ([130, 1], [4100, 2000], 2, 2, 128), ([40], [9000], 4, 4, 128), ([1023, 0, 513], [1023, 4, 800], 4, 1, 256),
    ([257], [700], 12, 4, 256)], ids=str)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_form(prompts, q, torch_cuda, lens, ctx, h, kvh, d, bf16):
    test_attention(q, torch_cuda, lens, ctx, h, kvh, d, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_prompt_form_rows_without_keys(prompts, q, torch_cuda, bf16, d):
    test_attention_rows_without_keys(q, torch_cuda, bf16, d)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,m", [(1, 200), (5, 300), (100, 100), (150, 260), (90, 1200)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_prompt_form_hidden_keys_have_no_influence(prompts, q, torch_cuda, bf16, n, m, bad):
    test_attention_hidden_keys_have_no_influence(q, torch_cuda, bf16, n, m, bad)


def test_prompt_form_infinite_value(prompts, q, torch_cuda):
    test_attention_infinite_value_reaches_its_element_only(q, torch_cuda)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_form_strides(prompts, q, torch_cuda, bf16):
    test_attention_strides(q, torch_cuda, bf16)


def test_prompt_form_large_scores(prompts, q, torch_cuda):
    test_attention_large_scores(q, torch_cuda)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_form_bad_ranges(prompts, q, torch_cuda, bf16):
    """As test_attention_bad_ranges, with sequences whose keys are split beside those that have none."""
    torch = torch_cuda
    lens, ctx = [30, 150, 7], [600, 700, 40]
    qq, kk, vv, at_k = attn_inputs(torch, 8, lens, ctx, 2, 1, 128, bf16)
    dev = [x.cuda() for x in (qq, kk, vv)]
    want, tol = attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(128))
    for start, length in ((-1, 700), (641, 700), (600, -1), (1 << 40, 700), (0, 1341)):
        got = attn_run(q, torch, *dev, lens, [600, length, 40], [at_k[0], start, at_k[2]], max_k=700)
        assert torch.isnan(got[30:180]).all()
        for a, b in ((0, 30), (180, 187)):
            attn_check(torch, got[a:b], (want[a:b], tol[a:b]), bf16)
    out = torch.full(qq.shape, 7.0, dtype=qq.dtype, device="cuda")
    ws = torch.empty(q.attention_seq_workspace(187, 3, 4096, 700, 2, 1, 128), dtype=torch.uint8, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q.attention_seq(out, *dev, i32([0, 30, 188, 187]), torch.tensor(at_k, dtype=torch.int64, device="cuda"), i32(ctx), ws, 4096, 700)
    attn_check(torch, out[:30], (want[:30], tol[:30]), bf16)
    assert (out[30:] == 7).all()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_k", [129, 300, 700, 20000])
def test_prompt_form_places_in_the_workspace(q, torch_cuda, bf16, max_k):
    """max_k is a bound on what the workspace holds, not on the keys: what finds no place there is not split.  Long keys
    and short ones in turn, and the longest sequence last."""
    torch = torch_cuda
    lens, ctx = [70, 3, 0, 129, 64, 1, 70, 2, 300], [900, 3, 10, 1500, 64, 2500, 400, 2, 3000]
    qq, kk, vv, at_k = attn_inputs(torch, 15, lens, ctx, 4, 2, 128, bf16)
    want = attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(128))
    attn_check(torch, attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k, max_q=4096, max_k=max_k), want, bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, 4096])
def test_attention_of_many_sequences(q, torch_cuda, bf16, max_q):
    """More than the 64 sequences that a wave looks at together; long ones among empty and short ones."""
    torch = torch_cuda
    lens = [(5 * i) % 9 for i in range(150)]
    ctx = [n + (7 * i) % 40 for i, n in enumerate(lens)]
    for i, n, m in ((3, 140, 900), (64, 1, 1500), (149, 70, 70)):
        lens[i], ctx[i] = n, m
    qq, kk, vv, at_k = attn_inputs(torch, 10, lens, ctx, 4, 2, 128, bf16)
    got = attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k, max_q=max_q)
    attn_check(torch, got, attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(128)), bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_prompt_forms_captured(q, torch_cuda, bf16):
    """Chunks of the delta rule and split tiles of attention in one graph, replayed with other bounds, key ranges and
    inputs on the device and eager calls between; every replay against the eager result."""
    torch = torch_cuda
    rows, h, kvh, d, dt = 700, 8, 2, 128, torch.bfloat16 if bf16 else torch.float32
    g = gen(torch, 12)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    qq, kk, vv, out = rnd(rows, h, d), rnd(2000, kvh, d), rnd(2000, kvh, d), torch.empty(rows, h, d, dtype=dt, device="cuda")
    dk, dv, dout = torch.nn.functional.normalize(rnd(rows, 4, 128).float(), dim=-1).to(dt), rnd(rows, h, 128), rnd(rows, h, 128)
    lg, be = -torch.rand(rows, h, generator=g).cuda(), torch.rand(rows, h, generator=g).cuda()
    S0 = torch.randn(3, h, 128, 128, generator=g).cuda()
    S = S0.clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cu, ks, kl = i32([0, 500, 500, 700]), torch.tensor([0, 0, 900], dtype=torch.int64, device="cuda"), i32([1500, 0, 300])
    aw = torch.empty(q.attention_seq_workspace(rows, 3, rows, 2000, h, kvh, d), dtype=torch.uint8, device="cuda")
    dw = torch.empty(q.delta_rule_seq_workspace(rows, 3, h, rows, k_heads=4, dtype=q.BF16 if bf16 else q.F32), dtype=torch.uint8, device="cuda")

    def step():
        q.attention_seq(out, qq, kk, vv, cu, ks, kl, aw, 4096, 2000)
        q.delta_rule_seq(dout, dk, dk, dv, lg, be, S, cu, dw, rows)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for bounds, at, n in (([0, 500, 500, 700], [0, 0, 900], [1500, 0, 300]), ([0, 3, 690, 700], [100, 0, 1990], [1800, 687, 10]),
                          ([0, 0, 1, 1], [0, 5, 0], [0, 2000, 0])):
        cu.copy_(i32(bounds))
        ks.copy_(torch.tensor(at, device="cuda"))
        kl.copy_(i32(n))
        qq.copy_(rnd(rows, h, d))
        want = []
        for run in (step, graph.replay, graph.replay):
            S.copy_(S0)
            out.fill_(7.0), dout.fill_(7.0)
            run()
            torch.cuda.synchronize()
            want.append([x.clone() for x in (out, dout, S)])
        for got in want[1:]:     # (the last sequence's keys end behind the array: NaN, in every run)
            assert all(((x == y) | (x.isnan() & y.isnan())).all() for x, y in zip(got, want[0]))
        assert torch.isnan(want[0][0]).any() == (n[1] == 2000) and torch.isfinite(want[0][1]).all()
        assert (want[0][0][bounds[-1]:] == 7).all() and (want[0][1][bounds[-1]:] == 7).all()


def apart(torch, x, ld):
    """x's rows `ld` elements apart, the last ones behind 2^32 bytes."""
    far = torch.empty((x.shape[0] - 1) * ld + x[0].numel(), dtype=x.dtype, device="cuda")
    far = far.as_strided(x.shape, (ld, x.stride(1), 1))
    far.copy_(x)
    return far


@pytest.mark.parametrize("ld", [1 << 21, 1 << 24])     # (from 2^24 on: the form for few rows)
@pytest.mark.parametrize("max_q", [1, 4096])
def test_attention_rows_far_apart(q, torch_cuda, ld, max_q):
    torch = torch_cuda
    rows = 1100 if ld == 1 << 21 else 300
    lens, ctx = [40, 1, 200], [rows, 250, rows - 60]
    qq, kk, vv, _ = attn_inputs(torch, 13, lens, [rows], 4, 2, 128, True)
    at_k = [0, rows - 250, 60]
    want = attn_oracle(torch, qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(128))
    far = [apart(torch, x.cuda(), ld) for x in (kk, vv)]
    attn_check(torch, attn_run(q, torch, qq.cuda(), *far, lens, ctx, at_k, max_q=max_q), want, True)


@pytest.mark.parametrize("max_len", [1, 1100])
def test_delta_rows_far_apart(q, torch_cuda, max_len):
    torch = torch_cuda
    g, t, h, ld = gen(torch, 14), 1100, 2, 1 << 20
    n = lambda *s: torch.randn(*s, generator=g).cuda()
    qq, kk, vv = (torch.nn.functional.normalize(n(t, h, 128), dim=-1) for _ in range(3))
    lg, be, cu = -torch.rand(t, h, generator=g).cuda(), torch.rand(t, h, generator=g).cuda(), torch.tensor([0, 70, 1100], dtype=torch.int32, device="cuda")
    ws = torch.empty(q.delta_rule_seq_workspace(t, 2, h, max_len), dtype=torch.uint8, device="cuda")
    res = []
    for f in (lambda x: x, lambda x: apart(torch, x, ld)):
        S, out = torch.ones(2, h, 128, 128, device="cuda"), f(torch.empty_like(vv))
        q.delta_rule_seq(out, f(qq), f(kk), f(vv), lg, be, S, cu, ws, max_len)
        res.append((out.contiguous(), S))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


# ------------------------------------------------------------------ calls that cannot be answered

def test_refused_tensors(q, torch_cuda):
    torch = torch_cuda
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")
    w, s, x, sx, y = z(32, 64, dt=torch.int8), z(32), z(4, 64, dt=torch.int8), z(4), z(4, 32)
    with pytest.raises(TypeError):
        q.gemm_i8_w8a8(y.half(), w, s, x, sx)
    with pytest.raises(ValueError):
        q.gemm_i8_w8a8(y, w, s, x, z(5))
    with pytest.raises(ValueError):
        q.gemm_i8_w8a8(y, w, s, z(4, 128, dt=torch.int8)[:, ::2], sx)
    with pytest.raises(ValueError):
        q.gemm_i8_w8a8(y, z(64, 32, dt=torch.int8).t(), s, x, sx)
    with pytest.raises(q.QHError):
        q.gemm_i8_w8a8(y, w, s, z(4, 80, dt=torch.int8)[:, 8:72], sx)       # 8 bytes off
    with pytest.raises(q.QHError):
        q.gemm_i8_w8a8(y[:1].expand(4, 32), w, s, x, sx)                    # one output row for all tokens
    a, cu, S = z(4, 2, 128), z(2, dt=torch.int32), z(1, 2, 128, 128)
    with pytest.raises(ValueError):
        q.delta_rule_seq(z(4, 2, 128), a, a, a, z(4, 2), z(4, 2), S, z(3, dt=torch.int32), None, 4)
    with pytest.raises(TypeError):
        q.delta_rule_seq(z(4, 2, 128), a, a, a, z(4, 2), z(4, 2), S, z(2, dt=torch.int64), None, 4)
    with pytest.raises(TypeError):
        q.delta_rule_seq(z(4, 2, 128), a, a.bfloat16(), a, z(4, 2), z(4, 2), S, cu, None, 4)
    with pytest.raises(q.QHError):
        q.delta_rule_seq(a, a, a, a, z(4, 2), z(4, 2), S, cu, None, 4)      # in place
    with pytest.raises(q.QHError):
        q.delta_rule_seq(z(4, 3, 128), z(4, 2, 128), z(4, 2, 128), z(4, 3, 128), z(4, 3), z(4, 3), z(1, 3, 128, 128), cu, None, 4)
    ks, kl = z(1, dt=torch.int64), z(1, dt=torch.int32)
    with pytest.raises(ValueError):
        q.attention_seq(z(4, 2, 128), a, z(9, 1, 128), z(8, 1, 128), cu, ks, kl, None, 4, 9)
    with pytest.raises(q.QHError):
        q.attention_seq(z(4, 2, 64), z(4, 2, 64), z(9, 1, 64), z(9, 1, 64), cu, ks, kl, None, 4, 9)
    with pytest.raises(q.QHError):
        q.attention_seq(a, a, z(9, 1, 128), z(9, 1, 128), cu, ks, kl, None, 4, 9)


def test_tensors_elsewhere(q, torch_cuda, monkeypatch):
    """Operands in host memory or on another device than the current one are refused, each of them; module parameters
    are tensors like others; a workspace that is too small is refused."""
    torch = torch_cuda
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")
    i8 = torch.int8
    ops = [z(4, 32), z(32, 64, dt=i8), z(32), z(4, 64, dt=i8), z(4)]
    for i in range(5):
        with pytest.raises(TypeError):
            q.gemm_i8_w8a8(*[x.cpu() if k == i else x for k, x in enumerate(ops)])
    q.gemm_i8_w8a8(*[torch.nn.Parameter(x, requires_grad=False) for x in ops])
    a, kv, cu, ks, kl = z(4, 2, 128), z(9, 1, 128), z(2, dt=torch.int32), z(1, dt=torch.int64), z(1, dt=torch.int32)
    d, S, g = z(4, 2, 128), z(1, 2, 128, 128), z(4, 2)
    attn = [z(4, 2, 128), a, kv, z(9, 1, 128), cu, ks, kl]
    delta = [d, a, z(4, 2, 128), z(4, 2, 128), g, z(4, 2), S, cu]
    for i in range(len(attn)):
        with pytest.raises(TypeError):
            q.attention_seq(*[x.cpu() if k == i else x for k, x in enumerate(attn)], None, 4, 9)
    for i in range(len(delta)):
        with pytest.raises(TypeError):
            q.delta_rule_seq(*[x.cpu() if k == i else x for k, x in enumerate(delta)], None, 4)
    with pytest.raises(TypeError):
        q.attention_seq(*attn, torch.empty(64, dtype=torch.uint8), 4, 9)
    with pytest.raises(q.QHError):
        q.attention_seq(*attn, torch.empty(256, dtype=torch.uint8, device="cuda"), 4, 1000)
    with pytest.raises(q.QHError):
        q.delta_rule_seq(*delta, torch.empty(256, dtype=torch.uint8, device="cuda"), 1000)
    monkeypatch.setattr(q._Short, "device", lambda: 1)
    for call in (lambda: q.gemm_i8_w8a8(*ops), lambda: q.attention_seq(*attn, None, 4, 9), lambda: q.delta_rule_seq(*delta, None, 4)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ streams, graphs, together

def test_other_stream(q, torch_cuda):
    torch = torch_cuda
    lens, ctx = [80, 5], [80, 300]
    qq, kk, vv, at_k = attn_inputs(torch, 12, lens, ctx, 8, 2, 256, True)
    dev = [x.cuda() for x in (qq, kk, vv)]
    host, dd = delta_inputs(torch, 12, lens, 2, 2, False)
    want, S = attn_run(q, torch, *dev, lens, ctx, at_k), host[5].cuda()
    wo = delta_run(q, torch, dd, S, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        S2 = host[5].cuda()
        got, o2 = attn_run(q, torch, *dev, lens, ctx, at_k), delta_run(q, torch, dd, S2, lens)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(o2, wo) and torch.equal(S, S2)


def test_block_of_operators_captured(q, torch_cuda):
    """The operators as a layer would chain them over packed prompts: activations quantised, one projection to
    q, k, v and the gates, attention over the cache that the keys were written to, the delta rule on the same
    projection, and an output projection of both; captured once, replayed between eager work, each replay
    equal to the eager result on that replay's inputs; and each stage against 64 bits on its own inputs."""
    torch = torch_cuda
    lens, past = [70, 1, 0, 33], [0, 50, 0, 7]
    t, hid, h, kvh, d = sum(lens), 512, 4, 2, 128
    ctx = [a + b for a, b in zip(lens, past)]
    cols = [h * d, kvh * d, kvh * d, h]                    # attention's q, k, v; the delta rule's beta logits
    n_out, slot = sum(cols) + (16 - h), 128
    g = gen(torch, 13)
    W = torch.randint(-127, 128, (n_out, hid), generator=g, dtype=torch.int8).cuda()
    ws = (torch.rand(n_out, generator=g) / (73 * math.sqrt(hid)) + 1e-4).cuda()
    Wo = torch.randint(-127, 128, (hid, 2 * h * d), generator=g, dtype=torch.int8).cuda()
    wos = (torch.rand(hid, generator=g) / (73 * math.sqrt(2 * h * d))).cuda()
    seq = torch.tensor(sum([[i] * n for i, n in enumerate(lens)], []))
    rows = torch.cat([torch.arange(p, p + n) for p, n in zip(past, lens)]) + slot * seq
    rows = rows.cuda()
    cu = torch.tensor(starts(lens), dtype=torch.int32, device="cuda")
    ks = (torch.arange(len(lens)) * slot).to(torch.int64).cuda()
    kl = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    x = torch.randn(t, hid, generator=g).cuda()
    K0, V0 = torch.randn(len(lens) * slot, kvh, d, generator=g).cuda(), torch.randn(len(lens) * slot, kvh, d, generator=g).cuda()
    S0 = (torch.randn(len(lens), h, 128, 128, generator=g) * 0.1).cuda()
    K, V, S = K0.clone(), V0.clone(), S0.clone()
    xq, sx = torch.empty(t, hid, dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda")
    y, both = torch.empty(t, n_out, device="cuda"), torch.empty(t, 2 * h, d, device="cuda")
    bq, bs, z = torch.empty(t, 2 * h * d, dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda"), torch.empty(t, hid, device="cuda")
    decay, beta = torch.full((t, h), -0.1, device="cuda"), torch.empty(t, h, device="cuda")
    qn, kn = torch.empty(t, h, d, device="cuda"), torch.empty(t, kvh, d, device="cuda")
    w1 = torch.empty(q.attention_seq_workspace(t, len(lens), max(lens), max(ctx), h, kvh, d), dtype=torch.uint8, device="cuda")
    w2 = torch.empty(q.delta_rule_seq_workspace(t, len(lens), h, max(lens)), dtype=torch.uint8, device="cuda")

    def step():
        q.quant_rows(xq, sx, x, t, hid)
        q.gemm_i8_w8a8(y, W, ws, xq, sx)
        qh, kh, vh = (y[:, a:a + n].view(t, -1, d) for a, n in ((0, h * d), (h * d, kvh * d), (h * d + kvh * d, kvh * d)))
        K[rows], V[rows] = kh, vh
        q.attention_seq(both[:, :h], qh, K, V, cu, ks, kl, w1, max(lens), max(ctx))
        qn.copy_(qh / (qh.square().sum(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(d))
        kn.copy_(kh / (kh.square().sum(-1, keepdim=True) + 1e-6).sqrt())
        beta.copy_(torch.sigmoid(y[:, sum(cols[:3]):sum(cols)]))
        q.delta_rule_seq(both[:, h:], qn[:, ::h // kvh], kn, qh, decay, beta, S, cu, w2, max(lens))
        q.quant_rows(bq, bs, both.view(t, -1), t, 2 * h * d)
        q.gemm_i8_w8a8(z, Wo, wos, bq, bs)

    def reset(scale):
        x.copy_(x0 * scale)
        K.copy_(K0), V.copy_(V0), S.copy_(S0)

    def eager(scale):
        reset(scale)
        step()
        return [v.clone() for v in (z, both, K, V, S)]

    x0 = x.clone()
    want = {s: eager(s) for s in (1.0, 0.5, -2.0)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for s in (1.0, 0.5, -2.0, 1.0, 0.5):
        reset(s)
        graph.replay()
        torch.cuda.synchronize()
        for got, exp in zip((z, both, K, V, S), want[s]):
            assert torch.equal(got, exp)
        again = eager(s)                          # the program's own work between the replays
        assert torch.equal(again[0], want[s][0])
    # the last eager step's stages
    c = lambda v: v.cpu()
    qh, vh = c(y[:, :h * d]).view(t, h, d), None
    attn_check(torch, both[:, :h], attn_oracle(torch, qh, c(K), c(V), lens, ctx, ks.tolist(), 1 / math.sqrt(d)), False)
    host = (c(qn[:, ::h // kvh]), c(kn), qh, c(decay), c(beta), c(S0))
    delta_check(torch, both[:, h:], S, delta_oracle(torch, *host, lens), lens, False)
    acc = (c(bq).double() @ c(Wo).double().t()).float()
    assert torch.equal(c(z), (acc * c(bs)[:, None]) * c(wos)[None, :])
