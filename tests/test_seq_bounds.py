"""Operators over packed sequences: bounds tight enough to see a lost part of a product, a lost step or a form that no
other test reaches.  On the CPU each bound is shown to fail for a planted mistake in the oracle's place; on the device
the kernels are held to it.

Attention, bfloat16.  A product with P adds to the fp32 bound (tests/test_gpu_seq_ops.py) what P's rounding takes: the form for
few rows multiplies V with P in two bfloat16 parts, the first cut (p - hi < 2^-7 p) and the second rounded (2^-8 of itself) and moved
up by 2^-18 p, 2^-14 sum p |v| in all; the form for prompts rounds each probability once, 2^-8 sum p |v|.  Both round the output
once, 2^-8 of it.

Delta rule.  Every rounding is taken as independent, half a step u = 2^-24 of the value at most, and carried through the
recursion in 64 bits as a covariance over the state's rows (summed over its columns): a token's sums of 128 products
are off by sqrt(128) u of the root of the products' squares, its delta and the state by u of themselves, the decay by
u (1 + |g|); later tokens pass an error on as they pass the state on, e^g (I - beta k k^T).  An output is off by what its query reads
of that, and by its own sum.  The norms over a head's columns may be three times that deviation (they scatter by
a few per cent).  In chunks the kernel sums in another order, of the same length; what its parts of bfloat16 leave out of a
product, 2^-21, is 0.7 u sqrt(128) of a sum in the same sense.
"""
import functools
import math
import os
import subprocess

import pytest

import test_gpu_seq_ops as ops
import test_seq_ops as seq_ops
from conftest import ROOT

U, BF = ops.U, ops.BF
FEW, PROMPTS = 2.0 ** -14, BF      # what P's rounding takes, of sum p |v|


def attn_limit(torch, args, bf16, p_rounding):
    """(64-bit result, how far a kernel's result may be from it)."""
    qq, kk, vv, lens, ctx, at_k, scale = args
    want, tol = ops.attn_oracle(torch, *args)
    if not bf16:
        return want, tol + U * want.abs()
    pv = ops.attn_oracle(torch, qq, kk, vv.abs(), lens, ctx, at_k, scale)[0]
    tol = tol + p_rounding * pv
    return want, tol + BF * (want.abs() + tol)


def within(got, limit):
    want, lim = limit
    err = (got.double().cpu()[:want.shape[0]] - want).abs()
    return bool((err <= lim).all())


# ------------------------------------------------------------------ attention

def plain_attention(torch, args, p_of):
    """The 64-bit result with P replaced by p_of(P), the maximum's probability being 1 as in the kernels."""
    qq, kk, vv, lens, ctx, at_k, scale = args
    h, kvh = qq.shape[1], kk.shape[1]
    out, at = torch.zeros(qq.shape, dtype=torch.float64), 0
    for n, m, ks in zip(lens, ctx, at_k):
        for hh in range(h if n and m else 0):
            a, b, v = (x.double() for x in (qq[at:at + n, hh], kk[ks:ks + m, hh // (h // kvh)], vv[ks:ks + m, hh // (h // kvh)]))
            s = a @ b.t() * scale
            s = s.masked_fill(torch.arange(m)[None, :] > torch.arange(n)[:, None] + (m - n), -math.inf)
            none = (s == -math.inf).all(-1, keepdim=True)
            p = torch.exp(s - s.amax(-1, keepdim=True).masked_fill(none, 0.0))
            out[at:at + n, hh] = (p_of(p) @ v / p.sum(-1, keepdim=True)).masked_fill(none, 0.0)
        at += n
    return out.to(torch.bfloat16)


def once(p):
    return p.bfloat16().double()


def two_parts(p):
    import torch
    hi = (p.float().view(torch.int32) & -65536).view(torch.float32).double()
    return hi + (p - hi + p * 2.0 ** -18).bfloat16().double()


@pytest.mark.parametrize("lens,ctx", [([1, 1, 1], [7, 300, 33]), ([1], [5000]), ([16], [200])], ids=str)
def test_bounds_see_how_probabilities_are_rounded(lens, ctx):
    import torch
    qq, kk, vv, at_k = ops.attn_inputs(torch, sum(ctx), lens, ctx, 2, 1, 128, True)
    args = (qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(128))
    few, prompts = (attn_limit(torch, args, True, r) for r in (FEW, PROMPTS))
    assert within(plain_attention(torch, args, two_parts), few)
    assert within(plain_attention(torch, args, once), prompts)
    assert not within(plain_attention(torch, args, once), few)


@pytest.mark.parametrize("m,lost,p_rounding", [(5000, 32, PROMPTS), (2500, 16, PROMPTS), (5000, 32, FEW), (2500, 16, FEW)])
def test_bounds_see_a_lost_step(m, lost, p_rounding):
    """One step of one wave of the smallest work, among thousands of keys."""
    import torch
    qq, kk, vv, at_k = ops.attn_inputs(torch, m, [1], [m], 8, 2, 256, True)
    args = (qq, kk, vv, [1], [m], at_k, 1 / 16.0)
    limit = attn_limit(torch, args, True, p_rounding)

    def without(p):
        p = p.clone()
        p[:, 640:640 + lost] = 0
        return p

    assert within(plain_attention(torch, args, once if p_rounding == PROMPTS else two_parts), limit)
    assert not within(plain_attention(torch, args, without), limit)


FORMS = [  # lens, keys, heads, kv heads, dim: P's rounding shows where few keys cancel, a lost step where there are many
    ([1, 1, 1], [7, 300, 33], 8, 2, 256), ([1], [5000], 8, 2, 256), ([16, 3], [200, 90], 4, 1, 128), ([1, 1], [2500, 15], 4, 4, 128),
    ([260, 1], [261, 900], 2, 1, 256), ([130], [700], 6, 2, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,ctx,h,kvh,d", FORMS, ids=str)
@pytest.mark.parametrize("max_q,p_rounding", [(1, FEW), (4096, PROMPTS)], ids=["few", "prompts"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_attention_rounding(q, torch_cuda, lens, ctx, h, kvh, d, max_q, p_rounding, bf16):
    torch = torch_cuda
    qq, kk, vv, at_k = ops.attn_inputs(torch, sum(lens) + sum(ctx), lens, ctx, h, kvh, d, bf16)
    got = ops.attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k, max_q=max_q)
    want, lim = attn_limit(torch, (qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(d)), bf16, p_rounding)
    err = (got.cpu().double() - want).abs()
    assert (err <= lim).all(), (err / lim.clamp(min=1e-30)).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [1, 4096], ids=["few", "prompts"])
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_infinite_value_that_every_row_sees(q, torch_cuda, max_q, bf16):
    """An infinity in V among keys of which every row sees all stays one, whatever probability it has."""
    torch = torch_cuda
    for key in (0, 5, 170):
        qq, kk, vv, at_k = ops.attn_inputs(torch, 4, [3], [300], 2, 1, 128, bf16, qscale=0.2)
        clean = ops.attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), [3], [300], at_k, max_q=max_q)
        vv[key, 0, 3], vv[key, 0, 9] = math.inf, -math.inf
        got = ops.attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), [3], [300], at_k, max_q=max_q)
        assert (got[:, :, 3] == math.inf).all() and (got[:, :, 9] == -math.inf).all()
        got[:, :, 3], got[:, :, 9] = clean[:, :, 3], clean[:, :, 9]
        assert torch.equal(got, clean)


# ------------------------------------------------------------------ delta rule

DEVIATIONS = 3


def delta_bound(torch, qq, kk, vv, g, beta, S, lens):
    """64-bit outputs and states, and the deviations of a token's (head's) and of a state's norms."""
    qq, kk, vv, g, beta, S = (x.double() for x in (qq, kk, vv, g, beta, S))
    rep, h = vv.shape[1] // kk.shape[1], vv.shape[1]
    out, S, at, u2 = torch.zeros_like(vv), S.clone(), 0, U * U
    dev_out, dev_S = torch.zeros(vv.shape[:2], dtype=torch.float64), torch.zeros(S.shape[:2], dtype=torch.float64)
    for i, n in enumerate(lens):
        s, C = S[i], torch.zeros(h, 128, 128, dtype=torch.float64)
        for t in range(at, at + n):
            k, q, b, e = kk[t].repeat_interleave(rep, 0), qq[t].repeat_interleave(rep, 0), beta[t], torch.exp(g[t])
            s = s * e[:, None, None]
            rows = s.square().sum(-1)
            x = torch.einsum("hkv,hk->hv", s, k)
            d = (vv[t] - x) * b[:, None]
            var = u2 * (b * b * (128 * (k * k * rows).sum(-1) + x.square().sum(-1) + vv[t].square().sum(-1)) + d.square().sum(-1))
            Ck = torch.einsum("hij,hj->hi", C, k)
            kk2 = k[:, :, None] * k[:, None, :]
            C = C - b[:, None, None] * (k[:, :, None] * Ck[:, None, :] + Ck[:, :, None] * k[:, None, :])
            C = (C + (b * b * (Ck * k).sum(-1))[:, None, None] * kk2) * (e * e)[:, None, None] + var[:, None, None] * kk2
            s = s + k[:, :, None] * d[:, None, :]
            now = s.square().sum(-1)
            C = C + torch.diag_embed(u2 * ((1 + g[t].square())[:, None].clamp(max=4) * rows + now))
            out[t] = torch.einsum("hkv,hk->hv", s, q)
            dev_out[t] = torch.sqrt(torch.einsum("hi,hij,hj->h", q, C, q) + u2 * (128 * (q * q * now).sum(-1) + out[t].square().sum(-1)))
        S[i], dev_S[i] = s, torch.sqrt(torch.diagonal(C, dim1=-2, dim2=-1).sum(-1))
        at += n
    return out, S, dev_out, dev_S


def delta_excess(out, S, bound, bf16):
    """The largest part of what the bound allows that an output's and a state's norm are off by."""
    want, wS, dev_out, dev_S = bound
    eo = (out.double().cpu()[:want.shape[0]] - want).norm(dim=-1)
    lo = DEVIATIONS * dev_out + (BF * (want.norm(dim=-1) + DEVIATIONS * dev_out) if bf16 else 0)
    eS = (S.double().cpu() - wS).flatten(2).norm(dim=-1)
    part = lambda e, lim: (e / lim.clamp(min=1e-300)).masked_fill(e == 0, 0.0)
    top = lambda x: x.max().item() if x.numel() else 0.0
    return top(part(eo, lo)), top(part(eS, DEVIATIONS * dev_S))


def cut(torch, x):
    """A float as the sum of three bfloat16."""
    parts, x = [], x.float().contiguous()
    for _ in range(3):
        p = (x.view(torch.int32) & -65536).view(torch.float32)
        parts.append(p.double())
        x = x - p
    return parts


def delta_in_chunks(torch, qq, kk, vv, g, beta, S, lens, lost=None):
    """The chunked form with products of three parts, rounded to fp32 once; `lost`: the product without its third parts."""
    qq, kk, vv, g, beta, S = (x.float() for x in (qq, kk, vv, g, beta, S))
    out, S, rep, at = torch.zeros_like(vv), S.clone(), vv.shape[1] // kk.shape[1], 0

    def mul(name, x, y):
        a, b = cut(torch, x), cut(torch, y)
        return sum(a[i] @ b[j] for i in range(3) for j in range(3) if i + j <= (1 if name == lost else 2)).float()

    for i, n in enumerate(lens):
        for h in range(vv.shape[1]):
            s = S[i, h]
            for a in range(at, at + n, 64):
                z = min(a + 64, at + n)
                q, k, v, b = qq[a:z, h // rep], kk[a:z, h // rep], vv[a:z, h], beta[a:z, h, None]
                c = torch.cumsum(g[a:z, h].double(), 0)
                e, ec, rest = torch.exp(c[:, None] - c[None, :]).float(), torch.exp(c).float()[:, None], torch.exp(c[-1] - c).float()[:, None]
                A = torch.tril(b * e * mul("K K^T", k, k.t()), -1)
                P = torch.tril(e * mul("Q K^T", q, k.t()))
                T = torch.linalg.solve_triangular(torch.eye(z - a) + A, torch.eye(z - a), upper=False)
                d = mul("T R", T, b * v - b * ec * mul("K S", k, s))
                out[a:z, h] = mul("Q S", q, s) * ec + mul("P d", P, d)
                s = s * ec[-1] + mul("K^T d", k.t(), d * rest)
            S[i, h] = s
        at += n
    return out, S


PRODUCTS = ["K K^T", "Q K^T", "K S", "T R", "K^T d", "Q S", "P d"]


def host_inputs(monkeypatch, *args, **kw):
    import torch
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "cuda", lambda x: x)
        return ops.delta_inputs(torch, *args, **kw)[0]


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_delta_bounds_see_lost_parts(monkeypatch, bf16):
    """The chunked form passes, each of its products without third parts fails, as do operands cut to bfloat16."""
    import torch
    lens = [200, 1, 0, 70]
    host = host_inputs(monkeypatch, 7, lens, 1, 2, bf16, decay=0.05)
    bound = delta_bound(torch, *host, lens)
    off = lambda *a: max(delta_excess(*a, bound, False))      # (before the outputs' own rounding)
    assert off(*delta_in_chunks(torch, *host, lens)) <= 0.5
    for lost in PRODUCTS if not bf16 else ["K S", "T R", "K^T d", "Q S", "P d"]:      # (bfloat16 q and k have one part)
        assert off(*delta_in_chunks(torch, *host, lens, lost=lost)) > 1, lost
    if not bf16:
        for i in range(3):
            cutoff = list(host)
            cutoff[i] = cut(torch, host[i])[0].float()
            assert off(*delta_in_chunks(torch, *cutoff, lens)) > 100


def test_delta_bounds_hold_for_the_recursion(monkeypatch):
    """Token by token in fp32, whatever the decay, within the bound."""
    import torch
    for lens, decay in (([130], 1.0), ([15, 1, 17], 1.0), ([150], 30.0), ([160], 0.0)):
        host = host_inputs(monkeypatch, 3, lens, 1, 2, False, decay=decay)
        qq, kk, vv, g, beta, S = (x.clone() for x in host)
        out, at = torch.zeros_like(vv), 0
        for i, n in enumerate(lens):
            for t in range(at, at + n):
                k, q = kk[t].expand(2, 128), qq[t].expand(2, 128)
                s = S[i] * torch.exp(g[t])[:, None, None]
                d = (vv[t] - (s * k[:, :, None]).sum(1)) * beta[t][:, None]
                S[i] = s + k[:, :, None] * d[:, None, :]
                out[t] = (S[i] * q[:, :, None]).sum(1)
            at += n
        assert max(delta_excess(out, S, delta_bound(torch, *host, lens), False)) <= 0.5


CUT = r"""
#include <cmath>
#include <cstdio>
#include "qh_seq.hpp"
using namespace qh;
// the three parts come to the float, and the partial products that are left out to less than 2^-21 of a product
int main() {
  uint64_t r = 88172645463325252ull;
  double most = 0;
  for (int i = 0; i < 4000000; ++i) {
    float f[2];
    double p[2][3];
    for (int j = 0; j < 2; ++j) {
      r ^= r << 13, r ^= r >> 7, r ^= r << 17;
      // any significand, half of them with long runs of ones; exponents whose parts are normal numbers
      uint32_t u = (uint32_t)(r >> 20) & 0x807fffffu;
      if (r & 1) u |= 0x007fffffu >> (r >> 60);
      u |= (uint32_t)(100 + (r >> 8) % 50) << 23;
      if (i == 0) u = 0x3f80ffffu;   // below 1 + 2^-7
      f[j] = __builtin_bit_cast(float, u);
      const Cut c = cut_float(f[j]);
      for (int k = 0; k < 3; ++k) p[j][k] = __builtin_bit_cast(float, c.p[k] & 0xffff0000u);
      if (p[j][0] + p[j][1] + p[j][2] != (double)f[j] || (c.p[2] & 0xffffu) != 0) return std::printf("%a is not its parts\n", f[j]), 1;
    }
    const double left = p[0][1] * p[1][2] + p[0][2] * p[1][1] + p[0][2] * p[1][2], of = std::fabs(left / ((double)f[0] * f[1]));
    if (of > most) most = of;
  }
  std::printf("%a\n", most);
  return most < 0x1p-21 && most > 0x1p-22 ? 0 : 2;
}
"""


def test_cut_of_a_float(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(CUT)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "qwen_fpga_amd", "csrc"),
                    "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("decay", [1.0, 0.05])
@pytest.mark.parametrize("max_len", [None, 1], ids=["", "steps"])
@pytest.mark.parametrize("lens,kh,h", ops.DELTA, ids=str)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_delta_precision(q, torch_cuda, lens, kh, h, bf16, max_len, decay):
    torch = torch_cuda
    host, dev = ops.delta_inputs(torch, 3 * sum(lens) + h, lens, kh, h, bf16, decay=decay)
    S = host[5].cuda()
    out = ops.delta_run(q, torch, dev, S, lens, max_len=max_len)
    assert max(delta_excess(out, S, delta_bound(torch, *host, lens), bf16)) <= 1


# ------------------------------------------------------------------ int8 matrix product

# both forms and both sizes of each in several units or tiles along both sides, the last ones ragged and whole; inner
# dimensions that end inside a step of 64, inside the loads ahead and far behind them
GEMM_TILES = [
    (257, 8321, 1040), (1500, 1540, 1024), (1100, 2049, 3584), (640, 4096, 1024), (130, 8324, 272), (258, 8192, 32), (384, 7040, 64),
    (300, 2048, 1040), (256, 2048, 1008), (513, 1028, 3584), (193, 1344, 208), (130, 517, 1008),
    (47, 1000, 1040), (64, 1024, 512), (100, 800, 2064), (33, 68, 4096), (100, 130, 1040), (129, 68, 80),
]


def test_every_form_of_the_product_is_reached(tmp_path):
    """By the launch's own rule, each form with several units or tiles of tokens and of rows, ragged and whole, beyond its
    loads ahead, and with outputs in one store of four and not."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text('#include <cstdio>\n#include <cstdlib>\n#include "qh_seq.hpp"\nint main(int n, char** v) { for (int i = 1; i + 1 < n; i += 2) { '
                   'auto f = qh::gemm_form(atoi(v[i]), atoi(v[i + 1]), 4096); std::printf("%d %d\\n", f.unit, f.tile); } }')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "qwen_fpga_amd", "csrc"), "-o", str(exe), str(src)],
                   check=True)
    r = subprocess.run([str(exe)] + [str(x) for t, o, _ in GEMM_TILES for x in (t, o)], capture_output=True, text=True, check=True)
    forms = [tuple(map(int, line.split())) for line in r.stdout.split("\n") if line]
    assert set(forms) == {(16, 0), (32, 0), (0, 64), (0, 128)}
    for form in set(forms):
        of = [s for s, f in zip(GEMM_TILES, forms) if f == form]
        tok, row = form[0] or form[1], form[1] or 16
        many = [(t, o, k) for t, o, k in of if t > tok and o > row]
        assert any(t % tok for t, _, _ in many) and any(o % row for _, o, _ in many), form
        assert any(k > 1000 and k % 64 for _, _, k in many) and any(o % 4 == 0 for _, o, _ in many), form
        if form[1]:
            assert any(t % tok == 0 and o % row == 0 for t, o, _ in many), form
            assert any(t % tok > tok // 2 or t % tok == 0 for t, _, _ in many), form      # (the waves of a tile's second half)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,out,inn", GEMM_TILES)
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("wide", [False, True], ids=["rows", "contiguous"])
def test_gemm_tiles(q, torch_cuda, tokens, out, inn, bf16, wide):
    """Equal bits; contiguous outputs (one store for four where out is a multiple of 4) and inside wider rows."""
    torch = torch_cuda
    if not wide:
        return ops.test_gemm(q, torch_cuda, tokens, out, inn, bf16)
    g = ops.gen(torch, tokens + out + inn)
    w = torch.randint(-128, 128, (out, inn), generator=g, dtype=torch.int8)
    x = torch.randint(-128, 128, (tokens, inn), generator=g, dtype=torch.int8)
    sw, sx = torch.rand(out, generator=g) * 1e-2, torch.rand(tokens, generator=g)
    want = (x.double() @ w.double().t()).float() * sx[:, None] * sw[None, :]
    y = torch.full((tokens, out), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    q.gemm_i8_w8a8(y, w.cuda(), sw.cuda(), x.cuda(), sx.cuda())
    assert torch.equal(y.cpu(), want.to(y.dtype))


# ------------------------------------------------------------------ delta rule: what is not finite

@functools.lru_cache(None)
def many_heads(bf16):
    import torch
    lens = [150, 70]
    host, _ = ops.delta_inputs(torch, 14, lens, 16, 64, bf16, decay=0.05, fused=False)
    return lens, host, delta_bound(torch, *host, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta", "S"])
@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=str)
def test_delta_non_finite_inputs_of_many_heads(q, torch_cuda, bf16, which, bad):
    """Enough heads for two column tiles a workgroup in bfloat16, key heads with four value heads each: a value that is not
    finite (in a whole chunk's middle, of one value head or one key head) reaches that head's later tokens only, and the other
    heads' and sequences' states and outputs keep the bound."""
    torch = torch_cuda
    lens, clean, bound = many_heads(bf16)
    h, hit, at, host = 64, 22, 75, [x.clone() for x in clean]
    i = ["q", "k", "v", "g", "beta", "S"].index(which)
    if which == "S":
        host[5][0, hit, :, 9] = bad
    elif which in ("q", "k"):
        host[i][at, hit // 4, 5] = bad
    else:
        host[i][(at, hit) if which != "v" else (at, hit, 37)] = bad
    S = host[5].cuda()
    out = ops.delta_run(q, torch, [x.cuda() for x in host[:5]], S, lens).cpu()
    S = S.cpu()
    heads = [hit] if which not in ("q", "k") else list(range(hit // 4 * 4, hit // 4 * 4 + 4))
    rest = [x for x in range(h) if x not in heads]
    first = 0 if which == "S" else at
    pick = lambda o, s, a, b, hh: delta_excess(o[a:b][:, hh], s[:0], (bound[0][a:b][:, hh], bound[1][:0], bound[2][a:b][:, hh], bound[3][:0]), bf16)[0]
    states = lambda i, hh: delta_excess(out[:0], S[i:i + 1, hh], (bound[0][:0], bound[1][i:i + 1, hh], bound[2][:0], bound[3][i:i + 1, hh]), bf16)[1]
    assert pick(out, S, 0, 220, rest) <= 1 and states(0, rest) <= 1 and states(1, list(range(h))) <= 1
    assert pick(out, S, 150, 220, heads) <= 1
    if first:
        assert pick(out, S, 0, first, heads) <= 1
    if which == "q":
        assert not torch.isfinite(out[at, heads]).any() and pick(out, S, at + 1, 150, heads) <= 1 and states(0, heads) <= 1
    elif which == "S":
        assert not torch.isfinite(S[0, hit, :, 9]).any() and not torch.isfinite(out[:150, hit, 9]).any()
        keep = [c for c in range(128) if c != 9]
        assert torch.isfinite(S[0, hit][:, keep]).all() and torch.isfinite(out[:150, hit][:, keep]).all()
    elif which == "v":      # one column
        keep = [c for c in range(128) if c != 37]
        assert not torch.isfinite(S[0, hit, :, 37]).any() and torch.isfinite(S[0, hit][:, keep]).all()
        assert not torch.isfinite(out[at:150, hit, 37]).any() and torch.isfinite(out[:150, hit][:, keep]).all()
    else:
        assert not torch.isfinite(S[0, heads]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("which", ["v", "q", "k", "beta", "g"])
def test_delta_overflow_of_finite_inputs(q, torch_cuda, bf16, which):
    """A finite value from which a token's delta, state or output overflows has no influence on the tokens before it."""
    torch = torch_cuda
    lens, at = [100, 80], 75
    host, _ = ops.delta_inputs(torch, 21, lens, 2, 2, bf16, decay=0.05, fused=False)
    bound = delta_bound(torch, *host, lens)
    big = [x.clone() for x in host]
    if which == "v":            # the second delta is -2 * 3e38, the first and all inputs are finite
        big[1][at + 1, 0] = big[1][at, 0]
        big[2][at, 0], big[2][at + 1, 0] = 3e38, -3e38
        big[3][at:at + 2, 0], big[4][at:at + 2, 0] = 0.0, 1.0
    else:
        big[["q", "k", "", "g", "beta"].index(which)][at, 0] = 150.0 if which == "g" else 3e38
    S = host[5].cuda()
    out = ops.delta_run(q, torch, [x.cuda() for x in big[:5]], S, lens).cpu()
    assert not torch.isfinite(out[at:100, 0]).all()
    for rows, heads in ((slice(0, at), [0, 1]), (slice(0, 100), [1]), (slice(100, 180), [0, 1])):
        part = (bound[0][rows][:, heads], bound[1][:0], bound[2][rows][:, heads], bound[3][:0])
        assert delta_excess(out[rows][:, heads], S[:0], part, bf16)[0] <= 1
    assert delta_excess(out[:0], S[1:], (bound[0][:0], bound[1][1:], bound[2][:0], bound[3][1:]), bf16)[1] <= 1


# ------------------------------------------------------------------ operands in one buffer

VIEWS = r"""
#include <cstdio>
#include <map>
#include <random>
#include "qh_seq_view.hpp"
using namespace qh;
// against every byte in turn: an answer of "apart" is always right, and so is "writable"; the layouts that are used in
// earnest are known for what they are
int main() {
  std::mt19937 g(5);
  auto pick = [&](std::initializer_list<int> v) { return *(v.begin() + g() % v.size()); };
  const uintptr_t base = 1 << 20;
  long apart = 0, write = 0;
  for (int it = 0; it < 60000; ++it) {
    View v[2];
    std::map<uintptr_t, int> bytes[2];
    bool twice[2] = {false, false};
    const int ld = 8 * pick({0, 1, 2, 3, 4, 6, 8, 12}), hs = 8 * pick({0, 1, 2, 3, 4, 9});
    for (int i = 0; i < 2; ++i) {
      v[i] = {nullptr, pick({1, 2, 3, 4}), pick({1, 2, 3}), 8 * pick({1, 1, 2}), g() % 3 ? ld : 8 * pick({1, 2, 4, 5, 8, 16}),
              g() % 3 ? hs : 8 * pick({1, 2, 3, 8, 16}), 2};
      v[i].p = reinterpret_cast<const void*>(base + 16 * (g() % 12));
      for (int r = 0; r < v[i].rows; ++r)
        for (int h = 0; h < v[i].heads; ++h)
          for (int d = 0; d < v[i].dim * 2; ++d) twice[i] |= ++bytes[i][v[i].at() + 2 * (r * v[i].ld + h * v[i].hs) + d] > 1;
      if (!v[i].countable()) return std::printf("not countable\n"), 1;
      if (v[i].writable()) {
        ++write;
        if (twice[i]) return std::printf("%d rows %d heads of %d, %d and %d apart, taken as writable\n", (int)v[i].rows, (int)v[i].heads,
                                         (int)v[i].dim, (int)v[i].ld, (int)v[i].hs), 1;
      }
    }
    if (overlap(v[0], v[1]) != overlap(v[1], v[0])) return std::printf("not symmetric\n"), 1;
    if (!overlap(v[0], v[1])) {
      ++apart;
      for (auto& b : bytes[0])
        if (bytes[1].count(b.first)) return std::printf("%d: taken as apart\n", it), 1;
    }
  }
  if (apart < 5000 || write < 5000) return std::printf("%ld apart, %ld writable\n", apart, write), 1;
  auto at = [&](int64_t el) { return reinterpret_cast<const void*>(base + 2 * el); };
  const View out{at(128), 40, 8, 128, 8 * 256, 256, 2}, q{at(0), 40, 8, 128, 8 * 256, 256, 2};   // halves of each head
  if (overlap(out, q) || !overlap(View{at(64), 40, 8, 128, 8 * 256, 256, 2}, q)) return std::printf("halves\n"), 1;
  const View odd{at(0), 3, 4, 128, 2 * 128, 5 * 128, 2};   // every other row of head-major rows, five a head
  if (!odd.writable()) return std::printf("every other row\n"), 1;
  // (strides of dimensions with one entry do not count, whatever they are)
  const View one{at(0), 1, 1, 128, INT64_MAX, INT64_MIN, 2}, next{at(128), 1, 1, 128, INT64_MIN, INT64_MAX, 2};
  if (!one.writable() || !one.countable() || overlap(one, next) || !overlap(one, one) || !overlap(one, q)) return std::printf("one entry\n"), 1;
  if (View{at(0), 1 << 30, 4, 128, (int64_t)1 << 39, 128, 4}.countable() || View{at(0), 4, 1 << 30, 128, 128, (int64_t)1 << 39, 4}.countable())
    return std::printf("too far\n"), 1;
  return 0;
}
"""


def test_views(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(VIEWS)
    subprocess.run(["g++", "-std=c++17", "-O0", "-Wall", "-Wextra", "-Werror", "-ftrapv", "-I", os.path.join(ROOT, "qwen_fpga_amd", "csrc"),
                    "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_strides_too_far_to_count(q):
    """Refused before a span is counted (the products would not fit 64 bits)."""
    a, far = seq_ops.Args(q), (1 << 40) - 16
    assert a.delta(tokens=1 << 29, heads=2, ldo=far) == q.QH_ERANGE
    assert a.delta(tokens=1 << 29, heads=2, ldo=256, ldb=far) == q.QH_ERANGE
    assert a.attn(q_rows=1 << 24, ldq=far) == q.QH_ERANGE
    assert a.attn(k_rows=1 << 30, ldv=far) == q.QH_ERANGE


def test_more_sequences_than_a_search_is_for(q):
    """Every workgroup looks through all of them: a million would take minutes."""
    a = seq_ops.Args(q)
    assert a.attn(n_seq=65537, q_rows=70000) == q.QH_ERANGE and a.attn(n_seq=1 << 20, q_rows=1 << 20) == q.QH_ERANGE
    assert q.attention_seq_workspace(70000, 65537, 1, 1000, 2, 1, 128) == 0 < q.attention_seq_workspace(70000, 65536, 1, 1000, 2, 1, 128)


def test_sizes_beyond_an_int(q, monkeypatch):
    """Refused, where the C ABI would be given their low 32 bits: by the calls, with tensors that hold no memory, and by
    the workspaces' queries."""
    import torch
    monkeypatch.setattr(q, "_on", lambda t, what: None)
    monkeypatch.setattr(q, "_op", lambda name: lambda *a: pytest.fail(f"{name} was called with {a}"))
    f32, i8, i32, i64 = torch.float32, torch.int8, torch.int32, torch.int64

    def z(*shape, dt=f32, many=None):      # a dimension of `many` entries in one place
        t = torch.empty([1 if i == many else n for i, n in enumerate(shape)], dtype=dt, device="meta")
        return t.expand(*shape) if many is not None else t

    def refused(call, *args):
        with pytest.raises(q.QHError) as e:
            call(*args)
        assert e.value.status == q.QH_ERANGE

    for big in ((1 << 32) + 4, 1 << 32, 1 << 31):
        refused(q.gemm_i8_w8a8, z(big, 16), z(16, 32, dt=i8), z(16), z(big, 32, dt=i8, many=0), z(big))
        refused(q.gemm_i8_w8a8, z(4, big), z(big, 32, dt=i8), z(big), z(4, 32, dt=i8), z(4))
        a, k = z(big, 2, 128, many=0), z(9, 1, 128)
        refused(q.delta_rule_seq, a, a, a, a, z(big, 2), z(big, 2), z(1, 2, 128, 128), z(2, dt=i32), None, 4)
        refused(q.attention_seq, a, a, k, k, z(2, dt=i32), z(1, dt=i64), z(1, dt=i32), None, 4, 9)
        refused(q.attention_seq, z(4, 2, 128), z(4, 2, 128), k, k, z(big + 1, dt=i32), z(big, dt=i64), z(big, dt=i32), None, 4, 9)
        a, g = z(4, 2, 128), z(4, 2)
        refused(q.delta_rule_seq, a, a, a, a, g, g, z(1, 2, 128, 128), z(2, dt=i32), None, big)
        refused(q.attention_seq, a, a, k, k, z(2, dt=i32), z(1, dt=i64), z(1, dt=i32), None, 4, big)
        refused(q.attention_seq, a, a, k, k, z(2, dt=i32), z(1, dt=i64), z(1, dt=i32), None, big, 9)
        refused(q.delta_rule_seq_workspace, big, 1, 2, 100)
        refused(q.delta_rule_seq_workspace, 100, 1, 2, big)
        refused(q.attention_seq_workspace, big, 1, 4, 9, 2, 1, 128)
        refused(q.attention_seq_workspace, 4, 1, 4, big, 2, 1, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_outputs_beside_their_inputs(q, torch_cuda, bf16):
    """Outputs in the gate halves of the projection whose query halves are read, and in every other row of head-major
    rows of odd number: as elsewhere, and the rest of the buffer as it was."""
    torch = torch_cuda
    lens, ctx, h, kvh, d = [40, 1, 0, 30], [40, 90, 3, 31], 4, 2, 128
    qq, kk, vv, at_k = ops.attn_inputs(torch, 5, lens, ctx, h, kvh, d, bf16)
    t, dev = sum(lens), [x.cuda() for x in (qq, kk, vv)]
    want = ops.attn_run(q, torch, *dev, lens, ctx, at_k)
    both = torch.cat([dev[0], torch.full_like(dev[0], 7.0)], -1)
    ops.attn_run(q, torch, both[:, :, :d], *dev[1:], lens, ctx, at_k, out=both[:, :, d:])
    assert torch.equal(both[:, :, d:], want) and torch.equal(both[:, :, :d], dev[0])
    rows = torch.full((h, 2 * t - 1, d), 7.0, dtype=qq.dtype, device="cuda")
    ops.attn_run(q, torch, *dev, lens, ctx, at_k, out=rows[:, ::2].transpose(0, 1))
    assert torch.equal(rows[:, ::2].transpose(0, 1), want) and (rows[:, 1::2] == 7).all()
    host, dd = ops.delta_inputs(torch, 8, lens, 4, 4, bf16, fused=False)
    S, S2 = host[5].cuda(), host[5].cuda()
    want = ops.delta_run(q, torch, dd, S, lens)
    both = torch.cat([dd[2], torch.full_like(dd[2], 7.0)], -1)
    ops.delta_run(q, torch, dd[:2] + [both[:, :, :128]] + dd[3:], S2, lens, out=both[:, :, 128:])
    assert torch.equal(both[:, :, 128:], want) and torch.equal(both[:, :, :128], dd[2]) and torch.equal(S, S2)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("cu", [[0, 300, 0, 300, 0, 310], [0, 310, 5, 200, 90, 310], [0, 70, 70, 10, 250, 250]], ids=str)
def test_sequences_that_share_rows(q, torch_cuda, bf16, cu):
    """Bounds that go back: the calls end, and leave alone what lies around their outputs, states and workspaces."""
    torch = torch_cuda
    t, h, kvh, n, dt = 320, 4, 2, len(cu) - 1, torch.bfloat16 if bf16 else torch.float32
    g = ops.gen(torch, 3)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    qq, kk, vv = rnd(t, h, 128), rnd(2000, kvh, 128), rnd(2000, kvh, 128)
    dk = torch.nn.functional.normalize(rnd(t, kvh, 128).float(), dim=-1).to(dt)

    def room(need):      # a workspace inside a larger array of one value
        buf = torch.full((need + 1024,), 0x5A, dtype=torch.uint8, device="cuda")
        return buf, buf[512:512 + need] if need else None

    for max_q, max_k in ((1, 1), (1, 2000), (320, 2000), (4096, 2000), (4096, 300)):
        buf, ws = room(q.attention_seq_workspace(t, n, max_q, max_k, h, kvh, 128))
        out = torch.full((t + 2, h, 128), 7.0, dtype=dt, device="cuda")
        q.attention_seq(out[1:-1], qq, kk, vv, i32(cu), torch.arange(n, device="cuda") * 10, i32([1900] * n), ws, max_q, max_k)
        assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[311:] == 7).all()
        assert (buf[:512] == 0x5A).all() and (buf[-512:] == 0x5A).all()
    for max_len in (1, 320):
        buf, ws = room(q.delta_rule_seq_workspace(t, n, h, max_len, k_heads=kvh, dtype=q.BF16 if bf16 else q.F32))
        S, out = torch.full((n + 2, h, 128, 128), 0.5, device="cuda"), torch.full((t + 2, h, 128), 7.0, dtype=dt, device="cuda")
        q.delta_rule_seq(out[1:-1], dk, dk, qq, torch.full((t, h), -0.1, device="cuda"), torch.full((t, h), 0.5, device="cuda"), S[1:-1], i32(cu),
                         ws, max_len)
        assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[311:] == 7).all()
        assert (S[0] == 0.5).all() and (S[-1] == 0.5).all() and (buf[:512] == 0x5A).all() and (buf[-512:] == 0x5A).all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_k", [100, 400])
def test_attention_of_thousands_of_sequences(q, torch_cuda, max_k):
    """One token each; empty ones and long ones among them."""
    torch = torch_cuda
    lens = [i % 7 != 3 for i in range(2500)]
    ctx = [1 + (37 * i) % 90 for i in range(2500)]
    for i in (0, 64, 1000, 2499):
        lens[i], ctx[i] = 1, 390
    lens = [int(n) for n in lens]
    qq, kk, vv, at_k = ops.attn_inputs(torch, 17, lens, ctx, 2, 1, 128, True)
    got = ops.attn_run(q, torch, qq.cuda(), kk.cuda(), vv.cuda(), lens, ctx, at_k, max_k=max_k)
    want, lim = attn_limit(torch, (qq, kk, vv, lens, ctx, at_k, 1 / math.sqrt(128)), True, FEW)
    assert ((got.cpu().double() - want).abs() <= lim).all()


# ------------------------------------------------------------------ calls beside one another

@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_calls_at_the_same_time(q, torch_cuda, bf16):
    """Two streams, each with outputs, states and workspaces of its own, over the same inputs, in both forms; and the two
    captured and replayed beside each other: every result that of a call alone."""
    torch = torch_cuda
    lens, ctx, at_k = [260, 1, 130], [2000, 900, 1500], [0, 1000, 500]      # (keys that sequences share)
    t, h, kvh = sum(lens), 8, 2
    qq, kk, vv, _ = ops.attn_inputs(torch, 19, lens, [2000], h, kvh, 128, bf16)
    host, dev = ops.delta_inputs(torch, 19, lens, 2, h, bf16, fused=False)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    args = [x.cuda() for x in (qq, kk, vv)] + [i32(ops.starts(lens)), torch.tensor(at_k, device="cuda"), i32(ctx)]
    S0, cu = host[5].cuda(), i32(ops.starts(lens))

    class Call:
        def __init__(self, max_q, max_len):
            u8 = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")
            self.max_q, self.max_len, self.S = max_q, max_len, S0.clone()
            self.out, self.do = torch.empty_like(args[0]), torch.empty_like(dev[2])
            self.w1, self.w2 = u8(q.attention_seq_workspace(t, 3, max_q, 2000, h, kvh, 128)), u8(q.delta_rule_seq_workspace(t, 3, h, max_len))

        def run(self):
            self.S.copy_(S0)
            q.attention_seq(self.out, *args, self.w1, self.max_q, 2000)
            q.delta_rule_seq(self.do, *dev, self.S, cu, self.w2, self.max_len)

        def all(self):
            return [self.out, self.do, self.S]

    for max_q, max_len in ((1, 260), (4096, 260), (260, 1)):
        calls, streams = [Call(max_q, max_len), Call(max_q, max_len)], [torch.cuda.Stream(), torch.cuda.Stream()]
        calls[0].run()
        want = [x.clone() for x in calls[0].all()]
        graphs = []
        for c in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                c.run()
            graphs.append(g)
        for replay in (False, True, True):
            for c in calls:
                for x in c.all():
                    x.zero_()
            torch.cuda.synchronize()
            for _ in range(3):
                for c, s, g in zip(calls, streams, graphs):
                    with torch.cuda.stream(s):
                        g.replay() if replay else c.run()
            torch.cuda.synchronize()
            for c in calls:
                assert all(torch.equal(x, y) for x, y in zip(c.all(), want))
    scale = 1 / math.sqrt(128)
    wo, lim = attn_limit(torch, (qq, kk, vv, lens, ctx, at_k, scale), bf16, PROMPTS)
    assert ((want[0].cpu().double() - wo).abs() <= lim).all()
    assert max(delta_excess(want[1], want[2], delta_bound(torch, *host, lens), bf16)) <= 1
