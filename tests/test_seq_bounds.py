"""Operators over packed sequences: bounds tight enough to see a lost part of a product, a lost step or a form that no
other test reaches.  On the CPU each bound is shown to fail for a planted mistake in the oracle's place; on the device
the kernels are held to it.

Attention, bfloat16.  A product with P adds to the fp32 bound (tests/test_gpu_seq_ops.py) what P's rounding takes: the form for
few rows multiplies V with P in two bfloat16 parts, the first cut (p - hi < 2^-7 p) and the second rounded (2^-8 of itself) and moved
up by 2^-18 p, 2^-14 sum p |v| in all; the form for prompts rounds each probability once, 2^-8 sum p |v|.  Both round the output
once, 2^-8 of it.
"""
import math

import pytest

import test_gpu_seq_ops as ops

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
