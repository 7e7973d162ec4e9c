"""The operators over packed sequences, as cases that can be timed and checked.

Kinds (a case is a dict of plain values; ``kind`` names one of these):

  gemm   int8 activations of many tokens times an int8 weight, a scale for each token and output row
         (gemm_i8_w8a8; the activations come from quant_rows, one row a token)
  delta  the gated delta rule over packed sequences, each with its own state (delta_rule_seq)
  attn   causal attention of packed queries over each sequence's rows of a K/V cache (attention_seq)

``lens`` is the text of each sequence's number of new tokens, ``ctx`` of each sequence's keys (the new ones
included; shorter texts repeat).  Sizes are the model's own (1024 hidden, 3584 inner, 248320 rows of
vocabulary, 16 DeltaNet heads of 128, 8 query and 2 key heads of 256) or generic.
"""
import math

import torch

own = False      # the plain forms; true: the framework's kernels

DEV = "cuda"
KD = 128         # key and value width of the delta rule


def listed():
    return [
        # the k or v projection of one token: the smallest call, where latency counts
        {"name": "gemm_kv_1", "kind": "gemm", "tokens": 1, "out": 512, "k": 1024, "bf16": False},
        # the down projection of a short prompt, both sizes odd
        {"name": "gemm_down_63", "kind": "gemm", "tokens": 63, "out": 1021, "k": 3584, "bf16": True},
        # the LM head for a batch of requests that decode together: the weight is what is read
        {"name": "gemm_head_16", "kind": "gemm", "tokens": 16, "out": 248320, "k": 1024, "bf16": False},
        # gate and up of a pasted document, ragged length
        {"name": "gemm_gateup_1500", "kind": "gemm", "tokens": 1500, "out": 7168, "k": 1024, "bf16": False},
        # the down projection of several documents together
        {"name": "gemm_down_4096", "kind": "gemm", "tokens": 4096, "out": 1024, "k": 3584, "bf16": True},
        # 32 requests that decode together: one token each, every state read and written
        {"name": "delta_decode_32", "kind": "delta", "lens": ",".join(["1"] * 32), "kh": 16, "h": 16, "bf16": False},
        # one pasted document in the framework's own precision: a chain over its tokens
        {"name": "delta_prompt_1500", "kind": "delta", "lens": "1500", "kh": 16, "h": 16, "bf16": False},
        # ragged documents packed together, an empty one among them, value heads that share key heads
        {"name": "delta_packed_7k", "kind": "delta", "lens": "2049,3,640,0,1111,1,2500,97,63,64,65,700", "kh": 16, "h": 32,
         "bf16": True},
        # 16 requests that decode together over caches of different lengths
        {"name": "attn_decode_16", "kind": "attn", "lens": "1", "n": 16, "h": 8, "kv": 2, "d": 256,
         "ctx": "8191,17,4096,1023,300,2048,5000,1,7777,64,640,3333,129,6001,15,2500", "bf16": False},
        # one request over a very long document
        {"name": "attn_decode_long", "kind": "attn", "lens": "1", "n": 1, "h": 8, "kv": 2, "d": 256, "ctx": "131071", "bf16": True},
        # one pasted document in the framework's own precision
        {"name": "attn_prompt_1500", "kind": "attn", "lens": "1500", "n": 1, "h": 8, "kv": 2, "d": 256, "ctx": "1500", "bf16": False},
        # ragged documents packed together, one of them behind a cached prefix
        {"name": "attn_packed_16k", "kind": "attn", "lens": "8000,1,2047,0,640,4100,257,1300", "n": 8, "h": 8, "kv": 2, "d": 256,
         "ctx": "8000,1,2047,0,640,4100,4353,1300", "bf16": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ragged(rng, total, n):
    """n lengths (some zero) that come to `total` at most."""
    w = [0.0 if n > 3 and rng.random() < 0.08 else rng.random() ** 2 + 0.002 for _ in range(n)]
    s = sum(w) or 1.0
    return [int(total * x / s) for x in w]


def draw(rng):
    kind = rng.choice(["gemm", "delta", "attn"])
    c = {"kind": kind, "bf16": rng.random() < 0.5}
    if kind == "gemm":
        if rng.random() < 0.15:                  # a vocabulary
            c["tokens"], c["out"], c["k"] = rng.randint(1, 16), _log(rng, 32000, 248320), 1024
        else:
            c["tokens"], c["out"], c["k"] = _log(rng, 1, 4096), _log(rng, 16, 8192), 16 * _log(rng, 4, 256)
        return c
    if kind == "delta":
        c["kh"], c["h"] = rng.choice([(16, 16), (16, 16), (16, 32), (4, 8), (2, 2)])
        if rng.random() < 0.4:                   # decoding together
            lens = [rng.choice([1, 1, 1, 1, 0, 2, 4]) for _ in range(_log(rng, 1, 48))]
            if sum(lens) == 0:
                lens[0] = 1
        else:
            lens = _ragged(rng, _log(rng, 40, 7000), rng.randint(1, 12))
            lens = [min(x, 2500) for x in lens]
        c["lens"] = ",".join(str(x) for x in lens)
        return c
    c["h"], c["kv"], c["d"] = rng.choice([(8, 2, 256), (8, 2, 256), (8, 2, 256), (8, 8, 128), (16, 4, 128), (16, 2, 256), (6, 2, 128)])
    if rng.random() < 0.45:                      # one token each
        c["n"] = _log(rng, 1, 32)
        lens = [1] * c["n"]
        top = min(131071, 65_000_000 // (c["n"] * c["kv"] * c["d"]))
        ctx = [_log(rng, 1, top) for _ in lens]
    else:
        c["n"] = rng.randint(1, 8)
        lens = _ragged(rng, _log(rng, 16, int(8000 * math.sqrt(2048 / (c["h"] * c["d"])))), c["n"])
        if sum(lens) == 0:
            lens[0] = 1
        # some behind a cached prefix, a long one where the new part is short
        ctx = [x + (_log(rng, 1, 12000 if x < 300 else 1000) if x and rng.random() < 0.3 else 0) for x in lens]
    c["lens"], c["ctx"] = ",".join(str(x) for x in lens), ",".join(str(x) for x in ctx)
    return c


def _ints(text, n=None):
    v = [int(x) for x in text.split(",")]
    return v if n is None else [v[i % len(v)] for i in range(n)]


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _starts(lens):
    s = [0]
    for x in lens:
        s.append(s[-1] + x)
    return s


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    dt = torch.bfloat16 if case["bf16"] else torch.float32
    s = {"case": case, "kind": kind}
    if kind == "gemm":
        t, out, k = case["tokens"], case["out"], case["k"]
        s["xq"] = torch.randint(-127, 128, (t, k), generator=g, device=DEV, dtype=torch.int8)
        s["sx"] = (0.5 + torch.rand(t, generator=g, device=DEV)) / 40.0
        s["w"] = torch.randint(-127, 128, (out, k), generator=g, device=DEV, dtype=torch.int8)
        s["sw"] = (0.5 + torch.rand(out, generator=g, device=DEV)) / (73.0 * math.sqrt(k))
        s["y"] = torch.empty(t, out, device=DEV, dtype=dt)
        return s
    if kind == "delta":
        lens = _ints(case["lens"])
        cu, kh, h = _starts(lens), case["kh"], case["h"]
        t = cu[-1]
        # q, k, v as the short convolution leaves them: one row of all heads a token; q and k normalised
        qkv = _randn(g, t, (2 * kh + h) * KD)
        qk = qkv[:, :2 * kh * KD].view(t, 2 * kh, KD)
        qk /= torch.sqrt((qk * qk).sum(-1, keepdim=True) + 1e-6)
        qk[:, :kh] /= math.sqrt(KD)
        qkv = qkv.to(dt)
        s["q"] = qkv[:, :kh * KD].view(t, kh, KD)
        s["k"] = qkv[:, kh * KD:2 * kh * KD].view(t, kh, KD)
        s["v"] = qkv[:, 2 * kh * KD:].view(t, h, KD)
        A = 1.0 + 15.0 * torch.rand(h, generator=g, device=DEV)
        s["g"] = -A * torch.log1p(torch.exp(_randn(g, t, h) - 3.0))
        s["beta"] = 1.0 / (1.0 + torch.exp(-_randn(g, t, h)))
        s["S"] = _randn(g, len(lens), h, KD, KD, scale=0.05)
        s["out"] = torch.empty(t, h, KD, device=DEV, dtype=dt)
        s["cu"], s["lens"] = torch.tensor(cu, dtype=torch.int32, device=DEV), lens
        if own:
            import qwen_fpga_amd as fw
            s["ws"] = torch.empty(fw.delta_rule_seq_workspace(t, len(lens), h, max(lens)), dtype=torch.uint8, device=DEV)
        return s
    n, h, kv, d = case["n"], case["h"], case["kv"], case["d"]
    lens, ctx = _ints(case["lens"], n), _ints(case["ctx"], n)
    cu, ks = _starts(lens), _starts(ctx)
    # the query half of a query and gate projection; caches packed one after another
    s["q"] = _randn(g, cu[-1], h, 2 * d, scale=1.5).to(dt)[:, :, :d]
    s["k"], s["v"] = _randn(g, max(ks[-1], 1), kv, d).to(dt), _randn(g, max(ks[-1], 1), kv, d).to(dt)
    s["out"] = torch.empty(cu[-1], h, d, device=DEV, dtype=dt)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    s["ks"] = torch.tensor(ks[:n], dtype=torch.int64, device=DEV)
    s["kl"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    s["lens"], s["ctx"] = lens, ctx
    if own:
        import qwen_fpga_amd as fw
        nb = fw.attention_seq_workspace(cu[-1], n, max(lens), max(ctx), h, kv, d)
        s["ws"] = torch.empty(nb, dtype=torch.uint8, device=DEV)
    return s


def run(s):
    if own:
        import qwen_fpga_amd as fw
        if s["kind"] == "gemm":
            fw.gemm_i8_w8a8(s["y"], s["w"], s["sw"], s["xq"], s["sx"])
            return s["y"]
        if s["kind"] == "delta":
            fw.delta_rule_seq(s["out"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["S"], s["cu"], s["ws"], max(s["lens"]))
            return {"out": s["out"], "S": s["S"]}
        fw.attention_seq(s["out"], s["q"], s["k"], s["v"], s["cu"], s["ks"], s["kl"], s["ws"], max(s["lens"]), max(s["ctx"]))
        return s["out"]
    return _PLAIN[s["kind"]](s)


# --------------------------------------------------------------------------- plain forms


def _gemm(s):
    y = torch.matmul(s["xq"].float(), s["w"].float().t())
    s["y"].copy_(y * s["sx"][:, None] * s["sw"][None, :])
    return s["y"]


def _delta(s):
    """Token by token, all sequences side by side (the longest first, so that those still running are a prefix)."""
    lens, h = s["lens"], s["case"]["h"]
    rep = h // s["case"]["kh"]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    idx = torch.tensor(order, device=DEV)
    at = s["cu"][:-1][idx].long()
    decay, beta = torch.exp(s["g"]), s["beta"]
    q, k, v = s["q"].float().repeat_interleave(rep, 1), s["k"].float().repeat_interleave(rep, 1), s["v"].float()
    S = s["S"][idx]
    for t in range(max(lens)):
        n = sum(1 for x in lens if x > t)
        r = at[:n] + t
        st = S[:n] * decay[r][:, :, None, None]
        kt = k[r]
        dl = (v[r] - torch.matmul(kt[:, :, None, :], st)[:, :, 0]) * beta[r][:, :, None]
        st = st + kt[:, :, :, None] * dl[:, :, None, :]
        s["out"][r] = torch.matmul(q[r][:, :, None, :], st)[:, :, 0].to(s["out"].dtype)
        S[:n] = st
    s["S"][idx] = S
    return {"out": s["out"], "S": s["S"]}


def _attn(s):
    c = s["case"]
    h, kv, d = c["h"], c["kv"], c["d"]
    at = ks = 0
    for n, m in zip(s["lens"], s["ctx"]):
        if n:
            kk = s["k"][ks:ks + m].float().permute(1, 2, 0).contiguous()          # [kv, d, m]
            vv = s["v"][ks:ks + m].float().transpose(0, 1).contiguous()           # [kv, m, d]
            cols = torch.arange(m, device=DEV)
            for a in range(0, n, 2048):
                b = min(a + 2048, n)
                qq = s["q"][at + a:at + b].float().transpose(0, 1).reshape(kv, -1, d)   # [kv, h / kv * rows, d]
                p = torch.matmul(qq, kk).view(h, b - a, m) / math.sqrt(d)
                p = p.masked_fill(cols[None, :] > torch.arange(a, b, device=DEV)[:, None] + (m - n), float("-inf"))
                p = torch.exp(p - p.amax(-1, keepdim=True))
                p = p / p.sum(-1, keepdim=True)
                o = torch.matmul(p.view(kv, -1, m), vv).view(h, b - a, d)
                s["out"][at + a:at + b] = o.transpose(0, 1).to(s["out"].dtype)
        at, ks = at + n, ks + m
    return s["out"]


_PLAIN = {"gemm": _gemm, "delta": _delta, "attn": _attn}


# --------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    kind, eb = case["kind"], 2 if case["bf16"] else 4
    if kind == "gemm":
        t, out, k = case["tokens"], case["out"], case["k"]
        return {"bytes": (t + out) * (k + 4) + eb * t * out, "flops": 2 * t * out * k}
    if kind == "delta":
        lens = _ints(case["lens"])
        t, n = sum(lens), sum(1 for x in lens if x)
        kh, h = case["kh"], case["h"]
        return {"bytes": t * (eb * KD * (2 * kh + 2 * h) + 8 * h) + 8 * n * h * KD * KD, "flops": 7 * KD * KD * h * t}
    n, h, kv, d = case["n"], case["h"], case["kv"], case["d"]
    lens, ctx = _ints(case["lens"], n), _ints(case["ctx"], n)
    pairs = sum(q * m - q * (q - 1) // 2 for q, m in zip(lens, ctx))
    return {"bytes": eb * d * (2 * h * sum(lens) + 2 * kv * sum(m for q, m in zip(lens, ctx) if q)), "flops": 4 * d * h * pairs}


# --------------------------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gemm":
        x, y = s["xq"].double(), []
        for a in range(0, case["out"], 32768):
            y.append((s["w"][a:a + 32768].double() @ x.t()).t() * s["sw"][a:a + 32768].double())
        return torch.cat(y, 1) * s["sx"].double()[:, None]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    if case["kind"] == "delta":
        rep = case["h"] // case["kh"]
        S, a = s["S"].double(), 0
        for i, n in enumerate(s["lens"]):
            M = S[i].transpose(1, 2).contiguous()                                 # [h, v, k]
            for t in range(a, a + n):
                kt, qt = (s[x][t].double().repeat_interleave(rep, 0)[:, :, None] for x in ("k", "q"))
                M = M * torch.exp(s["g"][t].double())[:, None, None]
                e = (s["v"][t].double()[:, :, None] - M @ kt) * s["beta"][t].double()[:, None, None]
                M = torch.baddbmm(M, e, kt.transpose(1, 2).contiguous())
                out[t] = (M @ qt)[:, :, 0]
            S[i] = M.transpose(1, 2)
            a += n
        return {"out": out, "S": S}
    h, kv, d = case["h"], case["kv"], case["d"]
    at = ks = 0
    for n, m in zip(s["lens"], s["ctx"]):
        for j in range(h if n else 0):
            kk, vv = (s[x][ks:ks + m, j // (h // kv)].double() for x in ("k", "v"))
            for a in range(0, n, 4096):
                b = min(a + 4096, n)
                sc = s["q"][at + a:at + b, j].double() @ (kk.t() / math.sqrt(d))
                hide = torch.ones(b - a, m, dtype=torch.bool, device=DEV).triu(a + m - n + 1)
                out[at + a:at + b, j] = torch.softmax(sc.masked_fill_(hide, -math.inf), -1) @ vv
        at, ks = at + n, ks + m
    return out
