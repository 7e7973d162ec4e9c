"""The operators around an int8 K/V cache, as cases that can be timed and checked.

Kinds (a case is a dict of plain values; ``kind`` names one of these):

  rope   the norms of queries and keys for each head with the position rotation (qk_norm_rope_seq)
  write  new keys and values quantised into the cache, and the rows read back as the values that they now stand
         for (kv_cache_write_i8, kv_cache_read_i8)
  read   rows of the cache gathered as values (kv_cache_read_i8)
  attn   causal attention of packed queries over each sequence's rows of the int8 cache (attention_seq_i8)

``h``, ``kv``, ``d`` are query heads, key heads and their width; ``lens`` is the text of each sequence's number of
new tokens, ``ctx`` of each sequence's keys (the new ones included; shorter texts repeat).  Sizes are the model's own
(8 query and 2 key heads of 256, 64 rotated, base 1e7) or generic.
"""
import math

import torch

own = False      # the plain forms; true: the framework's kernels

DEV = "cuda"
THETA, EPS = 1e7, 1e-6


def listed():
    return [
        # one request's next token far into a document: the smallest call, where latency counts
        {"name": "norm_rope_1", "kind": "rope", "tokens": 1, "h": 8, "kv": 2, "d": 256, "rot": 64, "first": 131071, "bf16": False},
        # one pasted document in the framework's own precision
        {"name": "norm_rope_1500", "kind": "rope", "tokens": 1500, "h": 8, "kv": 2, "d": 256, "rot": 64, "first": 0, "bf16": False},
        # ragged documents packed together
        {"name": "norm_rope_16k", "kind": "rope", "tokens": 16345, "h": 8, "kv": 2, "d": 256, "rot": 64, "first": 9, "bf16": True},
        # 32 requests that decode together, each into its own part of the cache, three places of the batch unused
        {"name": "write_32", "kind": "write", "tokens": 35, "kv": 2, "d": 256, "rows": 65536, "run": 1, "pad": 3, "bf16": False},
        # packed documents, each into rows of its own
        {"name": "write_16k", "kind": "write", "tokens": 16345, "kv": 2, "d": 256, "rows": 65536, "run": 1300, "pad": 0, "bf16": True},
        # a short cached prefix taken out for another use
        {"name": "read_640", "kind": "read", "tokens": 641, "kv": 2, "d": 256, "rows": 8192, "run": 641, "pad": 0, "bf16": False},
        # the caches of several long documents, in blocks
        {"name": "read_60k", "kind": "read", "tokens": 60001, "kv": 2, "d": 256, "rows": 131072, "run": 4000, "pad": 0, "bf16": True},
        # 16 requests that decode together over caches of different lengths
        {"name": "attn_i8_decode_16", "kind": "attn", "lens": "1", "n": 16, "h": 8, "kv": 2, "d": 256,
         "ctx": "8191,17,4096,1023,300,2048,5000,1,7777,64,640,3333,129,6001,15,2500", "bf16": False},
        # one request over a very long document
        {"name": "attn_i8_decode_long", "kind": "attn", "lens": "1", "n": 1, "h": 8, "kv": 2, "d": 256, "ctx": "131071", "bf16": True},
        # one pasted document in the framework's own precision
        {"name": "attn_i8_prompt_1500", "kind": "attn", "lens": "1500", "n": 1, "h": 8, "kv": 2, "d": 256, "ctx": "1500", "bf16": False},
        # the next part of a long prompt behind what the cache holds of it
        {"name": "attn_i8_part_512", "kind": "attn", "lens": "512", "n": 1, "h": 8, "kv": 2, "d": 256, "ctx": "8000", "bf16": True},
        # ragged documents packed together, one of them behind a cached prefix
        {"name": "attn_i8_packed_16k", "kind": "attn", "lens": "8000,1,2047,0,640,4100,257,1300", "n": 8, "h": 8, "kv": 2, "d": 256,
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
    kind = rng.choice(["rope", "write", "read", "attn", "attn"])
    c = {"kind": kind, "bf16": rng.random() < 0.5}
    c["h"], c["kv"], c["d"] = rng.choice([(8, 2, 256), (8, 2, 256), (8, 2, 256), (8, 8, 128), (16, 4, 128), (16, 2, 256), (6, 2, 128)])
    small = 2048 / (c["h"] * c["d"])
    if kind == "rope":
        c["tokens"] = _log(rng, 1, int(16000 * small))
        c["rot"] = rng.choice([64, 64, 32, 128, c["d"], 0])
        c["first"] = _log(rng, 1, 1000000) - 1
        return c
    if kind in ("write", "read"):
        c["tokens"] = _log(rng, 1, int((16000 if kind == "write" else 60000) * 512 / (c["kv"] * c["d"])))
        c["pad"] = rng.choice([0, 0, 1, c["tokens"] // 5])
        c["rows"] = c["tokens"] + _log(rng, 1, 65536)
        c["run"] = min(c["tokens"], _log(rng, 1, 4000))
        del c["h"]
        return c
    if rng.random() < 0.45:                      # one token each
        c["n"] = _log(rng, 1, 32)
        lens = [1] * c["n"]
        top = min(131071, 65_000_000 // (c["n"] * c["kv"] * c["d"]))
        ctx = [_log(rng, 1, top) for _ in lens]
    else:
        c["n"] = rng.randint(1, 8)
        lens = _ragged(rng, _log(rng, 16, int(8000 * math.sqrt(small))), c["n"])
        if sum(lens) == 0:
            lens[0] = 1
        # some behind a cached prefix, a long one where the new part is short
        ctx = [x + (_log(rng, 1, 12000 if x < 300 else 1000) if x and rng.random() < 0.3 else 0) for x in lens]
    c["lens"], c["ctx"] = ",".join(str(x) for x in lens), ",".join(str(x) for x in ctx)
    return c


def _ints(text, n):
    v = [int(x) for x in text.split(",")]
    return [v[i % len(v)] for i in range(n)]


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


def _cache(g, rows, kv, d):
    """A cache that holds something: codes and their scales, a scale for each row and head."""
    x = _randn(g, max(rows, 1), kv, d)
    s = x.abs().amax(-1) / 127.0
    return torch.round(x / s[..., None]).to(torch.int8), s


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    dt = torch.bfloat16 if case["bf16"] else torch.float32
    s = {"case": case, "kind": kind}
    if kind == "rope":
        t, h, kv, d = case["tokens"], case["h"], case["kv"], case["d"]
        # the query halves of a query and gate projection; keys in rows of their own
        s["q"] = _randn(g, t, h, 2 * d, scale=1.5).to(dt)[:, :, :d]
        s["k"] = _randn(g, t, kv, d, scale=0.7).to(dt)
        s["qw"], s["kw"] = _randn(g, d, scale=0.2), _randn(g, d, scale=0.2)
        s["pos"] = torch.arange(case["first"], case["first"] + t, dtype=torch.int32, device=DEV)
        s["qo"], s["ko"] = torch.empty(t, h, d, dtype=dt, device=DEV), torch.empty(t, kv, d, dtype=dt, device=DEV)
        return s
    if kind in ("write", "read"):
        t, kv, d, rows, run = case["tokens"], case["kv"], case["d"], case["rows"], case["run"]
        (s["kq"], s["ks"]), (s["vq"], s["vs"]) = _cache(g, rows, kv, d), _cache(g, rows, kv, d)
        # runs of neighbouring rows, the runs in any order; the batch's last places hold no token
        at = torch.randperm(rows // run, generator=g, device=DEV)
        slot = (at[:, None] * run + torch.arange(run, device=DEV)).reshape(-1)
        slot = torch.cat([slot, torch.arange(slot.numel(), rows, device=DEV)])[:t]
        n = t - case["pad"]
        slot[n:] = -1
        s["slot"], s["n"] = slot, n
        s["ko"], s["vo"] = torch.zeros(t, kv, d, dtype=dt, device=DEV), torch.zeros(t, kv, d, dtype=dt, device=DEV)
        if kind == "write":
            # keys with a few wide columns, as norms and rotations leave them; one row of keys and values a token
            row = _randn(g, t, 2 * kv, d) * (0.5 + 4.0 * torch.rand(d, generator=g, device=DEV) ** 8)
            row = row.to(dt)
            s["k"], s["v"] = row[:, :kv], row[:, kv:]
        return s
    n, h, kv, d = case["n"], case["h"], case["kv"], case["d"]
    lens, ctx = _ints(case["lens"], n), _ints(case["ctx"], n)
    cu, ks = _starts(lens), _starts(ctx)
    s["q"] = _randn(g, cu[-1], h, d, scale=1.5).to(dt)
    (s["kq"], s["ks"]), (s["vq"], s["vs"]) = _cache(g, ks[-1], kv, d), _cache(g, ks[-1], kv, d)
    s["out"] = torch.empty(cu[-1], h, d, device=DEV, dtype=dt)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    s["k_start"] = torch.tensor(ks[:n], dtype=torch.int64, device=DEV)
    s["k_len"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    s["lens"], s["ctx"] = lens, ctx
    if own:
        import qwen_fpga_amd as fw
        nb = fw.attention_seq_i8_workspace(cu[-1], n, max(lens), max(ctx), h, kv, d, fw.BF16 if case["bf16"] else fw.F32)
        s["ws"] = torch.empty(nb, dtype=torch.uint8, device=DEV)
    return s


def run(s):
    if own:
        import qwen_fpga_amd as fw
        if s["kind"] == "rope":
            fw.qk_norm_rope_seq(s["qo"], s["ko"], s["q"], s["k"], s["qw"], s["kw"], s["pos"], s["case"]["rot"], THETA, EPS)
            return {"q": s["qo"], "k": s["ko"]}
        if s["kind"] == "attn":
            fw.attention_seq_i8(s["out"], s["q"], s["kq"], s["ks"], s["vq"], s["vs"], s["cu"], s["k_start"], s["k_len"], s["ws"],
                                max(s["lens"]), max(s["ctx"]))
            return s["out"]
        if s["kind"] == "write":
            fw.kv_cache_write_i8(s["kq"], s["ks"], s["vq"], s["vs"], s["k"], s["v"], s["slot"])
        fw.kv_cache_read_i8(s["ko"], s["vo"], s["kq"], s["ks"], s["vq"], s["vs"], s["slot"])
        return {"k": s["ko"], "v": s["vo"]}
    return _PLAIN[s["kind"]](s)


# --------------------------------------------------------------------------- plain forms


def _rope(s):
    half = s["case"]["rot"] // 2
    turn = THETA ** (-torch.arange(half, dtype=torch.float64, device=DEV) / max(half, 1))
    a = s["pos"].double()[:, None, None] * turn          # in 64 bits: far positions are many turns
    cos, sin = torch.cos(a).float(), torch.sin(a).float()

    def one(x, w):
        x = x.float()
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * (1.0 + w)
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)

    s["qo"].copy_(one(s["q"], s["qw"]))
    s["ko"].copy_(one(s["k"], s["kw"]))
    return {"q": s["qo"], "k": s["ko"]}


def _write(s):
    slot = s["slot"][:s["n"]]

    def one(q, sc, x):
        x = x[:s["n"]].float()
        top = x.abs().amax(-1)
        f = torch.where(top > 0, top / 127.0, 1.0)
        q[slot] = torch.clamp(torch.round(x / f[..., None]), -127, 127).to(torch.int8)
        sc[slot] = f

    one(s["kq"], s["ks"], s["k"])
    one(s["vq"], s["vs"], s["v"])
    return _read(s)


def _read(s):
    slot = s["slot"][:s["n"]]
    s["ko"][:s["n"]] = (s["kq"][slot].float() * s["ks"][slot][..., None]).to(s["ko"].dtype)
    s["vo"][:s["n"]] = (s["vq"][slot].float() * s["vs"][slot][..., None]).to(s["vo"].dtype)
    return {"k": s["ko"], "v": s["vo"]}


def _attn(s):
    c = s["case"]
    h, kv, d = c["h"], c["kv"], c["d"]
    at = ks = 0
    for n, m in zip(s["lens"], s["ctx"]):
        if n:
            r = slice(ks, ks + m)
            kk = (s["kq"][r].float() * s["ks"][r][..., None]).permute(1, 2, 0).contiguous()       # [kv, d, m]
            vv = (s["vq"][r].float() * s["vs"][r][..., None]).transpose(0, 1).contiguous()        # [kv, m, d]
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


_PLAIN = {"rope": _rope, "write": _write, "read": _read, "attn": _attn}


# --------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    kind, eb = case["kind"], 2 if case["bf16"] else 4
    kv, d = case["kv"], case["d"]
    if kind == "rope":
        n, t = case["h"] + kv, case["tokens"]
        return {"bytes": 2 * eb * n * d * t + 4 * t + 8 * d, "flops": 6 * n * d * t}
    if kind in ("write", "read"):
        t = case["tokens"] - case["pad"]
        row = 2 * kv * (eb * d + d + 4)                     # values and codes with their scale, once
        passes = 2 if kind == "write" else 1
        return {"bytes": passes * (row * t + 8 * case["tokens"]), "flops": 2 * passes * kv * d * t}
    n, h = case["n"], case["h"]
    lens, ctx = _ints(case["lens"], n), _ints(case["ctx"], n)
    pairs = sum(q * m - q * (q - 1) // 2 for q, m in zip(lens, ctx))
    keys = sum(m for q, m in zip(lens, ctx) if q)
    return {"bytes": 2 * eb * d * h * sum(lens) + 2 * kv * (d + 4) * keys, "flops": 4 * d * h * pairs}


# --------------------------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    kind, d = case["kind"], case["d"]
    if kind == "rope":
        i = torch.arange(d, device=DEV)
        half, rot = case["rot"] // 2, case["rot"]
        ang = torch.zeros(case["tokens"], 1, d, dtype=torch.float64, device=DEV)
        if rot:
            w = torch.exp((i[:rot] % half).double() * (-math.log(THETA) / half))
            ang[:, 0, :rot] = torch.outer(s["pos"].double(), w)
        other = torch.where(i < half, i + half, torch.where(i < rot, i - half, i))
        sign = torch.where(i < half, -1.0, 1.0).double()
        out = {}
        for name, w in (("q", s["qw"]), ("k", s["kw"])):
            x = s[name].double()
            y = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / d + EPS) * (w.double() + 1.0)
            out[name] = y * torch.cos(ang) + y[..., other] * sign * torch.sin(ang)
        return out
    if kind in ("write", "read"):
        out = {}
        for name, src, q, sc in (("k", "k", "kq", "ks"), ("v", "v", "vq", "vs")):
            y = torch.zeros(s["ko"].shape, dtype=torch.float64, device=DEV)
            if kind == "read":
                y[:s["n"]] = torch.index_select(s[q], 0, s["slot"][:s["n"]]).double() * torch.index_select(s[sc], 0, s["slot"][:s["n"]]).double().unsqueeze(-1)
            else:
                x = s[src][:s["n"]].double()
                f = x.abs().max(-1, keepdim=True).values / 127
                y[:s["n"]] = torch.round(x / f.clamp_min(1e-300)) * f
            out[name] = y
        return out
    h, kv = case["h"], case["kv"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    at = ks = 0
    for n, m in zip(s["lens"], s["ctx"]):
        for j in range(h if n else 0):
            kk, vv = (s[x][ks:ks + m, j // (h // kv)].double() * s[f][ks:ks + m, j // (h // kv), None].double()
                      for x, f in (("kq", "ks"), ("vq", "vs")))
            for a in range(0, n, 4096):
                b = min(a + 4096, n)
                sc = s["q"][at + a:at + b, j].double() @ (kk.t() / math.sqrt(d))
                hide = torch.ones(b - a, m, dtype=torch.bool, device=DEV).triu(a + m - n + 1)
                out[at + a:at + b, j] = torch.softmax(sc.masked_fill_(hide, -math.inf), -1) @ vv
        at, ks = at + n, ks + m
    return out
