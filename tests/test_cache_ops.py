"""Operators around an int8 K/V cache, on the CPU: the rules that the kernels take from their header (which rows of the
cache a token may name, the scale of a row), the host's refusals and the workspace's sizes."""
import ctypes
import os
import subprocess
import sys

import pytest

from conftest import ROOT

RULES = r"""
#include <cmath>
#include <cstdio>
#include <cstring>
#include <cstdint>
#include <climits>
#include <initializer_list>
#include "qh_seq.hpp"
using namespace qh;
#define REQUIRE(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  for (int64_t rows : {(int64_t)0, (int64_t)1, (int64_t)100, (int64_t)1 << 34})
    for (int64_t s : {INT64_MIN, (int64_t)-1, (int64_t)0, (int64_t)1, (int64_t)99, (int64_t)100, ((int64_t)1 << 34) - 1, (int64_t)1 << 34, INT64_MAX})
      REQUIRE(has_slot(s, rows) == (s >= 0 && s < rows));
  // a scale is never 0 and a code never past 127 by more than a rounding, down to the smallest number
  REQUIRE(code_scale(0.0f) == 1.0f);
  for (uint32_t u = 1; u < 0x7f800000u; u += u < 200000 ? 1 : 9973) {
    float top;
    std::memcpy(&top, &u, 4);
    const float s = code_scale(top);
    REQUIRE(s > 0.0f && std::isfinite(s));
    if (top / 127.0f > 0.0f) REQUIRE(s == top / 127.0f);
    const float r = std::nearbyint(top / s);
    REQUIRE(r >= 1.0f && r <= 191.0f && (top < 0x1p-120f || r == 127.0f));   // (clipped to 127 after that)
  }
  return 0;
}
"""


def test_rules(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(RULES)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "qwen_fpga_amd", "csrc"), "-o",
                    str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


class Args:
    """A call's arguments by name: good ones (host addresses that no kernel reads, since every call here is refused or
    has nothing to do), and the ones that a case changes."""

    def __init__(self, q):
        self.q = q
        self.buf = ctypes.create_string_buffer(1 << 20)
        base = (ctypes.addressof(self.buf) + 255) & ~255
        self.at = lambda i: base + (i << 15)
        self.names = {}

    def call(self, name, d, kw):
        assert set(kw) <= set(d)
        d.update(kw)
        return self.q._op(name)(*d.values())

    def rope(self, **kw):
        at = self.at
        return self.call("qh_qk_norm_rope_seq", dict(
            q_out=at(0), ldqo=256, hsqo=128, k_out=at(1), ldko=128, hsko=128, q=at(2), ldq=256, hsq=128, k=at(3), ldk=128, hsk=128,
            type=0, q_norm=at(4), k_norm=at(5), pos=at(6), tokens=3, heads=2, kv_heads=1, d=128, rope_dim=64, theta=1e7, eps=1e-6,
            stream=None), kw)

    def write(self, **kw):
        at = self.at
        return self.call("qh_kv_cache_write_i8", dict(
            kq=at(0), ldkq=256, hskq=128, ks=at(1), ldks=2, hsks=1, vq=at(2), ldvq=256, hsvq=128, vs=at(3), ldvs=2, hsvs=1, k=at(4),
            ldk=256, hsk=128, v=at(5), ldv=256, hsv=128, type=0, slot=at(6), rows=9, tokens=3, kv_heads=2, d=128, stream=None), kw)

    def read(self, **kw):
        at = self.at
        return self.call("qh_kv_cache_read_i8", dict(
            k=at(4), ldk=256, hsk=128, v=at(5), ldv=256, hsv=128, type=0, kq=at(0), ldkq=256, hskq=128, ks=at(1), ldks=2, hsks=1,
            vq=at(2), ldvq=256, hsvq=128, vs=at(3), ldvs=2, hsvs=1, slot=at(6), rows=9, tokens=3, kv_heads=2, d=128, stream=None), kw)

    def attn(self, **kw):
        at = self.at
        return self.call("qh_attention_seq_i8", dict(
            out=at(0), ldo=256, hso=128, q=at(1), ldq=256, hsq=128, type=0, kq=at(2), ldkq=128, hskq=128, ks=at(3), ldks=1, hsks=1,
            vq=at(4), ldvq=128, hsvq=128, vs=at(5), ldvs=1, hsvs=1, cu_q=at(6), k_start=at(7), k_len=at(8), n_seq=1, q_rows=3,
            k_rows=9, max_q=3, max_k=9, heads=2, kv_heads=1, d=128, scale=0.1, ws=at(10), ws_bytes=1 << 18, stream=None), kw)


@pytest.fixture(scope="module")
def args(q):
    return Args(q)


def changed(kw, at):
    """'a+8': a's address moved; 'a=b': a at b's address."""
    if not isinstance(kw, str):
        return kw
    name, what = kw.replace("=", "+").split("+")
    return {name: at[what] if "=" in kw else at[name] + int(what)}


@pytest.mark.parametrize("kw", [
    dict(type=2), dict(tokens=-1), dict(heads=0), dict(kv_heads=0), dict(d=64), dict(rope_dim=-16), dict(rope_dim=8), dict(rope_dim=144),
    dict(theta=0.0), dict(theta=0.999), dict(theta=float("nan")), dict(theta=float("inf")), dict(eps=-1.0), dict(eps=float("nan")), dict(q_out=None),
    dict(k_out=None), dict(q=None), dict(k=None), dict(q_norm=None), dict(k_norm=None), dict(pos=None), dict(ldqo=128), dict(ldqo=0),
    dict(hsqo=64), dict(ldko=64), dict(ldq=258), dict(hsk=128, ldk=-128), "q_out+4", "k+8", "q_norm+4", "k_norm+8", "q_out=k", "q_out=k_out",
    "k_out=q", "k_out=pos", "q_out=q_norm", "q+128", dict(ldq=128, hsq=384),
], ids=str)
def test_norm_rope_refusals(q, args, kw):
    at = dict(q_out=args.at(0), k_out=args.at(1), q=args.at(2), k=args.at(3), q_norm=args.at(4), k_norm=args.at(5), pos=args.at(6))
    kw = changed(kw, at)
    if kw in ({"q": at["q"] + 128}, dict(ldq=128, hsq=384)):     # in place, but a row or a stride off
        kw = {**kw, "q_out": at["q"]}
    assert args.rope(**kw) == q.QH_EINVAL


def test_norm_rope_nothing_to_do_and_ranges(q, args):
    assert args.rope(tokens=0, q=None, pos=None) == q.QH_OK
    assert args.rope(tokens=(1 << 23) + 1) == q.QH_ERANGE
    assert args.rope(tokens=1 << 23, heads=2047, kv_heads=1 << 30) == q.QH_ERANGE
    assert args.rope(ldq=(1 << 40) - 4, tokens=1 << 23) == q.QH_ERANGE


REFUSED = [
    dict(type=3), dict(tokens=-1), dict(rows=-1), dict(kv_heads=0), dict(d=192), dict(kq=None), dict(ks=None), dict(vq=None), dict(vs=None),
    dict(k=None), dict(v=None), dict(slot=None), dict(ldkq=8), dict(hskq=-128), dict(ldks=-1), dict(hsvs=1 << 40), dict(ldvq=1 << 40),
    dict(ldk=2), dict(hsv=6), "kq+8", "vq+4", "ks+2", "vs+1", "k+4", "v+8",
]


@pytest.mark.parametrize("kw", REFUSED + [
    dict(ldkq=128), dict(hskq=64), dict(ldks=1), dict(hsks=0), dict(ldvs=0), dict(ldvq=0),      # two elements in one place
    "kq=vq", "kq=ks", "kq=k", "kq=slot", "ks=vs", "ks=vq", "vs=v", "vq=k", "vs=slot",
], ids=str)
def test_cache_write_refusals(q, args, kw):
    at = {n: args.at(i) for i, n in enumerate(("kq", "ks", "vq", "vs", "k", "v", "slot"))}
    assert args.write(**changed(kw, at)) == q.QH_EINVAL


@pytest.mark.parametrize("kw", REFUSED + [
    dict(ldk=128), dict(ldv=0), dict(hsk=64), "k=v", "k=kq", "v=vs", "k=slot", "v=vq", "k=ks",
], ids=str)
def test_cache_read_refusals(q, args, kw):
    at = {n: args.at(i) for i, n in enumerate(("kq", "ks", "vq", "vs", "k", "v", "slot"))}
    assert args.read(**changed(kw, at)) == q.QH_EINVAL


def test_cache_nothing_to_do_and_ranges(q, args):
    for call in (args.write, args.read):
        assert call(tokens=0, slot=None) == q.QH_OK and call(rows=0, kq=None) == q.QH_OK
        assert call(tokens=(1 << 25) + 1) == q.QH_ERANGE
        assert call(rows=1 << 40) == q.QH_ERANGE
        assert call(rows=(1 << 40) - 1, ldkq=(1 << 40) - 16) == q.QH_ERANGE      # past 2^61 bytes
    # K's and V's codes (and scales) side by side in the rows of one buffer share nothing
    at = args.at(0)
    side = dict(kq=at, vq=at + 256, ldkq=512, ldvq=512, ks=args.at(1), vs=args.at(1) + 8, ldks=4, ldvs=4)
    assert args.write(tokens=0, **side) == q.QH_OK and args.write(slot=None, **side) == q.QH_EINVAL
    assert args.write(**{**side, "vq": at + 240}) == q.QH_EINVAL and args.write(**{**side, "vs": args.at(1) + 4}) == q.QH_EINVAL


@pytest.mark.parametrize("kw", [
    dict(type=7), dict(n_seq=-1), dict(q_rows=-1), dict(k_rows=-1), dict(max_q=-1), dict(max_k=-1), dict(heads=0), dict(kv_heads=0),
    dict(heads=3, kv_heads=2), dict(d=64), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None), dict(q=None),
    dict(kq=None), dict(ks=None), dict(vq=None), dict(vs=None), dict(cu_q=None), dict(k_start=None), dict(k_len=None), dict(ldo=130),
    dict(ldo=0), dict(hso=0), dict(ldq=-256), dict(ldkq=8), dict(ldvq=-16), dict(ldks=-1), dict(hsq=2), "out+8", "kq+8", "vq+4", "ks+2",
    "vs+1", "out=q", "out=kq", "out=ks", "out=vq", "out=vs", "out=cu_q", "out=k_start", "out=k_len",
], ids=str)
def test_attention_refusals(q, args, kw):
    at = {n: args.at(i) for i, n in enumerate(("out", "q", "kq", "ks", "vq", "vs", "cu_q", "k_start", "k_len"))}
    assert args.attn(**changed(kw, at)) == q.QH_EINVAL


def test_attention_nothing_to_do_ranges_and_workspace(q, args):
    assert args.attn(q_rows=0) == q.QH_OK and args.attn(n_seq=0) == q.QH_OK
    assert args.attn(max_k=(1 << 30) + 1) == q.QH_ERANGE
    assert args.attn(n_seq=65537) == q.QH_ERANGE
    assert args.attn(q_rows=1 << 30, heads=4) == q.QH_ERANGE and args.attn(q_rows=33000000) == q.QH_ERANGE
    for name in ("ldkq", "ldvq", "ldks", "ldvs"):
        assert args.attn(**{name: 1 << 24}) == q.QH_ERANGE
        assert args.attn(k_rows=1, cu_q=None, **{name: 1 << 24}) == q.QH_EINVAL    # (one row has no next one)
    need = q.attention_seq_i8_workspace(3, 1, 1, 100000, 2, 1, 128)   # few rows, many keys: the keys are split
    assert need > 0
    for ws in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=args.at(10) + 16), dict(ws=args.at(1)), dict(ws=args.at(3) - 256)):
        assert args.attn(max_q=1, max_k=100000, **{"ws_bytes": need, **ws}) == q.QH_EINVAL
    assert q.attention_seq_i8_workspace(0, 1, 1, 100000, 2, 1, 128) == 0
    with pytest.raises(q.QHError):
        q.attention_seq_i8_workspace(1 << 32, 1, 1, 100000, 2, 1, 128)


def test_python_checks_need_no_gpu(q):
    import torch

    f, i8 = lambda *s: torch.zeros(*s), lambda *s: torch.zeros(*s, dtype=torch.int8)
    cache = lambda: (i8(9, 1, 128), f(9, 1), i8(9, 1, 128), f(9, 1))
    slot = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="CUDA"):
        q.qk_norm_rope_seq(f(2, 2, 128), f(2, 1, 128), f(2, 2, 128), f(2, 1, 128), f(128), f(128), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="CUDA"):
        q.kv_cache_write_i8(*cache(), f(2, 1, 128), f(2, 1, 128), slot)
    with pytest.raises(TypeError, match="CUDA"):
        q.kv_cache_read_i8(f(2, 1, 128), f(2, 1, 128), *cache(), slot)
    with pytest.raises(TypeError, match="CUDA"):
        q.attention_seq_i8(f(2, 2, 128), f(2, 2, 128), *cache(), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64),
                           torch.zeros(1, dtype=torch.int32), None, 2, 2)
    with pytest.raises(ValueError, match="dimensions"):
        q.kv_cache_write_i8(*cache(), f(2, 128), f(2, 128), slot)


@pytest.mark.parametrize("call", [
    "qk_norm_rope_seq(f(2, 2, 128), f(2, 1, 128), f(2, 2, 128), f(2, 1, 128), f(128), f(128), torch.zeros(2, dtype=torch.int32))",
    "kv_cache_write_i8(*c, f(2, 1, 128), f(2, 1, 128), s)",
    "kv_cache_read_i8(f(2, 1, 128), f(2, 1, 128), *c, s)",
    "attention_seq_i8(f(2, 2, 128), f(2, 2, 128), *c, s[:0].int(), s[:1], s[:1].int(), None, 2, 2)",
], ids=lambda c: c.split("(")[0])
def test_any_operator_may_be_the_first(call):
    """The library is loaded by the first call, whichever it is: the operands' types are known then (here, that they are not on the GPU)."""
    code = ("import torch, qwen_fpga_amd as q\n"
            "f, i8, s = torch.zeros, lambda *n: torch.zeros(*n, dtype=torch.int8), torch.zeros(2, dtype=torch.int64)\n"
            "c = i8(9, 1, 128), f(9, 1), i8(9, 1, 128), f(9, 1)\n"
            f"try:\n    q.{call}\nexcept TypeError as e:\n    assert 'CUDA' in str(e), e\nelse:\n    raise SystemExit('taken')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0, r.stderr


def prompts(q, q_rows, n_seq, max_q, max_k, heads, kv_heads, dim, bf16):
    """Whether a call takes the form for prompts, by its workspace: 512 places (or two tiles' and more) of `tile` rows; the one for
    few rows asks for those of 16 rows, or for none."""
    nb = q.attention_seq_i8_workspace(q_rows, n_seq, max_q, max_k, heads, kv_heads, dim, q.BF16 if bf16 else q.F32)
    tile, rows = 256 if bf16 else 128, q_rows * (heads // kv_heads)
    few = (min(rows // 16 + n_seq, rows) * kv_heads + 512) * (16 * dim + 32) * 4
    assert max_k > 3000                                  # (fewer keys may need no workspace in either form)
    if nb in (0, few):
        return False
    assert nb % (tile * (dim + 2) * 4) == 0 and 0 < nb // (tile * (dim + 2) * 4) <= 512
    return True


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 256), (8, 8, 128)])
def test_attention_form_of_mixed_calls(q, bf16, heads, kv_heads, dim):
    """Single tokens beside a short part of a prompt take the form for few rows, whatever the pairs come to when all rows see the
    longest keys; a long prompt beside a few of them takes the one for prompts, and so do equal sequences that fill tiles."""
    f = lambda *a: prompts(q, *a, heads, kv_heads, dim, bf16)
    for single, keys, part in ((31, 30000, 65), (31, 30000, 512), (255, 8000, 128), (31, 4000, 512), (100, 4000, 1000), (128, 4000, 300),
                               (60000, 8000, 4096)):
        assert not f(single + part, single + 1, part, keys)
    assert f(4096, 64, 4096, 8192) and f(4100, 256, 4096, 8192)           # places that are empty, as the rows tell, count for nothing
    assert f(7 + 8000, 8, 8000, 8000) and f(31 + 20000, 32, 20000, 20000)
    assert f(1, 1, 1 << 26, 4000) and f(300, 150, 1 << 26, 4000)          # a bound of many rows asks for it
    if heads > kv_heads:
        assert f(64 * 400, 64, 400, 4000)
    # as before for one sequence
    assert f(4000, 1, 4000, 8000) and f(512, 1, 512, 8000) and not f(512, 1, 512, 3001) and not f(1, 1, 1, 131071)


FORMS = r"""
#include <cstdio>
#include <initializer_list>
#include "qh_seq.hpp"
using namespace qh;
#define REQUIRE(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  auto one = [](int n, int past, int heads, int kv, int dim, bool bf16) {
    return attn_i8_prompts(n, 1, n, n + past, heads, kv, dim, bf16 ? 256 : 128, bf16);
  };
  for (bool bf16 : {false, true}) {
    for (int n : {1, 64, 512, 1024, 1500, 2000}) REQUIRE(!one(n, 0, 8, 2, 256, bf16) && !one(n, 0, 8, 8, 128, bf16));
    REQUIRE(!one(512, 1488, 8, 2, 256, bf16) && one(512, 3488, 8, 2, 256, bf16) && one(300, 15700, 8, 2, 256, bf16));
    REQUIRE(!one(512, 1488, 8, 8, 128, bf16) && one(512, 3488, 8, 8, 128, bf16) && !one(64, 31936, 8, 2, 256, bf16));
    REQUIRE(one(256, 3840, 16, 4, 128, bf16) && one(6000, 0, 8, 2, 256, bf16));
    REQUIRE(one(1 << 26, 0, 1, 1, 128, bf16) && attn_i8_prompts(1, 1, 1 << 26, 1, 1, 1, 128, bf16 ? 256 : 128, bf16));
  }
  REQUIRE(one(2300, 0, 8, 2, 256, true) && one(3000, 0, 8, 8, 128, true) && one(2300, 0, 16, 4, 128, true));
  REQUIRE(!one(2300, 0, 8, 2, 256, false) && !one(2000, 0, 16, 4, 128, false) && !one(1500, 0, 16, 4, 128, true));
  // the most that a call can have stays within 64 bits
  REQUIRE(attn_i8_prompts(0x7fffffff, 1, 0x7fffffff, 1 << 30, 1, 1, 128, 256, true));
  REQUIRE(!attn_i8_prompts(0x7fffffff / 64, 65536, 1, 1 << 30, 64, 1, 128, 256, true));
  return 0;
}
"""


def test_attention_form(tmp_path):
    """What was the faster form on the card, by the rule itself (which the few keys that need no workspace do not show)."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(FORMS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-ftrapv", "-I",
                    os.path.join(ROOT, "qwen_fpga_amd", "csrc"), "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


WAVES = r"""
#include <cstdio>
#include <initializer_list>
#include "qh_seq.hpp"
using namespace qh;
#define REQUIRE(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  for (bool bf16 : {false, true}) {
    // never a wave without rows
    for (int tokens : {1, 100, 1792, 1793, 4096, 16000, 1 << 23})
      for (int dim : {128, 256})
        for (int rows = 2; rows <= 512 / dim; ++rows) REQUIRE(norm_rope_waves(tokens, rows, dim, bf16) == 1);
    // rows of the call, not its tokens alone
    for (int tokens : {1, 1000, 2000, 3000, 8000}) REQUIRE(norm_rope_waves(tokens, 40, 256, bf16) == 4);
    REQUIRE(norm_rope_waves(1500, 10, 256, bf16) == 4 && norm_rope_waves(2000, 10, 256, bf16) == 1 && norm_rope_waves(2000, 20, 128, bf16) == 1);
    REQUIRE(norm_rope_waves(8000, 5, 256, bf16) == 1 && norm_rope_waves(1 << 23, 0x1fffffffell, 256, bf16) == 4);
  }
  REQUIRE(norm_rope_waves(8000, 10, 256, true) == 1 && norm_rope_waves(8000, 10, 256, false) == 4 && norm_rope_waves(4000, 10, 256, false) == 1);
  return 0;
}
"""


def test_norm_rope_waves(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(WAVES)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-ftrapv", "-I", os.path.join(ROOT, "qwen_fpga_amd", "csrc"),
                    "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
