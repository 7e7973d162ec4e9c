"""Operators over packed sequences, on the CPU: the index rules that bound device data (compiled from the
kernels' own header), the host's refusals, and the workspaces' sizes."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

SRC = r"""
#include <cstdio>
#include <cstdint>
#include <climits>
#include <initializer_list>
#include "qh_seq.hpp"
using namespace qh;
#define REQUIRE(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  const int bad[] = {INT_MIN, -7, -1, 0, 1, 2, 5, 63, 64, 65, 100, 101, INT_MAX - 1, INT_MAX};
  for (int a : bad)                       // whatever the bounds hold, the rows lie inside the array
    for (int b : bad)
      for (int rows : {0, 1, 64, 100}) {
        const SeqSpan s = seq_span(a, b, rows);
        REQUIRE(s.len >= 0 && s.start >= 0 && (int64_t)s.start + s.len <= rows);
        if (a >= 0 && a <= b && b <= rows) REQUIRE(s.start == a && s.len == b - a);
        else REQUIRE(s.len == 0);
      }
  const int64_t at[] = {INT64_MIN, -1, 0, 1, 50, 99, 100, 101, (int64_t)1 << 33, INT64_MAX};
  for (int64_t s : at)
    for (int n : bad)
      for (int64_t rows : {(int64_t)0, (int64_t)100, (int64_t)1 << 34}) {
        const int k = key_len(s, n, rows);
        if (s >= 0 && n >= 0 && n <= kMaxKeys && s <= rows && n <= rows - s) REQUIRE(k == n);
        else REQUIRE(k == -1);
      }
  for (int q : {0, 1, 2, 17, 64})         // a row sees no key past its own, and none of a bad range
    for (int k : {-1, 0, 1, 5, 17, 64, 1000, kMaxKeys})
      for (int r = 0; r < q; ++r) {
        const int n = keys_seen(r, q, k);
        REQUIRE(n >= 0 && (k < 0 ? n == 0 : n <= k));
        REQUIRE(n == 0 || (int64_t)n == (int64_t)r + 1 + k - q);
        if (r > 0) REQUIRE(n >= keys_seen(r - 1, q, k));
      }
  for (int tile : {1, 16, 32, 64, 128})   // the tiles of any packing fit the bound
    for (int n : {1, 2, 7})
      for (int base : {0, 1, 15, 16, 17, 127, 128, 129}) {
        int64_t rows = 0, t = 0;
        for (int i = 0; i < n; ++i) rows += base + i, t += seq_tiles(base + i, tile);
        REQUIRE(t <= seq_tiles_max(rows, n, tile));
      }
  REQUIRE(seq_tiles(INT_MAX, 16) == 134217728);
  return 0;
}
"""


def test_index_rules(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-ftrapv", "-I",
                    os.path.join(ROOT, "qwen_fpga_amd", "csrc"), "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


PAST = r"""
#include <cstdio>
#include <initializer_list>
#include "qh_seq.hpp"
using namespace qh;
// tiles_past counts the tiles whose last row sees more than `keys` keys: against each tile in turn
int main() {
  for (int len : {0, 1, 2, 31, 33, 64, 127, 300})
    for (int k : {-1, 0, 1, 5, 64, 200, 299, 300, 301, 1000, kMaxKeys})
      for (int G : {1, 2, 3, 4, 7, 32})
        for (int tile : {128, 256}) {
          const int nt = seq_tiles(len * G, tile);
          for (int64_t keys : {(int64_t)0, (int64_t)1, (int64_t)31, (int64_t)32, (int64_t)64, (int64_t)128, (int64_t)299, (int64_t)300,
                               (int64_t)999, (int64_t)1000, (int64_t)kMaxKeys, (int64_t)64 * kMaxKeys}) {
            int n = 0;
            for (int t = 0; t < nt; ++t) {
              const int last = ((t + 1) * tile < len * G ? (t + 1) * tile : len * G) - 1;
              n += keys_seen(last / G, len, k) > keys;
            }
            if (tiles_past(len, k, G, tile, nt, keys) != n) {
              std::printf("len %d keys %d G %d tile %d past %d: %d, not %d\n", len, k, G, tile, (int)keys, tiles_past(len, k, G, tile, nt, keys), n);
              return 1;
            }
          }
        }
  return 0;
}
"""


def test_tiles_past(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PAST)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-ftrapv", "-I",
                    os.path.join(ROOT, "qwen_fpga_amd", "csrc"), "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


class Args:
    """A call's arguments by name: good ones (host addresses that no kernel reads, since every call here is
    refused or has nothing to do), and the ones that a case changes."""

    def __init__(self, q):
        self.q = q
        self.buf = ctypes.create_string_buffer(1 << 20)
        base = (ctypes.addressof(self.buf) + 255) & ~255
        self.at = lambda i: base + (i << 15)

    def gemm(self, **kw):
        d = dict(y=self.at(0), ldy=32, type=0, w=self.at(4), scale=self.at(6), xq=self.at(7), ldx=64, sx=self.at(8), tokens=3,
                 out=32, inn=64, stream=None)
        assert set(kw) <= set(d)
        d.update(kw)
        return self.q._op("qh_gemm_i8_w8a8")(*d.values())

    def delta(self, **kw):
        d = dict(out=self.at(0), ldo=256, hso=128, q=self.at(1), ldq=128, hsq=128, k=self.at(2), ldk=128, hsk=128, v=self.at(3),
                 ldv=256, hsv=128, type=0, g=self.at(4), ldg=2, beta=self.at(5), ldb=2, S=self.at(8), cu=self.at(6), n_seq=1,
                 tokens=3, max_len=3, k_heads=1, heads=2, ws=self.at(20), ws_bytes=1 << 18, stream=None)
        assert set(kw) <= set(d)
        d.update(kw)
        return self.q._op("qh_delta_rule_seq")(*d.values())

    def attn(self, **kw):
        d = dict(out=self.at(0), ldo=256, hso=128, q=self.at(1), ldq=256, hsq=128, k=self.at(2), ldk=128, hsk=128, v=self.at(3),
                 ldv=128, hsv=128, type=0, cu_q=self.at(4), k_start=self.at(5), k_len=self.at(6), n_seq=1, q_rows=3, k_rows=9,
                 max_q=3, max_k=9, heads=2, kv_heads=1, d=128, scale=0.1, ws=self.at(8), ws_bytes=1 << 18, stream=None)
        assert set(kw) <= set(d)
        d.update(kw)
        return self.q._op("qh_attention_seq")(*d.values())


@pytest.fixture(scope="module")
def args(q):
    return Args(q)


@pytest.mark.parametrize("kw", [
    dict(type=2), dict(tokens=-1), dict(out=0), dict(inn=0), dict(inn=40), dict(inn=131072), dict(y=None), dict(w=None),
    dict(scale=None), dict(xq=None), dict(sx=None), dict(ldx=72), dict(ldx=-64), dict(ldy=31), dict(ldy=-32), dict(ldy=1 << 41),
    "w+8", "xq+8", "y+2", "y=xq", "y=sx", "y=w", "y=scale",
], ids=str)
def test_gemm_refusals(q, args, kw):
    if isinstance(kw, str):
        name, what = kw.replace("=", "+").split("+")
        at = {"w": args.at(4), "xq": args.at(7), "y": args.at(0), "sx": args.at(8), "scale": args.at(6)}
        kw = {name: at[what] if "=" in kw else at[name] + int(what)}
    assert args.gemm(**kw) == q.QH_EINVAL


def test_gemm_nothing_to_do_and_ranges(q, args):
    assert args.gemm(tokens=0, y=None, xq=None, sx=None) == q.QH_OK
    assert args.gemm(tokens=(1 << 20) + 1) == q.QH_ERANGE
    assert args.gemm(out=(1 << 24) + 1, ldy=1 << 25) == q.QH_ERANGE


@pytest.mark.parametrize("kw", [
    dict(type=-1), dict(n_seq=-1), dict(tokens=-1), dict(max_len=-1), dict(k_heads=0), dict(heads=0), dict(heads=3, k_heads=2),
    dict(out=None), dict(q=None), dict(k=None), dict(v=None), dict(g=None), dict(beta=None), dict(S=None), dict(cu=None),
    dict(ldo=255), dict(ldo=128), dict(hso=64), dict(ldo=0), dict(ldq=126), dict(ldk=-128), dict(hsv=2), dict(ldg=-1), dict(ldb=1 << 41),
    "out+4", "q+4", "S+4", "out=q", "out=k", "out=v", "out=g", "out=beta", "out=S", "S=q", "S=v", "S=cu",
], ids=str)
def test_delta_refusals(q, args, kw):
    if isinstance(kw, str):
        name, what = kw.replace("=", "+").split("+")
        at = {"out": args.at(0), "q": args.at(1), "k": args.at(2), "v": args.at(3), "g": args.at(4), "beta": args.at(5),
              "S": args.at(8), "cu": args.at(6)}
        kw = {name: at[what] if "=" in kw else at[name] + int(what)}
    assert args.delta(**kw) == q.QH_EINVAL


def test_delta_nothing_to_do_and_ranges(q, args):
    assert args.delta(tokens=0) == q.QH_OK and args.delta(n_seq=0) == q.QH_OK
    assert args.delta(n_seq=1 << 29) == q.QH_ERANGE
    assert args.delta(tokens=1 << 30, heads=4, k_heads=2) == q.QH_ERANGE


@pytest.mark.parametrize("kw", [
    dict(type=7), dict(n_seq=-1), dict(q_rows=-1), dict(k_rows=-1), dict(max_q=-1), dict(max_k=-1), dict(heads=0), dict(kv_heads=0),
    dict(heads=3, kv_heads=2), dict(d=64), dict(d=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None),
    dict(q=None), dict(k=None), dict(v=None), dict(cu_q=None), dict(k_start=None), dict(k_len=None), dict(ldo=130), dict(ldo=0),
    dict(hso=0), dict(ldq=-256), dict(ldk=2), dict(ldv=-4), dict(hsq=2), "out+8", "k+4", "v+8", "out=q", "out=k", "out=v",
    "out=cu_q", "out=k_start", "out=k_len",
], ids=str)
def test_attention_refusals(q, args, kw):
    if isinstance(kw, str):
        name, what = kw.replace("=", "+").split("+")
        at = {"out": args.at(0), "q": args.at(1), "k": args.at(2), "v": args.at(3), "cu_q": args.at(4), "k_start": args.at(5),
              "k_len": args.at(6)}
        kw = {name: at[what] if "=" in kw else at[name] + int(what)}
    assert args.attn(**kw) == q.QH_EINVAL


def test_attention_nothing_to_do_ranges_and_workspace(q, args):
    assert args.attn(q_rows=0) == q.QH_OK and args.attn(n_seq=0) == q.QH_OK
    assert args.attn(max_k=(1 << 30) + 1) == q.QH_ERANGE
    assert args.attn(q_rows=1 << 30, heads=4) == q.QH_ERANGE
    need = q.attention_seq_workspace(3, 1, 1, 100000, 2, 1, 128)   # few rows, many keys: the keys are split
    assert need > 0
    for ws in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=args.at(8) + 16), dict(ws=args.at(1))):
        assert args.attn(max_q=1, max_k=100000, **{"ws_bytes": need, **ws}) == q.QH_EINVAL
    assert q.attention_seq_workspace(0, 1, 1, 100000, 2, 1, 128) == 0


def test_more_workgroups_than_a_grid_has(q, args):
    assert args.delta(n_seq=450001) == q.QH_ERANGE
    assert q.delta_rule_seq_workspace(1000, 450001, 2, 1000, k_heads=1) == 0
    assert args.attn(q_rows=33000000) == q.QH_ERANGE and args.attn(q_rows=4100000, n_seq=4100000) == q.QH_ERANGE


def test_interleaved_slices_are_no_overlap(q, args):
    """Columns of one buffer: refused where they meet, taken (as far as the next refusal) where they do not."""
    at = args.at(0)
    row = dict(ldo=1024, ldq=1024, ldk=1024, ldv=1024)
    good = dict(out=at, q=at + 4 * 256, k=at + 4 * 384, v=at + 4 * 512, **row)   # 256 + 128 + 128 + 256 of 1024
    assert args.delta(tokens=0, **good) == q.QH_OK
    assert args.delta(cu=None, **good) == q.QH_EINVAL
    for shift in (4 * 252, -4 * 4):   # q begins inside out; q wraps into the row's start of out
        assert args.delta(**{**good, "q": at + shift if shift > 0 else at + 4 * 1024 + shift}) == q.QH_EINVAL


def test_python_checks_need_no_gpu(q):
    import torch

    f = lambda *s: torch.zeros(*s)
    with pytest.raises(TypeError, match="CUDA"):
        q.gemm_i8_w8a8(f(2, 16), torch.zeros(16, 32, dtype=torch.int8), f(16), torch.zeros(2, 32, dtype=torch.int8), f(2))
    with pytest.raises(TypeError, match="CUDA"):
        q.attention_seq(f(2, 2, 128), f(2, 2, 128), f(2, 1, 128), f(2, 1, 128), torch.zeros(2, dtype=torch.int32),
                        torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), None, 2, 2)
    with pytest.raises(ValueError, match="dimensions"):
        q.delta_rule_seq(f(2, 2, 128), f(2, 2, 128), f(2, 2, 128), f(2, 256), f(2, 2), f(2, 2), f(1, 2, 128, 128),
                         torch.zeros(2, dtype=torch.int32), None, 2)
