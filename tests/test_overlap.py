"""The host's check for tensors that share memory (csrc/hk_overlap.h), compiled for the CPU: against the bytes of small
layouts one by one, and on large ones."""
from __future__ import annotations

import subprocess

from conftest import ROOT

DRIVER = r"""
#include <stdio.h>
#include <stdlib.h>
#include <set>
#include <vector>
#include "hk_overlap.h"
using hk::Rows;

struct Layout { int64_t lo, elem, cols, n[3], step[3]; };
static Rows rows(const Layout& l) {
  Rows r(reinterpret_cast<void*>(l.lo), l.elem, l.cols);
  for (int i = 0; i < 3; ++i) r.along(l.n[i], l.step[i]);
  return r;
}
// every byte, once for each row it is in
static std::vector<int64_t> bytes(const Layout& l) {
  std::vector<int64_t> v;
  for (int64_t i = 0; i < l.n[0]; ++i)
    for (int64_t j = 0; j < l.n[1]; ++j)
      for (int64_t k = 0; k < l.n[2]; ++k)
        for (int64_t c = 0; c < l.elem * l.cols; ++c)
          v.push_back(l.lo + i * l.step[0] + j * l.step[1] + k * l.step[2] + c);
  return v;
}
static int64_t pick(int64_t lo, int64_t hi) { return lo + rand() % (hi - lo + 1); }

int main() {
  srand(1);
  int met = 0, apart = 0, self = 0, loose = 0;
  for (int t = 0; t < 300000; ++t) {
    Layout l[2];
    for (int w = 0; w < 2; ++w) {
      Layout& a = l[w];
      a.lo = 10000 + pick(0, 60), a.elem = 1 << pick(0, 2), a.cols = pick(0, 4);
      // views of a tensor [n0][n1][n2][pitch], in any order, with gaps
      const int64_t pitch = a.elem * (a.cols + pick(0, 9));
      int64_t inner = pitch;
      const int first = pick(0, 2);
      for (int i = 0; i < 3; ++i) {
        const int d = (first + i) % 3;
        a.n[d] = pick(rand() % 20 == 0 ? 0 : 1, 3);
        a.step[d] = inner;
        inner *= a.n[d] > 0 ? a.n[d] : 1;
        if (rand() % 4 == 0) inner += a.elem * pick(0, 3);
        if (rand() % 12 == 0) a.step[d] = a.elem * pick(-6, 6);  // anything at all
      }
      if (w == 1 && rand() % 2) {  // the same layout elsewhere
        const int64_t lo = a.lo;
        a = l[0];
        a.lo = rand() % 3 ? lo : a.lo;
      }
    }
    const auto x = bytes(l[0]), y = bytes(l[1]);
    const std::set<int64_t> sx(x.begin(), x.end()), sy(y.begin(), y.end());
    bool meet = false;
    for (int64_t b : sx) meet |= sy.count(b) > 0;
    const Rows a = rows(l[0]), b = rows(l[1]);
    if (hk::overlap(a, b) != meet || hk::overlap(b, a) != meet) return printf("overlap %d\n", t), 1;
    if (hk::overlaps_itself(a) != (sx.size() != x.size())) return printf("itself %d\n", t), 1;
    const bool same = a.same(b);
    if (same && x != y) return printf("same %d\n", t), 1;
    if (hk::overlap_unless_same(a, b) != (meet && !same)) return printf("unless same %d\n", t), 1;
    met += meet, apart += !meet, self += sx.size() != x.size(), loose += same;
  }
  if (met < 1000 || apart < 1000 || self < 1000 || loose < 1000) return printf("too few\n"), 1;

  // a packed projection [B][T][q + 2 k heads][d] of 2^40 bytes: its parts lie apart, shifted ones do not
  const int64_t d = 128, H = 16, K = 4, T = 1 << 20, B = 512, row = (H + 2 * K) * d * 2;
  auto part = [&](int64_t at, int64_t heads) {
    return Rows(reinterpret_cast<void*>(int64_t{1} << 20), 2, d).along(B, T * row).along(T, row).along(heads, 2 * d);
  };
  Rows q = part(0, H), k = part(0, K), v = part(0, K);
  k.lo += H * d * 2, v.lo += (H + K) * d * 2;
  if (hk::overlap(q, k) || hk::overlap(k, v) || hk::overlap(q, v) || hk::overlaps_itself(q)) return printf("packed\n"), 1;
  // the same rows in another order are other elements
  Rows one = Rows(reinterpret_cast<void*>(4096), 2, 8).along(5, 80).along(5, 16);
  Rows turned = Rows(reinterpret_cast<void*>(4096), 2, 8).along(5, 16).along(5, 80);
  if (one.same(turned) || !hk::overlap_unless_same(one, turned) || !one.same(one)) return printf("turned\n"), 1;
  k.lo -= 2;
  if (!hk::overlap(q, k) || hk::overlap(k, v)) return printf("shifted\n"), 1;
  // 65,535 batches whose rows interleave, and batches of them one row into each other
  Rows c = Rows(reinterpret_cast<void*>(4096), 2, 64).along(1 << 20, 65535 * 128).along(65535, 128);
  if (hk::overlaps_itself(c)) return printf("interleaved\n"), 1;
  Rows e = Rows(reinterpret_cast<void*>(4096), 2, 64).along(1000, 128).along(65535, 999 * 128);
  if (!hk::overlaps_itself(e)) return printf("one row\n"), 1;
  // no memory
  if (hk::overlap(Rows(nullptr, 2, 8), c) || hk::overlap(Rows(reinterpret_cast<void*>(4096), 2, 0), c)) return printf("none\n"), 1;
  printf("ok %d %d %d %d\n", met, apart, self, loose);
  return 0;
}
"""


def test_against_single_bytes(tmp_path):
    src = tmp_path / "overlap.cpp"
    src.write_text(DRIVER)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", f"-I{ROOT / 'hyperkernels_amd' / 'csrc'}",
                    str(src), "-o", str(tmp_path / "overlap")], check=True)
    out = subprocess.run([str(tmp_path / "overlap")], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout
