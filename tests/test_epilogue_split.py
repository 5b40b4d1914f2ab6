"""How the 8-bit product's epilogue splits a tile among its warps
(pz_epilogue.cuh, compiled here for the host): every token of every quarter of
the lanes has exactly one owner, whatever the number of tokens.  It is what
the warps walk over to store logits, and what each fills with NaN when its
wait for the sums runs out: a token without an owner would keep what the
buffer held, one with two could lose what its partner stored."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-zero_b200", "csrc")

MAIN = r"""
#include <cstdio>
#include "pz_epilogue.cuh"
template <int W> int check() {
  using Own = pz::EpilogueTokens<W>;
  for (int tokens = 0; tokens <= 256; tokens++) {
    int owners[4][288] = {};
    for (int e = 0; e < W; e++) {
      const int warp = e + 2;  // two warps before the epilogue's
      for (int c = Own::first(e); c < tokens; c += Own::STEP) {
        const int n = Own::count(c, tokens);
        if (n < 1 || n > 32) return 1;
        for (int j = 0; j < n; j++) owners[Own::quarter(warp)][c + j]++;
      }
    }
    for (int q = 0; q < 4; q++)
      for (int t = 0; t < 288; t++)
        if (owners[q][t] != (t < tokens ? 1 : 0)) {
          std::printf("W=%d tokens=%d quarter=%d token=%d owners=%d\n", W, tokens, q, t, owners[q][t]);
          return 1;
        }
  }
  return 0;
}
int main() { return check<4>() + check<8>() + check<12>(); }
"""


def test_every_token_has_one_owner(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "split.cpp", tmp_path / "split"
    src.write_text(MAIN)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
