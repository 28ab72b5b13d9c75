"""Which kernels the tested shapes of the 8-bit linear run, by the library's own rule compiled for
the CPU: every one that some shape gets. No GPU."""
import pathlib
import shutil
import subprocess

import pytest

from _serving_shapes import DECODE, TILES

CSRC = pathlib.Path(__file__).resolve().parent.parent / "turing-bf16_amd" / "csrc"

# the form of each line's (M, K, N), then a line "all" and the forms that a sweep over shapes finds
PROGRAM = r"""
#include <cstdio>
#include <set>
#include <string>
#include "gemm_i8_plan.h"
using namespace tbf16::i8;
std::string form(long M, long K, long N) {
  const Plan p = plan_of(M, K, N, K % 8 == 0, 256);
  char s[64];
  if (p.decode) snprintf(s, 64, "decode T=%d fused=%d", p.T, p.fused);
  else snprintf(s, 64, "tile=%d splits=%d narrow=%d", p.tile, p.splits, (int)(p.rows < kTiles[p.tile].bn));
  return s;
}
int main() {
  long M, K, N;
  while (scanf("%ld %ld %ld", &M, &K, &N) == 3) puts(form(M, K, N).c_str());
  std::set<std::string> all;
  for (M = 1; M < 20000; M += M < 20 ? 1 : M / 14)
    for (K = 8; K <= 131072; K += K / 8 * 2 + 1)
      for (N = 8; N < 140000; N += N / 14 + 1)
        if ((double)N * K < 1e9) all.insert(form(M, K, N)), all.insert(form(M, K / 8 * 8, N));
  puts("all");
  for (auto& s : all) puts(s.c_str());
}
"""


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("forms")
    (d / "forms.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(d / "forms.cpp"), "-o", str(d / "forms")], check=True)
    asked = "\n".join(" ".join(map(str, s)) for s in DECODE + TILES)
    out = subprocess.run([str(d / "forms")], input=asked, check=True, capture_output=True, text=True).stdout.splitlines()
    cut = out.index("all")
    return dict(zip(DECODE + TILES, out[:cut])), set(out[cut + 1:])


def test_every_form_is_tested(forms):
    tested, found = forms
    assert len(found) > 40
    assert found <= set(tested.values()), sorted(found - set(tested.values()))


def test_shapes_are_of_their_list(forms):
    tested, _ = forms
    assert all(tested[s].startswith("decode") for s in DECODE) and all(tested[s].startswith("tile") for s in TILES)
